// Causal sliding-window attention with sinks on (batch, length, channels)
// signals: forward on the matrix cores; backward with one wavefront a row.
#include "token_tile.h"

namespace circatt {
namespace {

using namespace tok;
constexpr float kLog2e = 1.4426950408889634f;

__device__ __forceinline__ int signal_length(const SlidingProblem &pr, int b) {
    if (pr.lengths == nullptr) return pr.L;
    const int n = pr.lengths[b];
    return n < 0 ? 0 : n < pr.L ? n : pr.L;
}

template <typename T>
struct Row {
    int b, i, hk, g, n;
    int64_t stat;  // in lse and dsum
    SignalKV<T> kv;
    // row numbers run over heads, then tokens, then signals
    __device__ Row(const SlidingProblem &pr, int64_t r) {
        const int h = (int)(r % pr.H);
        r /= pr.H;
        i = (int)(r % pr.L);
        b = (int)(r / pr.L);
        hk = h / pr.G;
        g = h - hk * pr.G;
        n = signal_length(pr, b);
        stat = (((int64_t)b * pr.Hk + hk) * pr.L + i) * pr.G + g;
        kv = SignalKV<T>{static_cast<const T *>(pr.k) + b * pr.k_batch + (int64_t)hk * pr.D,
                         static_cast<const T *>(pr.v) + b * pr.v_batch + (int64_t)hk * pr.D, pr.k_row, pr.v_row};
    }
    __device__ int64_t channel(const SlidingProblem &pr) const { return (int64_t)(hk * pr.G + g) * pr.D; }
};

// ---------------------------------------------------------------------------
// Forward.  A workgroup has 128 query rows of one head of keys, row r being head
// r % G of token r / G, so that the heads that share keys share their tiles and
// their window: 32 rows a wavefront, tiles of KT keys and values in LDS, the
// next tile on its way while one is worked on (two buffers, one barrier a tile).
// Workgroups that share a head of keys run on one XCD (ids 8 apart), whose L2
// then holds their common tiles.
template <typename T, int DP>
struct FwdShape {
    // Float32 rows are twice as long: half the keys fill the same LDS
    static constexpr int KT = sizeof(T) == 2 ? 64 : 32;
    static constexpr int TILE = KT * Tile<T, DP>::ROW;
};

struct BlockOrder {
    int block, unit;  // row block (last ones first), signal and head of keys
    // n units of blocks row blocks each over a grid of a multiple of 8
    __device__ BlockOrder(int n, int blocks) {
        const int64_t id = (int64_t)(blockIdx.x & 7) * (gridDim.x >> 3) + (blockIdx.x >> 3);
        unit = (int)(id / blocks);
        block = blocks - 1 - (int)(id - (int64_t)unit * blocks);
        if (unit >= n) unit = -1;
    }
};
unsigned grid8(int64_t n) { return (unsigned)((n + 7) / 8 * 8); }

// Rows [k0, k0 + KT) of one head from p (row bytes rb apart, n rows of D
// channels in all) into LDS; rows from n on and units from D on are zeros.
template <typename T, int DP, int KT, int THREADS>
__device__ __forceinline__ void fetch_rows(const T *p, int64_t row, int k0, int n, int D, const CIRCATT_LDS char *to) {
    typedef Tile<T, DP> Tl;
    const int rb = (int)(row * (int)sizeof(T)), units = D * (int)sizeof(T) / 16;
    const int64_t bytes = n > k0 ? (int64_t)(n - 1 - k0) * rb + units * 16 : 0;
    const dma::i4v rs = dma::dma_rsrc(reinterpret_cast<const float *>(p + k0 * row),
                                      (int)(bytes < dma::kMaxBytes ? bytes : dma::kMaxBytes));
    const int tid = threadIdx.x;
    const unsigned m0 = lds_byte(to) + uniform(tid >> 6) * 1024;
#pragma unroll
    for (int k = 0; k < KT * Tl::PC / THREADS; ++k) {
        const int slot = tid + k * THREADS, r = slot / Tl::PC, u = (slot % Tl::PC) ^ Tl::f(r);
        dma::dma16(rs, m0 + k * THREADS * 16, u < units ? r * rb + u * 16 : dma::kOut, 0);
    }
}

template <typename T, int DP>
__global__ __launch_bounds__(256, sizeof(T) == 4 && DP > 64 ? 1 : 2) void sliding_fwd(SlidingProblem pr, int blocks) {
    typedef FwdShape<T, DP> Sh;
    constexpr int KT = Sh::KT, NB = KT / 32;
    __shared__ char lds_mem[4 * Sh::TILE];
    const CIRCATT_LDS char *lds = (const CIRCATT_LDS char *)lds_mem;
    const BlockOrder w(pr.B * pr.Hk, blocks);
    if (w.unit < 0) return;
    const int b = w.unit / pr.Hk, hk = w.unit - b * pr.Hk, n = uniform(signal_length(pr, b));
    const int lane = threadIdx.x & 63, wave = uniform(threadIdx.x >> 6);
    const int rows = n * pr.G, r0 = w.block * 128, all_rows = pr.L * pr.G;
    const int r = r0 + 32 * wave + (lane & 31);
    T *y = static_cast<T *>(pr.y) + (int64_t)b * pr.L * pr.H * pr.D + (int64_t)hk * pr.G * pr.D;
    const int64_t stat = ((int64_t)b * pr.Hk + hk) * all_rows;
    // the wavefront's rows, those past the end doubling the last one
    const int rr = r < rows ? r : rows - 1, at = rows > 0 ? rr / pr.G : -1, g = rows > 0 ? rr - at * pr.G : 0;
    const int lo = uniform(at), hi = __builtin_amdgcn_readlane(at, 31);
    const bool live = r0 + 32 * wave < rows;
    if (r0 < rows) {
        const int last = r0 + 127 < rows ? r0 + 127 : rows - 1;
        const T *kh = static_cast<const T *>(pr.k) + b * pr.k_batch + (int64_t)hk * pr.D;
        const T *vh = static_cast<const T *>(pr.v) + b * pr.v_batch + (int64_t)hk * pr.D;
        const T *qh = static_cast<const T *>(pr.q) + b * pr.q_batch + (int64_t)hk * pr.G * pr.D;
        const Sight see{pr.W, pr.S};
        const TileList<KT> tiles(r0 / pr.G, last / pr.G, pr.W, pr.S);
        const float c = pr.scale * kLog2e;
        auto fetch = [&](int i) {
            const int k0 = tiles.key(i);
            fetch_rows<T, DP, KT, 256>(kh, pr.k_row, k0, n, pr.D, lds + (i & 1) * 2 * Sh::TILE);
            fetch_rows<T, DP, KT, 256>(vh, pr.v_row, k0, n, pr.D, lds + (i & 1) * 2 * Sh::TILE + Sh::TILE);
        };
        Rows<T, DP> x;
        fetch(0);
        x.start(qh + at * pr.q_row + (int64_t)g * pr.D, pr.D, lane);
        for (int i = 0; i < tiles.count; ++i) {
            dma_barrier();
            if (i + 1 < tiles.count) fetch(i + 1);
            const int k0 = tiles.key(i);
            const CIRCATT_LDS char *kt = lds + (i & 1) * 2 * Sh::TILE;
            if (!live || see.none(lo, hi, k0, KT)) continue;
            if (see.all(lo, hi, k0, KT)) x.template tile<NB, false>(kt, kt + Sh::TILE, lane, at, k0, see, 0, c);
            else x.template tile<NB, true>(kt, kt + Sh::TILE, lane, at, k0, see, 0, c);
        }
        if (live) {
            const float l = x.total(), inv = l == 0.f ? 0.f : 1.f / l;
            bool bad = false;
            if (r < rows) {
                bad = x.store(y + ((int64_t)at * pr.H + g) * pr.D, pr.D, lane, inv);
                if (pr.lse != nullptr && lane < 32)
                    pr.lse[stat + r] = l == 0.f ? INFINITY : x.m + __builtin_amdgcn_logf(l);
            }
            // A value that is not finite reaches, as 0 times itself, every row of
            // a wavefront whose tile holds it: such rows are formed again from
            // the keys that they see alone.
            uint64_t again = __ballot(bad);
            again = (again | again >> 32) & 0xffffffffu;
            const SignalKV<T> kv{kh, vh, pr.k_row, pr.v_row};
            for (; again; again &= again - 1) {
                const int j = __builtin_ctzll(again);
                const int aj = __builtin_amdgcn_readlane(at, j), gj = __builtin_amdgcn_readlane(g, j);
                forward_row(qh + aj * pr.q_row + (int64_t)gj * pr.D, y + ((int64_t)aj * pr.H + gj) * pr.D,
                            (float *)nullptr, kv, aj, pr.W, pr.S, pr.D, c);
            }
        }
    }
    // rows behind the signal's length
    if (r >= rows && r < all_rows) {
        const int t = r / pr.G, gt = r - t * pr.G;
        T *z = y + ((int64_t)t * pr.H + gt) * pr.D;
        for (int d = 4 * (lane >> 5); d < pr.D; d += 8) *reinterpret_cast<V4<T> *>(z + d) = V4<T>{};
        if (pr.lse != nullptr && lane < 32) pr.lse[stat + r] = INFINITY;
    }
}

template <typename T>
__global__ __launch_bounds__(256) void sliding_dq_rows(SlidingProblem pr) {
    const int64_t r = (int64_t)blockIdx.x * 4 + (threadIdx.x >> 6);
    if (r >= (int64_t)pr.B * pr.L * pr.H) return;
    const Row<T> w(pr, r);
    const int64_t out = ((int64_t)w.b * pr.L + w.i) * pr.H * pr.D + w.channel(pr);
    dq_row(static_cast<const T *>(pr.q) + w.b * pr.q_batch + w.i * pr.q_row + w.channel(pr),
           static_cast<const T *>(pr.y) + out,
           static_cast<const T *>(pr.dy) + w.b * pr.dy_batch + w.i * pr.dy_row + w.channel(pr),
           static_cast<T *>(pr.dq) + out, pr.lse[w.stat], pr.work + w.stat, w.kv, w.i < w.n ? w.i : -1, pr.W, pr.S,
           pr.D, pr.scale * kLog2e, pr.scale);
}

template <typename T>
__global__ __launch_bounds__(256) void sliding_dkdv_rows(SlidingProblem pr) {
    int64_t r = (int64_t)blockIdx.x * 4 + (threadIdx.x >> 6);
    if (r >= (int64_t)pr.B * pr.L * pr.Hk) return;
    const int hk = (int)(r % pr.Hk);
    r /= pr.Hk;
    const int j = (int)(r % pr.L), b = (int)(r / pr.L), n = signal_length(pr, b);
    const int64_t out = ((int64_t)b * pr.L + j) * pr.Hk * pr.D + (int64_t)hk * pr.D;
    const int64_t stat = ((int64_t)b * pr.Hk + hk) * pr.L * pr.G;
    dkdv_row(static_cast<const T *>(pr.k) + b * pr.k_batch + j * pr.k_row + (int64_t)hk * pr.D,
             static_cast<const T *>(pr.v) + b * pr.v_batch + j * pr.v_row + (int64_t)hk * pr.D,
             static_cast<const T *>(pr.q) + b * pr.q_batch + (int64_t)hk * pr.G * pr.D, pr.q_row,
             static_cast<const T *>(pr.dy) + b * pr.dy_batch + (int64_t)hk * pr.G * pr.D, pr.dy_row, pr.lse + stat,
             pr.work + stat, static_cast<T *>(pr.dk) + out, static_cast<T *>(pr.dv) + out, j, n, pr.W, pr.S, pr.G,
             pr.D, pr.scale * kLog2e, pr.scale);
}

template <typename T, int DP>
hipError_t forward(const SlidingProblem &pr, hipStream_t s) {
    const int blocks = (pr.L * pr.G + 127) / 128;
    sliding_fwd<T, DP><<<grid8((int64_t)pr.B * pr.Hk * blocks), 256, 0, s>>>(pr, blocks);
    return hipGetLastError();
}
template <int DT>
hipError_t forward(const SlidingProblem &pr, hipStream_t s) {
    typedef typename Elem<DT>::T T;
    return pr.D <= 32 ? forward<T, 32>(pr, s)
                      : pr.D <= 64 ? forward<T, 64>(pr, s) : pr.D <= 96 ? forward<T, 96>(pr, s) : forward<T, 128>(pr, s);
}
template <int DT>
hipError_t backward(const SlidingProblem &pr, hipStream_t s) {
    typedef typename Elem<DT>::T T;
    const int64_t rows = (int64_t)pr.B * pr.L * pr.H, keys = (int64_t)pr.B * pr.L * pr.Hk;
    sliding_dq_rows<T><<<(unsigned)((rows + 3) / 4), 256, 0, s>>>(pr);
    if (pr.dk != nullptr) sliding_dkdv_rows<T><<<(unsigned)((keys + 3) / 4), 256, 0, s>>>(pr);
    return hipGetLastError();
}

}  // namespace

int64_t sliding_bwd_workspace_floats(const SlidingProblem &pr) { return (int64_t)pr.B * pr.L * pr.H; }

hipError_t launch_sliding_fwd(const SlidingProblem &pr, hipStream_t s) {
    return pr.dtype == CIRCATT_F32 ? forward<0>(pr, s) : pr.dtype == CIRCATT_F16 ? forward<2>(pr, s) : forward<3>(pr, s);
}
hipError_t launch_sliding_bwd(const SlidingProblem &pr, hipStream_t s) {
    return pr.dtype == CIRCATT_F32 ? backward<0>(pr, s)
                                   : pr.dtype == CIRCATT_F16 ? backward<2>(pr, s) : backward<3>(pr, s);
}

}  // namespace circatt
