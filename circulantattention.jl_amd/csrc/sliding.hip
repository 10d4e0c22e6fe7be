// Causal sliding-window attention with sinks on (batch, length, channels)
// signals, forward and backward, on the matrix cores.
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
    typedef Ring<T, DP> Rg;
    constexpr int KT = Rg::KT, NB = Rg::NB;
    __shared__ char lds_mem[Rg::BYTES];
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
        const Feed<T, DP> fk(kh, pr.k_row, n, pr.D), fv(vh, pr.v_row, n, pr.D);
        const unsigned ring = lds_byte(lds);
        const int count = uniform(tiles.count);
        // places of K tile i + 1 (and i + 3, i) and V tile i (i + 1: the other)
        int kp = 0, vp = 1;
        auto round = [&](int i) {
            Rg::wait(i + 2 < count);
            if (i + 1 < count) fv.fetch(tiles.key(i + 1), ring + Rg::V + (vp ^ 1) * Rg::TILE);
            if (i + 3 < count) fk.fetch(tiles.key(i + 3), ring + (kp == 0 ? 2 : kp - 1) * Rg::TILE);
        };
        auto next = [&] {
            kp = kp == 2 ? 0 : kp + 1;
            vp ^= 1;
        };
        fk.fetch(tiles.key(0), ring);
        if (count > 1) fk.fetch(tiles.key(1), ring + Rg::TILE);
        Rows<T, DP> x;
        x.start(qh + at * pr.q_row + (int64_t)g * pr.D, pr.D, lane);
        // the tiles that this wavefront's rows see: from `first` to `end`, but for
        // those that the list leaves out
        int first = 0, end = live ? count - 1 : -1;
        while (first < end && see.none(lo, hi, tiles.key(first), KT)) ++first;
        while (end > first && see.none(lo, hi, tiles.key(end), KT)) --end;
        const unsigned row_at = Tile<T, DP>::row_lane(lane) + ring, col_at = Tile<T, DP>::col_lane(lane) + ring + Rg::V;
        float mx = 0.f;
        auto look = [&](f16v (&s)[NB], int i) {  // hide keys of tile i, largest score
            const int k0 = tiles.key(i);
            if (!see.all(lo, hi, k0, KT)) {
                asm volatile("");  // a branch: few tiles need it
#pragma unroll
                for (int m = 0; m < NB; ++m) {
                    const int b0 = at + 1 - k0 - 32 * m, s0 = pr.S - k0 - 32 * m;
                    const uint32_t half = (bits_between(b0 - pr.W, b0) | bits_between(0, b0 < s0 ? b0 : s0)) >> (4 * (lane >> 5));
#pragma unroll
                    for (int y = 0; y < 16; ++y)
                        if (!(half & place_bit(y))) s[m][y] = -INFINITY;
                }
            }
            mx = x.largest(s) * c;
        };
        auto step = [&](const f16v (&s)[NB], f16v (&t)[NB], int i) {
            round(i);
            V8<T> p[2 * NB];
            x.raise(mx);
            x.scores(row_at + kp * Rg::TILE, t);
            x.weigh(s, p, c);
            x.template add<NB>(col_at + vp * Rg::TILE, p);
            next();
            look(t, i + 1);
        };
        f16v a[NB], b[NB];
        int i = -1;
        for (; i < (live ? first - 1 : count); ++i, next()) round(i);
        if (live) {
            round(i);
            x.scores(row_at + kp * Rg::TILE, a);
            look(a, first);
            next();
            ++i;
            for (; i + 1 < end; i += 2) {
                step(a, b, i);
                step(b, a, i + 1);
            }
            if (i < end) {
                step(a, b, i);
#pragma unroll
                for (int m = 0; m < NB; ++m) a[m] = b[m];
                ++i;
            }
            round(i);
            V8<T> p[2 * NB];
            x.raise(mx);
            x.weigh(a, p, c);
            x.template add<NB>(col_at + vp * Rg::TILE, p);
            next();
            for (++i; i < count; ++i, next()) round(i);
        }
        if (live) {
            const float l = x.total(), inv = l == 0.f ? 0.f : 1.f / l;
            bool bad = false;
            if (r < rows) {
                bad = store_channels(x.o, y + ((int64_t)at * pr.H + g) * pr.D, pr.D, lane, inv);
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
        zero_channels(y + ((int64_t)t * pr.H + gt) * pr.D, pr.D, lane);
        if (pr.lse != nullptr && lane < 32) pr.lse[stat + r] = INFINITY;
    }
}

// ---------------------------------------------------------------------------
// Backward, queries: the forward's blocks and tiles.  A wavefront keeps q and dy
// of its 32 rows as second operands; for 32 keys at a time it forms S' = K Q'
// and dP' = V dY', from them dS' = P' (dP' - d) in the layout of a second
// operand, and dQ' += K' dS' with K' by the transposing reads.
template <typename T, int DP>
__global__ __launch_bounds__(256, sizeof(T) == 4 && DP > 32 ? 1 : 2) void sliding_dq(SlidingProblem pr, int blocks) {
    typedef FwdShape<T, DP> Sh;
    typedef Tile<T, DP> Tl;
    constexpr int KT = Sh::KT, STEPS = DP / 16, OT = DP / 32;
    __shared__ char lds_mem[4 * Sh::TILE];
    const CIRCATT_LDS char *lds = (const CIRCATT_LDS char *)lds_mem;
    const BlockOrder w(pr.B * pr.Hk, blocks);
    if (w.unit < 0) return;
    const int b = w.unit / pr.Hk, hk = w.unit - b * pr.Hk, n = uniform(signal_length(pr, b));
    const int lane = threadIdx.x & 63, wave = uniform(threadIdx.x >> 6);
    const int rows = n * pr.G, r0 = w.block * 128, all_rows = pr.L * pr.G;
    const int r = r0 + 32 * wave + (lane & 31);
    const int64_t head = (int64_t)b * pr.L * pr.H * pr.D + (int64_t)hk * pr.G * pr.D;
    T *dq = static_cast<T *>(pr.dq) + head;
    const int64_t stat = ((int64_t)b * pr.Hk + hk) * all_rows;
    const int rr = r < rows ? r : rows - 1, at = rows > 0 ? rr / pr.G : -1, g = rows > 0 ? rr - at * pr.G : 0;
    const int lo = uniform(at), hi = __builtin_amdgcn_readlane(at, 31);
    const bool live = r0 + 32 * wave < rows;
    if (r0 < rows) {
        const int last = r0 + 127 < rows ? r0 + 127 : rows - 1;
        const T *kh = static_cast<const T *>(pr.k) + b * pr.k_batch + (int64_t)hk * pr.D;
        const T *vh = static_cast<const T *>(pr.v) + b * pr.v_batch + (int64_t)hk * pr.D;
        const T *qh = static_cast<const T *>(pr.q) + b * pr.q_batch + (int64_t)hk * pr.G * pr.D;
        const T *gh = static_cast<const T *>(pr.dy) + b * pr.dy_batch + (int64_t)hk * pr.G * pr.D;
        const T *yh = static_cast<const T *>(pr.y) + head;
        const Sight see{pr.W, pr.S};
        const TileList<KT> tiles(r0 / pr.G, last / pr.G, pr.W, pr.S);
        const float c = pr.scale * kLog2e;
        auto fetch = [&](int i) {
            const int k0 = tiles.key(i);
            fetch_rows<T, DP, KT, 256>(kh, pr.k_row, k0, n, pr.D, lds + (i & 1) * 2 * Sh::TILE);
            fetch_rows<T, DP, KT, 256>(vh, pr.v_row, k0, n, pr.D, lds + (i & 1) * 2 * Sh::TILE + Sh::TILE);
        };
        fetch(0);
        V8<T> q[STEPS], dy[STEPS];
        f16v o[OT];
        float d = 0.f;
        const int64_t out = ((int64_t)at * pr.H + g) * pr.D;
#pragma unroll
        for (int k = 0; k < STEPS; ++k) {
            const int ch = 16 * k + 8 * (lane >> 5);
            q[k] = load8(qh + at * pr.q_row + (int64_t)g * pr.D, ch, pr.D);
            dy[k] = load8(gh + at * pr.dy_row + (int64_t)g * pr.D, ch, pr.D);
            const V8<T> y = load8(yh + out, ch, pr.D);
#pragma unroll
            for (int j = 0; j < 8; ++j) d = fmaf((float)y[j], (float)dy[k][j], d);
        }
        d += __shfl_xor(d, 32, 64);
        const float lse = pr.lse[stat + rr];
        if (r < rows && lane < 32) pr.work[stat + r] = d;
#pragma unroll
        for (int t = 0; t < OT; ++t) o[t] = f16v{};
        const unsigned row_at = Tl::row_lane(lane), col_at = Tl::col_lane(lane);
        for (int i = 0; i < tiles.count; ++i) {
            dma_barrier();
            if (i + 1 < tiles.count) fetch(i + 1);
            if (!live) continue;
            for (int m = 0; m < KT; m += 32) {
                const int k0 = tiles.key(i) + m;
                if (see.none(lo, hi, k0, 32)) continue;
                const unsigned to = lds_byte(lds) + (i & 1) * 2 * Sh::TILE + m * Tl::ROW;
                const unsigned kr = row_at + to, vr = kr + Sh::TILE, kc = col_at + to;
                f16v s = f16v{}, dp = f16v{};
#pragma unroll
                for (int k = 0; k < STEPS; ++k) {
                    s = mma(Tl::row(kr, 0, k), q[k], s);
                    dp = mma(Tl::row(vr, 0, k), dy[k], dp);
                }
#pragma unroll
                for (int x = 0; x < 16; ++x) s[x] = __builtin_amdgcn_exp2f(fmaf(s[x], c, -lse)) * (dp[x] - d);
                if (!see.all(lo, hi, k0, 32)) {
#pragma unroll
                    for (int x = 0; x < 16; ++x)
                        if (!see(at, k0 + 8 * (x >> 2) + 4 * (lane >> 5) + (x & 3))) s[x] = 0.f;
                }
                V8<T> ds[2];
#pragma unroll
                for (int x = 0; x < 16; ++x) ds[x >> 3][x & 7] = (T)s[x];
#pragma unroll
                for (int t = 0; t < OT; ++t)
#pragma unroll
                    for (int h = 0; h < 2; ++h) o[t] = mma(Tl::col(kc, 16 * h, t), ds[h], o[t]);
            }
        }
        if (live) {
            uint64_t again = __ballot(r < rows && store_channels(o, dq + out, pr.D, lane, pr.scale));
            again = (again | again >> 32) & 0xffffffffu;
            const SignalKV<T> kv{kh, vh, pr.k_row, pr.v_row};
            for (; again; again &= again - 1) {
                const int j = __builtin_ctzll(again);
                const int aj = __builtin_amdgcn_readlane(at, j), gj = __builtin_amdgcn_readlane(g, j);
                const int64_t oj = ((int64_t)aj * pr.H + gj) * pr.D, sj = stat + (int64_t)aj * pr.G + gj;
                dq_row(qh + aj * pr.q_row + (int64_t)gj * pr.D, yh + oj, gh + aj * pr.dy_row + (int64_t)gj * pr.D, dq + oj,
                       pr.lse[sj], pr.work + sj, kv, aj, pr.W, pr.S, pr.D, c, pr.scale);
            }
        }
    }
    if (r >= rows && r < all_rows) {
        const int t = r / pr.G;
        zero_channels(dq + ((int64_t)t * pr.H + r - t * pr.G) * pr.D, pr.D, lane);
    }
}

// ---------------------------------------------------------------------------
// Backward, keys: a workgroup has 128 keys of one head, 32 a wavefront, whose k
// and v it keeps as second operands, and walks the query rows that see them in
// tiles of QT rows of q and dy in LDS: S = Q K', dP = dY V' (lane: one key;
// registers: query rows), P and dS = P (dP - d) as second operands of
// dV' += dY' P and dK' += Q' dS with dY' and Q' by the transposing reads.
//
// Blocks whose walk is long (sinks are seen to the signal's end; a causal
// window without end; few signals and heads) are split over workgroups by the
// tiles of the walk: each leaves Float32 partial sums, added up in order by
// sliding_dkdv_join.
template <typename T, int DP>
struct BwdShape {
    static constexpr int QT = sizeof(T) == 2 ? 64 : 32;
    static constexpr int TILE = QT * Tile<T, DP>::ROW;
    static constexpr int PART = 128 * DP * 2;  // floats of one partial pair
};

// How the walk is split: blocks of keys below `far` see the signal's end.
struct WalkSplit {
    int blocks, far, parts_far, parts;  // of 128 keys; workgroups a block of each kind
    FastDiv heads;                      // G
    int64_t units, far_units;           // workgroups for one signal and head of keys
};

struct Walk {
    int first, count;  // packed query rows from first on, tiles
    __device__ Walk(const SlidingProblem &pr, int kb, int n, int QT) {
        const int k0 = kb * 128, kn = k0 + 127 < n - 1 ? k0 + 127 : n - 1;
        int end = n;
        if (k0 >= pr.S && n - kn > pr.W) end = kn + pr.W;
        first = k0 * pr.G;
        count = k0 < n ? ((end - k0) * pr.G + QT - 1) / QT : 0;
    }
};

// Packed query rows [r0, r0 + QT) of a head group: row r is head r % G of token
// r / G; rows behind token n - 1 are zeros.
template <typename T, int DP, int QT>
__device__ __forceinline__ void fetch_packed(const T *p, int64_t row, int r0, int G, FastDiv dg, int n, int D,
                                             const CIRCATT_LDS char *to) {
    typedef Tile<T, DP> Tl;
    const int rb = (int)(row * (int)sizeof(T)), units = D * (int)sizeof(T) / 16;
    const int t0 = uniform(fdiv(r0, dg));
    const int64_t bytes = n > t0 ? (int64_t)(n - 1 - t0) * rb + G * units * 16 : 0;
    const dma::i4v rs = dma::dma_rsrc(reinterpret_cast<const float *>(p + t0 * row),
                                      (int)(bytes < dma::kMaxBytes ? bytes : dma::kMaxBytes));
    const int tid = threadIdx.x;
    const unsigned m0 = lds_byte(to) + uniform(tid >> 6) * 1024;
#pragma unroll
    for (int k = 0; k < QT * Tl::PC / 256; ++k) {
        const int slot = tid + k * 256, rl = slot / Tl::PC, u = (slot % Tl::PC) ^ Tl::f(rl);
        const int t = fdiv(r0 + rl, dg), g = r0 + rl - t * G;
        dma::dma16(rs, m0 + k * 4096, u < units ? (t - t0) * rb + (g * units + u) * 16 : dma::kOut, 0);
    }
}
// QT floats from p on into LDS by the calling wavefront, zeros behind p[rows - 1]
template <int QT>
__device__ __forceinline__ void fetch_stats(const float *p, int r0, int rows, const CIRCATT_LDS char *to) {
    const dma::i4v rs = dma::dma_rsrc(p + r0, rows > r0 ? (rows - r0 < QT ? rows - r0 : QT) * 4 : 0);
    const int lane = threadIdx.x & 63;
    const unsigned m0 = lds_byte(to);
    if (lane < QT)
        asm volatile("s_nop 0\n\tbuffer_load_dword %0, %1, 0 offen lds" : : "v"(lane * 4), "s"(rs), "{m0}"(m0) : "memory");
}

// the partial sums behind rowsum(dy y), at a multiple of 16 bytes
__device__ __forceinline__ float *partials(const SlidingProblem &pr) {
    return pr.work + (((int64_t)pr.B * pr.Hk * pr.L * pr.G + 3) & ~(int64_t)3);
}

template <typename T, int DP>
__global__ __launch_bounds__(256, sizeof(T) == 4 && DP > 32 ? 1 : 2) void sliding_dkdv(SlidingProblem pr, WalkSplit sp) {
    typedef BwdShape<T, DP> Sh;
    typedef Tile<T, DP> Tl;
    constexpr int QT = Sh::QT, STEPS = DP / 16, OT = DP / 32;
    __shared__ char lds_mem[4 * Sh::TILE + 4 * QT * 4];
    const CIRCATT_LDS char *lds = (const CIRCATT_LDS char *)lds_mem;
    // workgroup numbers of one unit: far blocks part by part, then the others
    const int64_t id = (int64_t)(blockIdx.x & 7) * (gridDim.x >> 3) + (blockIdx.x >> 3);
    const int64_t unit = id / sp.units;
    if (unit >= (int64_t)pr.B * pr.Hk) return;
    const int in = (int)(id - unit * sp.units);
    const bool is_far = in < sp.far_units;
    const int parts = is_far ? sp.parts_far : sp.parts;
    const int kb = is_far ? in / parts : sp.far + (in - (int)sp.far_units) / parts;
    const int part = (is_far ? in : in - (int)sp.far_units) % parts;
    const int b = (int)(unit / pr.Hk), hk = (int)(unit - (int64_t)b * pr.Hk), n = uniform(signal_length(pr, b));
    const int lane = threadIdx.x & 63, wave = uniform(threadIdx.x >> 6);
    const Walk walk(pr, kb, n, QT);
    const int i0 = (int)((int64_t)walk.count * part / parts), i1 = (int)((int64_t)walk.count * (part + 1) / parts);
    const int j0 = kb * 128 + 32 * wave, j = j0 + (lane & 31), jj = j < n ? j : n - 1;
    const int rows = n * pr.G;
    const bool live = j0 < n;
    const T *kh = static_cast<const T *>(pr.k) + b * pr.k_batch + (int64_t)hk * pr.D;
    const T *vh = static_cast<const T *>(pr.v) + b * pr.v_batch + (int64_t)hk * pr.D;
    const T *qh = static_cast<const T *>(pr.q) + b * pr.q_batch + (int64_t)hk * pr.G * pr.D;
    const T *gh = static_cast<const T *>(pr.dy) + b * pr.dy_batch + (int64_t)hk * pr.G * pr.D;
    const int64_t stat = ((int64_t)b * pr.Hk + hk) * pr.L * pr.G;
    const float *lse = pr.lse + stat, *dsum = pr.work + stat;
    const Sight see{pr.W, pr.S};
    const float c = pr.scale * kLog2e;
    f16v dk[OT], dv[OT];
#pragma unroll
    for (int t = 0; t < OT; ++t) dk[t] = dv[t] = f16v{};
    if (i0 < i1) {
        const CIRCATT_LDS char *stats = lds + 4 * Sh::TILE;
        auto fetch = [&](int i) {
            const int r0 = walk.first + i * QT;
            const CIRCATT_LDS char *to = lds + (i & 1) * 2 * Sh::TILE;
            fetch_packed<T, DP, QT>(qh, pr.q_row, r0, pr.G, sp.heads, n, pr.D, to);
            fetch_packed<T, DP, QT>(gh, pr.dy_row, r0, pr.G, sp.heads, n, pr.D, to + Sh::TILE);
            if (wave == 0) fetch_stats<QT>(lse, r0, rows, stats + (i & 1) * QT * 8);
            if (wave == 1) fetch_stats<QT>(dsum, r0, rows, stats + (i & 1) * QT * 8 + QT * 4);
        };
        fetch(i0);
        V8<T> k[STEPS], v[STEPS];
#pragma unroll
        for (int s = 0; s < STEPS; ++s) {
            k[s] = load8(kh + jj * pr.k_row, 16 * s + 8 * (lane >> 5), pr.D);
            v[s] = load8(vh + jj * pr.v_row, 16 * s + 8 * (lane >> 5), pr.D);
        }
        const unsigned row_at = Tl::row_lane(lane), col_at = Tl::col_lane(lane);
        for (int i = i0; i < i1; ++i) {
            dma_barrier();
            if (i + 1 < i1) fetch(i + 1);
            if (!live) continue;
            for (int m = 0; m < QT; m += 32) {
                const int r0 = walk.first + i * QT + m;
                // tokens of the 32 rows
                const int t0 = uniform(fdiv(r0, sp.heads)), t1 = uniform(fdiv(r0 + 31, sp.heads));
                if (t0 >= n || j0 > t1 || (j0 + 31 <= t0 - pr.W && j0 >= pr.S)) continue;
                const unsigned to = lds_byte(lds) + (i & 1) * 2 * Sh::TILE + m * Tl::ROW;
                const unsigned qr = row_at + to, gr = qr + Sh::TILE, qc = col_at + to, gc = qc + Sh::TILE;
                const CIRCATT_LDS char *st = stats + (i & 1) * QT * 8 + (m + 4 * (lane >> 5)) * 4;
                f16v s = f16v{}, dp = f16v{};
#pragma unroll
                for (int x = 0; x < STEPS; ++x) {
                    s = mma(Tl::row(qr, 0, x), k[x], s);
                    dp = mma(Tl::row(gr, 0, x), v[x], dp);
                }
#pragma unroll
                for (int x = 0; x < 16; x += 4) {
                    const f4v ls = *(const CIRCATT_LDS f4v *)(st + 8 * x);
                    const f4v dd = *(const CIRCATT_LDS f4v *)(st + QT * 4 + 8 * x);
#pragma unroll
                    for (int y = 0; y < 4; ++y) {
                        s[x + y] = __builtin_amdgcn_exp2f(fmaf(s[x + y], c, -ls[y]));
                        dp[x + y] = s[x + y] * (dp[x + y] - dd[y]);
                    }
                }
                if (!(j0 + 31 <= t0 && (j0 > t1 - pr.W || j0 + 32 <= pr.S))) {
#pragma unroll
                    for (int x = 0; x < 16; ++x)
                        if (!see(fdiv(r0 + 8 * (x >> 2) + 4 * (lane >> 5) + (x & 3), sp.heads), j)) s[x] = dp[x] = 0.f;
                }
                V8<T> p[2], ds[2];
#pragma unroll
                for (int x = 0; x < 16; ++x) {
                    p[x >> 3][x & 7] = (T)s[x];
                    ds[x >> 3][x & 7] = (T)dp[x];
                }
#pragma unroll
                for (int t = 0; t < OT; ++t)
#pragma unroll
                    for (int h = 0; h < 2; ++h) {
                        dv[t] = mma(Tl::col(gc, 16 * h, t), p[h], dv[t]);
                        dk[t] = mma(Tl::col(qc, 16 * h, t), ds[h], dk[t]);
                    }
            }
        }
    }
    if (parts > 1) {
        const int64_t slot = is_far ? unit * sp.far_units + in
                                    : (sp.parts_far > 1 ? (int64_t)pr.B * pr.Hk * sp.far_units : 0) +
                                          unit * (sp.units - sp.far_units) + (in - sp.far_units);
        float *w = partials(pr) + slot * Sh::PART + (32 * wave + (lane & 31)) * DP;
#pragma unroll
        for (int t = 0; t < OT; ++t)
#pragma unroll
            for (int i = 0; i < 16; i += 4) {
                const int d = 32 * t + 2 * i + 4 * (lane >> 5);
                *reinterpret_cast<f4v *>(w + d) = f4v{dk[t][i], dk[t][i + 1], dk[t][i + 2], dk[t][i + 3]};
                *reinterpret_cast<f4v *>(w + 128 * DP + d) = f4v{dv[t][i], dv[t][i + 1], dv[t][i + 2], dv[t][i + 3]};
            }
        return;
    }
    const int64_t out = ((int64_t)b * pr.L + j) * pr.Hk * pr.D + (int64_t)hk * pr.D;
    T *kd = static_cast<T *>(pr.dk) + out, *vd = static_cast<T *>(pr.dv) + out;
    bool bad = false;
    if (j < n) {
        bad = store_channels(dk, kd, pr.D, lane, pr.scale);
        bad |= store_channels(dv, vd, pr.D, lane, 1.f);
    } else if (j < pr.L) {
        zero_channels(kd, pr.D, lane);
        zero_channels(vd, pr.D, lane);
    }
    uint64_t again = __ballot(bad);
    again = (again | again >> 32) & 0xffffffffu;
    for (; again; again &= again - 1) {
        const int x = j0 + __builtin_ctzll(again);
        const int64_t ox = ((int64_t)b * pr.L + x) * pr.Hk * pr.D + (int64_t)hk * pr.D;
        dkdv_row(kh + x * pr.k_row, vh + x * pr.v_row, qh, pr.q_row, gh, pr.dy_row, lse, dsum,
                 static_cast<T *>(pr.dk) + ox, static_cast<T *>(pr.dv) + ox, x, n, pr.W, pr.S, pr.G, pr.D, c, pr.scale);
    }
}

// The partial sums of split blocks, in the order of their parts: a wavefront a
// key.
template <typename T, int DP>
__global__ __launch_bounds__(256) void sliding_dkdv_join(SlidingProblem pr, WalkSplit sp) {
    constexpr int PART = BwdShape<T, DP>::PART;
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    const int first = sp.parts_far > 1 ? 0 : sp.far, last = sp.parts > 1 ? sp.blocks : sp.far;
    const int64_t id = (int64_t)blockIdx.x * 4 + wave, keys = (int64_t)(last - first) * 128;
    const int64_t unit = id / keys;
    if (unit >= (int64_t)pr.B * pr.Hk) return;
    const int j = first * 128 + (int)(id - unit * keys), kb = j >> 7;
    if (j >= pr.L) return;
    const bool is_far = kb < sp.far;
    const int parts = is_far ? sp.parts_far : sp.parts;
    const int64_t slot = is_far ? unit * sp.far_units + (int64_t)kb * parts
                                : (sp.parts_far > 1 ? (int64_t)pr.B * pr.Hk * sp.far_units : 0) +
                                      unit * (sp.units - sp.far_units) + (int64_t)(kb - sp.far) * parts;
    const float *w = partials(pr) + slot * PART + (j & 127) * DP;
    Pair k{0.f, 0.f}, v{0.f, 0.f};
    for (int i = 0; i < parts; ++i, w += PART) {
        const Pair a = load_row(w, lane, DP), c = load_row(w + 128 * DP, lane, DP);
        k.a += a.a;
        k.b += a.b;
        v.a += c.a;
        v.b += c.b;
    }
    const int b = (int)(unit / pr.Hk), hk = (int)(unit - (int64_t)b * pr.Hk), n = signal_length(pr, b);
    const int64_t head = (int64_t)hk * pr.D, out = ((int64_t)b * pr.L + j) * pr.Hk * pr.D + head;
    T *kd = static_cast<T *>(pr.dk) + out, *vd = static_cast<T *>(pr.dv) + out;
    k.a *= pr.scale;
    k.b *= pr.scale;
    store_row(kd, lane, pr.D, k);
    store_row(vd, lane, pr.D, v);
    // as in sliding_dkdv: not finite, or not in the type's range
    const float sum = fabsf((float)(T)k.a) + fabsf((float)(T)k.b) + fabsf((float)(T)v.a) + fabsf((float)(T)v.b);
    if (__any(!(sum < INFINITY)) && j < n) {
        const int64_t stat = ((int64_t)b * pr.Hk + hk) * pr.L * pr.G;
        dkdv_row(static_cast<const T *>(pr.k) + b * pr.k_batch + j * pr.k_row + head,
                 static_cast<const T *>(pr.v) + b * pr.v_batch + j * pr.v_row + head,
                 static_cast<const T *>(pr.q) + b * pr.q_batch + head * pr.G, pr.q_row,
                 static_cast<const T *>(pr.dy) + b * pr.dy_batch + head * pr.G, pr.dy_row, pr.lse + stat, pr.work + stat,
                 kd, vd, j, n, pr.W, pr.S, pr.G, pr.D, pr.scale * kLog2e, pr.scale);
    }
}

// Tiles of the longest walk of blocks kb0 .. (all of one kind).
int64_t walk_tiles(const SlidingProblem &pr, int64_t k0, bool far, int QT) {
    const int64_t tokens = far || pr.L - k0 < 128 + (int64_t)pr.W - 1 ? pr.L - k0 : 128 + (int64_t)pr.W - 1;
    return (tokens * pr.G + QT - 1) / QT;
}

// Parts of about 1/768 of all tiles, three rounds of the chip's 256 compute
// units, and not below 16 tiles: writing and adding up a partial pair takes as
// long as some 4 tiles.
WalkSplit walk_split(const SlidingProblem &pr) {
    const int QT = pr.dtype == CIRCATT_F32 ? 32 : 64;
    WalkSplit sp;
    sp.blocks = (pr.L + 127) / 128;
    sp.far = (pr.S + 127) / 128 < sp.blocks ? (pr.S + 127) / 128 : sp.blocks;
    int64_t all = 0;
    for (int kb = 0; kb < sp.blocks; ++kb) all += walk_tiles(pr, (int64_t)kb * 128, kb < sp.far, QT);
    all *= (int64_t)pr.B * pr.Hk;
    const int64_t part = all / 768 > 16 ? all / 768 : 16;
    auto parts = [&](int kb, bool far) { return (int)((walk_tiles(pr, (int64_t)kb * 128, far, QT) + part - 1) / part); };
    sp.parts_far = sp.far > 0 ? parts(0, true) : 1;
    sp.parts = sp.far < sp.blocks ? parts(sp.far, false) : 1;
    sp.heads = make_fastdiv(pr.G);
    sp.far_units = (int64_t)sp.far * sp.parts_far;
    sp.units = sp.far_units + (int64_t)(sp.blocks - sp.far) * sp.parts;
    return sp;
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
template <typename T, int DP>
hipError_t backward(const SlidingProblem &pr, hipStream_t s) {
    const int blocks = (pr.L * pr.G + 127) / 128;
    sliding_dq<T, DP><<<grid8((int64_t)pr.B * pr.Hk * blocks), 256, 0, s>>>(pr, blocks);
    if (pr.dk != nullptr) {
        const WalkSplit sp = walk_split(pr);
        sliding_dkdv<T, DP><<<grid8((int64_t)pr.B * pr.Hk * sp.units), 256, 0, s>>>(pr, sp);
        const int64_t split = (sp.parts_far > 1 ? sp.far : 0) + (sp.parts > 1 ? sp.blocks - sp.far : 0);
        if (split > 0) sliding_dkdv_join<T, DP><<<(unsigned)(pr.B * pr.Hk * split * 32), 256, 0, s>>>(pr, sp);
    }
    return hipGetLastError();
}
template <int DT>
hipError_t backward(const SlidingProblem &pr, hipStream_t s) {
    typedef typename Elem<DT>::T T;
    return pr.D <= 32 ? backward<T, 32>(pr, s)
                      : pr.D <= 64 ? backward<T, 64>(pr, s) : pr.D <= 96 ? backward<T, 96>(pr, s) : backward<T, 128>(pr, s);
}

}  // namespace

int64_t sliding_bwd_workspace_floats(const SlidingProblem &pr) {
    const WalkSplit sp = walk_split(pr);
    const int64_t slots = (sp.parts_far > 1 ? sp.far_units : 0) + (sp.parts > 1 ? sp.units - sp.far_units : 0);
    const int DP = (pr.D + 31) / 32 * 32;
    // the partial sums start at a multiple of 16 bytes
    return (int64_t)pr.B * pr.Hk * pr.L * pr.G + 4 + pr.B * (int64_t)pr.Hk * slots * 128 * DP * 2;
}

hipError_t launch_sliding_fwd(const SlidingProblem &pr, hipStream_t s) {
    return pr.dtype == CIRCATT_F32 ? forward<0>(pr, s) : pr.dtype == CIRCATT_F16 ? forward<2>(pr, s) : forward<3>(pr, s);
}
hipError_t launch_sliding_bwd(const SlidingProblem &pr, hipStream_t s) {
    return pr.dtype == CIRCATT_F32 ? backward<0>(pr, s)
                                   : pr.dtype == CIRCATT_F16 ? backward<2>(pr, s) : backward<3>(pr, s);
}

}  // namespace circatt
