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
// their window: 32 rows a wavefront, tiles of 64 keys (Float32: 32) and values in
// LDS (Ring).  Workgroups that share a head of keys run on one XCD (ids 8 apart),
// whose L2 then holds their common tiles.
//
// Bound by the products and the softmax between them, and by the blocks' starts and
// ends: a wavefront's tile is 32 products of 32 cycles and, by the counters, some 270
// other vector instructions with starts and edges, 32 of them exponentials of 8
// cycles.  8192 tokens, 32 heads of 128 over 8, window 1024, 4 sinks, bf16: 167 to 170
// us, 770 TFLOP/s of the pairs that are seen (870 of those formed: edges of tiles); the
// same without a window 540 us, 1020 TFLOP/s, where a large library product of this
// card reaches 1190.  From windows of 128 (4 tiles a block, 76 us) to none (64 tiles)
// the time is 45 us and 7.7 for a tile in every block: the 45, some 6 tiles' time, are
// the cold start and the end of 2048 blocks in four rounds, a quarter of the time at
// window 1024.  Copies of the kernel without its DMA, or with operands from registers
// instead of LDS, take 21 and 32 us less (both: 53).  Two rounds in one run (the next
// tile's scores among this one's exponentials) take 166 us where one after another took
// 175; explicit orders of the run's instructions, wavefront priorities, operands read
// earlier and tiles of 32 keys in five places changed nothing or lost (177 us).  For
// training it also stores what y's rounding took: 2 x 4096 tokens, 16 heads of 128, 63
// us without, 73 with.
//
// Backward, queries: the same blocks with tiles in two buffers.
template <typename T, int DP>
struct DqShape {
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
int64_t grid8(int64_t n) { return (n + 7) / 8 * 8; }

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

template <typename T>
__device__ __forceinline__ SignalKV<T> signal_rows(const SlidingProblem &pr, int b, int hk) {
    return SignalKV<T>{static_cast<const T *>(pr.k) + b * pr.k_batch + (int64_t)hk * pr.D,
                       static_cast<const T *>(pr.v) + b * pr.v_batch + (int64_t)hk * pr.D, pr.k_row, pr.v_row};
}

template <typename T, int DP>
__global__ __launch_bounds__(256, sizeof(T) == 4 && DP > 64 ? 1 : 2) void sliding_fwd(SlidingProblem pr, int blocks) {
    typedef Ring<T, DP> Rg;
    constexpr int KT = Rg::KT, NB = Rg::NB;
    __shared__ __attribute__((aligned(1024))) char lds_mem[Rg::BYTES];
    const CIRCATT_LDS char *lds = (const CIRCATT_LDS char *)lds_mem;
    const BlockOrder w(pr.B * pr.Hk, blocks);
    if (w.unit < 0) return;
    const int b = w.unit / pr.Hk, hk = w.unit - b * pr.Hk, n = uniform(signal_length(pr, b));
    const int lane = threadIdx.x & 63, wave = uniform(threadIdx.x >> 6);
    const int rows = n * pr.G, r0 = w.block * 128, all_rows = pr.L * pr.G;
    const int r = r0 + 32 * wave + (lane & 31);
    T *y = static_cast<T *>(pr.y) + (int64_t)b * pr.L * pr.H * pr.D + (int64_t)hk * pr.G * pr.D;
    T *rest = pr.y_rest == nullptr ? nullptr : static_cast<T *>(pr.y_rest) + (y - static_cast<T *>(pr.y));
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
                asm volatile("");
#pragma unroll
                for (int m = 0; m < NB; ++m) hide_keys(s[m], see.bits(at, k0 + 32 * m), lane);
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
        f16v sa[NB], sb[NB];
        int i = -1;
        for (; i < (live ? first - 1 : count); ++i, next()) round(i);
        if (live) {
            round(i);
            x.scores(row_at + kp * Rg::TILE, sa);
            look(sa, first);
            next();
            ++i;
            for (; i + 1 < end; i += 2) {
                step(sa, sb, i);
                step(sb, sa, i + 1);
            }
            if (i < end) {
                step(sa, sb, i);
#pragma unroll
                for (int m = 0; m < NB; ++m) sa[m] = sb[m];
                ++i;
            }
            round(i);
            V8<T> p[2 * NB];
            x.raise(mx);
            x.weigh(sa, p, c);
            x.template add<NB>(col_at + vp * Rg::TILE, p);
            next();
            for (++i; i < count; ++i, next()) round(i);
        }
        uint32_t again = 0;
        if (live) {
            // a row sees its own token at least: without a sum of weights all that it sees
            // has the score -inf, and its softmax is NaN
            const float l = x.total(), inv = 1.f / l;
            bool bad = false;
            if (r < rows) {
                bad = store_channels(x.o, y + ((int64_t)at * pr.H + g) * pr.D, pr.D, lane, inv);
                if (rest != nullptr) store_rests(x.o, rest + ((int64_t)at * pr.H + g) * pr.D, pr.D, lane, inv);
                if (pr.lse != nullptr && lane < 32) pr.lse[stat + r] = x.m + __builtin_amdgcn_logf(l);
            }
            // A value that is not finite reaches, as 0 times itself, every row of
            // a wavefront whose tile holds it: where such a value is among the keys
            // that the tiles hide from some row (before the rows' windows, behind the
            // first row, and behind the sinks), rows that are not finite are formed
            // again from the keys that they see alone.  (Not where the sum of the
            // weights is NaN or 0: then the row is, whatever it sees.)
            again = rows_of(__ballot(bad && l > 0.f));
            if (again != 0) {
                const SlidingProblem pe = argument_again<SlidingProblem>();
                const SignalKV<T> kv = signal_rows<T>(pe, b, hk);
                auto tile_end = [&](int j) { return (int)((int64_t)j + KT - j % KT < n ? j + KT - j % KT : n); };
                const int window = r0 / pe.G - pe.W + 1;
                if (!bad_values(kv, window > 0 ? window / KT * KT : 0, hi - pe.W + 1, pe.D) &&
                    !bad_values(kv, lo + 1, tile_end(hi), pe.D) &&
                    !(pe.S % KT != 0 && bad_values(kv, pe.S, tile_end(pe.S), pe.D)))
                    again = 0;
            }
        }
        // (The list lies in a K tile: the last round, whose barrier is behind all, reads
        // none.)
        share_repairs<4, false>((CIRCATT_LDS uint32_t *)lds, wave, wave, again, 0, [&](int i, bool, bool) {
            const SlidingProblem pe = argument_again<SlidingProblem>();
            const int aj = (r0 + i) / pe.G, h = hk * pe.G + r0 + i - aj * pe.G;
            const int64_t out = (((int64_t)b * pe.L + aj) * pe.H + h) * pe.D;
            forward_row(static_cast<const T *>(pe.q) + b * pe.q_batch + aj * pe.q_row + (int64_t)h * pe.D,
                        static_cast<T *>(pe.y) + out, pe.y_rest == nullptr ? nullptr : static_cast<T *>(pe.y_rest) + out,
                        signal_rows<T>(pe, b, hk), aj, pe.W, pe.S, pe.D, pe.scale * kLog2e);
        });
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
// operand, and dQ' += K' dS' with K' by the transposing reads.  dS is rounded to
// the element type there, as P is in the forward.  d = <dy, y> takes y with what
// its rounding took (y_rest): where few keys carry a row, the score gradients
// cancel most, and with the rounded y alone the error of dq was up to 3 times that
// of a form that rounds only its results, now 1.6.  2 x 4096 tokens, 16 heads of 128
// over 4, window 512, bf16: 88 us, 550 TFLOP/s of the pairs that are seen.
template <typename T, int DP>
__global__ __launch_bounds__(256, sizeof(T) == 4 && DP > 32 ? 1 : 2) void sliding_dq(SlidingProblem pr, int blocks) {
    typedef DqShape<T, DP> Sh;
    typedef Tile<T, DP> Tl;
    constexpr int KT = Sh::KT, STEPS = DP / 16, OT = DP / 32;
    __shared__ __attribute__((aligned(1024))) char lds_mem[4 * Sh::TILE];
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
        const T *eh = pr.y_rest == nullptr ? nullptr : static_cast<const T *>(pr.y_rest) + head;
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
            const V8<T> e = eh == nullptr ? V8<T>{} : load8(eh + out, ch, pr.D);
#pragma unroll
            for (int j = 0; j < 8; ++j) d = fmaf((float)y[j] + (float)e[j], (float)dy[k][j], d);
        }
        d += __shfl_xor(d, 32, 64);
        const float lse = pr.lse[stat + rr];
        float rest = 0.f;
#pragma unroll
        for (int t = 0; t < OT; ++t) o[t] = f16v{};
        const unsigned row_at = Tl::row_lane(lane), col_at = Tl::col_lane(lane);
        loads_here();
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
                products<T, 2 * STEPS, 4>([&](int i) { return Tl::row(i & 1 ? vr : kr, 0, i >> 1); },
                                          [&](int i, V8<T> a) {
                                              if (i & 1) dp = mma(a, dy[i >> 1], dp);
                                              else s = mma(a, q[i >> 1], s);
                                          });
#pragma unroll
                for (int x = 0; x < 16; ++x) s[x] = __builtin_amdgcn_exp2f(fmaf(s[x], c, -lse)) * (dp[x] - d);
                if (!see.all(lo, hi, k0, 32)) {
                    asm volatile("");  // a branch: few tiles need it
                    const uint32_t half = see.bits(at, k0) >> (4 * (lane >> 5));
#pragma unroll
                    for (int x = 0; x < 16; ++x)
                        if (!(half & place_bit(x))) s[x] = 0.f;
                }
                V8<T> ds[2];
#pragma unroll
                for (int x = 0; x < 16; ++x) {
                    rest += s[x];
                    ds[x >> 3][x & 7] = (T)s[x];
                }
                products<T, 2 * OT, 4>([&](int i) { return Tl::col(kc, 16 * (i & 1), i >> 1); },
                                       [&](int i, V8<T> a) { o[i >> 1] = mma(a, ds[i & 1], o[i >> 1]); });
            }
        }
        // <dy, y> of the exact y is sum_j p_j <dy, v_j>: d and what the score gradients,
        // whose sum is zero, left of it (P's rounding in y)
        rest += other_half(rest);
        if (r < rows && lane < 32) pr.work[stat + r] = d + rest;
        if (live) {
            // formed again as in the forward, and where Float16 could not hold a score
            // gradient; a row whose statistics are not finite is not, whatever it sees
            const bool bad = r < rows && store_channels(o, dq + out, pr.D, lane, pr.scale);
            uint32_t again = rows_of(__ballot(bad && is_finite(lse) && is_finite(d)));
            const SignalKV<T> kv{kh, vh, pr.k_row, pr.v_row};
            if (again != 0) __threadfence_block();  // other lanes' stores
            for (; again; again &= again - 1) {
                const int j = __builtin_ctz(again);
                const int aj = __builtin_amdgcn_readlane(at, j), gj = __builtin_amdgcn_readlane(g, j);
                const int64_t oj = ((int64_t)aj * pr.H + gj) * pr.D, sj = stat + (int64_t)aj * pr.G + gj;
                dq_row(qh + aj * pr.q_row + (int64_t)gj * pr.D, yh + oj, eh == nullptr ? eh : eh + oj,
                       gh + aj * pr.dy_row + (int64_t)gj * pr.D, dq + oj, pr.lse[sj], pr.work + sj, kv, aj, pr.W, pr.S, pr.D,
                       c, pr.scale);
            }
        }
    }
    if (r >= rows && r < all_rows) {
        const int t = r / pr.G;
        zero_channels(dq + ((int64_t)t * pr.H + r - t * pr.G) * pr.D, pr.D, lane);
    }
}

// ---------------------------------------------------------------------------
// Backward, keys: a wavefront keeps k and v of 32 keys as second operands and
// walks the query rows that see them, 32 at a time: S = Q K', dP = dY V' (lane:
// one key; registers: query rows), P and dS = P (dP - d) as second operands of
// dV' += dY' P and dK' += Q' dS with dY' and Q' by the transposing reads.
//
// A workgroup has 128 keys of one head and NG groups of four wavefronts, which
// take turns at tiles of QT rows of q and dy in LDS (two buffers each) and add up
// at the end: one workgroup fills a compute unit's registers, and a block of keys
// needs no second workgroup for it.  Where blocks are still few, their walks are
// split over `parts` workgroups, whose Float32 sums sliding_dkdv_join adds up in
// order.  At the size above 109 us, 600 TFLOP/s; the operands and sums of 32 keys
// take 192 of a lane's 256 registers, and what is left bounds how far ahead
// operands can be read.  An earlier form, workgroups of one group whose walks were
// split in three for a full chip, took 187 us and 23 more to add up; barriers of a group
// alone, by a count in LDS, changed nothing.
//
// The rows that see a sink from behind its block's window are another walk,
// sliding_dkdv_far's, for 32 keys and with a wavefront for every tile: a few
// sinks would leave most of a workgroup of 128 keys idle (18 us at the size above).
template <typename T, int DP>
struct BwdShape {
    static constexpr int QT = sizeof(T) == 2 ? 64 : 32;
    static constexpr int TILE = QT * Tile<T, DP>::ROW;
    // Float32 operands and sums of wide heads take more than half the registers
    static constexpr int NG = sizeof(T) == 2 || DP <= 32 ? 2 : 1;
    static constexpr int PART = 128 * DP * 2;  // floats of one pair of partial sums
    static constexpr int FAR_PART = 32 * DP * 2;
    static constexpr int FAR_TILE = 32 * Tile<T, DP>::ROW;
};

struct WalkSplit {
    int blocks, parts;   // of 128 keys; workgroups a block
    int far, far_parts;  // groups of 32 sinks that rows behind their window see; workgroups each
    FastDiv heads;       // G
    int64_t far_at, part_at;  // floats before the far sums and the parts' in the workspace
};

// Tokens [begin, end) behind the window of the block of keys that key k0 is in.
struct FarRows {
    int first, count;  // packed query rows, and those behind them
    __device__ FarRows(const SlidingProblem &pr, int k0, int n) {
        const int last = k0 / 128 * 128 + 127;
        const int begin = n - pr.W > last ? last + pr.W : n;
        first = begin * pr.G;
        count = (n - begin) * pr.G;
    }
};

// Packed query rows [r0, r0 + ROWS) of a head group by THREADS threads, this one
// the tid-th: row r is head r % G of token r / G; rows behind token n - 1 are zeros.
template <typename T, int DP, int ROWS, int THREADS>
__device__ __forceinline__ void fetch_packed(const T *p, int64_t row, int r0, int G, FastDiv dg, int n, int D, int tid,
                                             unsigned to) {
    typedef Tile<T, DP> Tl;
    const int rb = (int)(row * (int)sizeof(T)), hb = D * (int)sizeof(T);
    const int t0 = uniform(fdiv(r0, dg));
    const int64_t bytes = n > t0 ? (int64_t)(n - 1 - t0) * rb + G * hb : 0;
    const dma::i4v rs = dma::dma_rsrc(reinterpret_cast<const float *>(p + t0 * row),
                                      (int)(bytes < dma::kMaxBytes ? bytes : dma::kMaxBytes));
    const unsigned m0 = to + uniform(tid >> 6) * 1024;
#pragma unroll
    for (int k = 0; k < ROWS * Tl::PC / THREADS; ++k) {
        const int slot = tid + k * THREADS, rl = slot / Tl::PC, u = ((slot % Tl::PC) ^ Tl::f(rl)) * 16;
        const int t = fdiv(r0 + rl, dg), g = r0 + rl - t * G;
        // units from D on stay out of the buffer whatever is added
        const unsigned off = (unsigned)((t - t0) * rb + g * hb) + (unsigned)(u < hb ? u : dma::kOut);
        dma::dma16(rs, m0 + k * THREADS * 16, (int)off, 0);
    }
}
// COUNT floats from p + r0 on into LDS by the calling wavefront, zeros behind p[rows - 1]
template <int COUNT>
__device__ __forceinline__ void fetch_stats(const float *p, int r0, int rows, unsigned to) {
    const dma::i4v rs = dma::dma_rsrc(p + r0, rows > r0 ? (rows - r0 < COUNT ? rows - r0 : COUNT) * 4 : 0);
    const int lane = threadIdx.x & 63;
    if (lane < COUNT)
        asm volatile(CIRCATT_SCALARS_READY "buffer_load_dword %0, %1, 0 offen lds"
                     :
                     : "v"(lane * 4), "s"(rs), "{m0}"(to)
                     : "memory");
}

// One wavefront's 32 keys: operands, sums, and 32 query rows' share of them.
template <typename T, int DP>
struct KeySums {
    typedef Tile<T, DP> Tl;
    static constexpr int STEPS = DP / 16, OT = DP / 32, AHEAD = 4;
    V8<T> k[STEPS], v[STEPS];
    f16v dk[OT], dv[OT];

    __device__ __forceinline__ void start(const T *kr, const T *vr, int D, int lane) {
#pragma unroll
        for (int s = 0; s < STEPS; ++s) {
            k[s] = load8(kr, 16 * s + 8 * (lane >> 5), D);
            v[s] = load8(vr, 16 * s + 8 * (lane >> 5), D);
        }
        clear();
        loads_here();
    }
    __device__ __forceinline__ void clear() {
#pragma unroll
        for (int t = 0; t < OT; ++t) dk[t] = dv[t] = f16v{};
    }
    // rows of q and dy at the lane's places qr, gr (row), then qc, gc (col); lse and d
    // of the rows at LDS bytes st and st + stride; half: the rows that see the key, a
    // bit each, unless every one does
    struct Weights {
        V8<T> p[2], ds[2];
    };
    __device__ __forceinline__ void weigh(unsigned qr, unsigned gr, unsigned st, int stride, bool every, uint32_t half,
                                          float c, Weights &w) const {
        f16v s = f16v{}, dp = f16v{};
        products<T, 2 * STEPS, AHEAD - 1>([&](int i) { return Tl::row(i & 1 ? gr : qr, 0, i >> 1); },
                                      [&](int i, V8<T> a) {
                                          if (i & 1) dp = mma(a, v[i >> 1], dp);
                                          else s = mma(a, k[i >> 1], s);
                                      });
#pragma unroll
        for (int x = 0; x < 16; x += 4) {
            const f4v ls = *(const CIRCATT_LDS f4v *)(st + 8 * x);
            const f4v dd = *(const CIRCATT_LDS f4v *)(st + stride + 8 * x);
#pragma unroll
            for (int y = 0; y < 4; ++y) {
                s[x + y] = __builtin_amdgcn_exp2f(fmaf(s[x + y], c, -ls[y]));
                dp[x + y] = s[x + y] * (dp[x + y] - dd[y]);
            }
        }
        if (!every) {
            asm volatile("");  // a branch: few rows need it
#pragma unroll
            for (int x = 0; x < 16; ++x)
                if (!(half & place_bit(x))) s[x] = dp[x] = 0.f;
        }
#pragma unroll
        for (int x = 0; x < 16; ++x) {
            w.p[x >> 3][x & 7] = (T)s[x];
            w.ds[x >> 3][x & 7] = (T)dp[x];
        }
    }
    __device__ __forceinline__ void add(unsigned qc, unsigned gc, const Weights &w) {
        products<T, 4 * OT, AHEAD>([&](int i) { return Tl::col(i & 1 ? qc : gc, 16 * ((i >> 1) & 1), i >> 2); },
                                   [&](int i, V8<T> a) {
                                       if (i & 1) dk[i >> 2] = mma(a, w.ds[(i >> 1) & 1], dk[i >> 2]);
                                       else dv[i >> 2] = mma(a, w.p[(i >> 1) & 1], dv[i >> 2]);
                                   });
    }
    // through LDS or a workspace, one float for every register and lane
    template <typename P>
    __device__ __forceinline__ void put(P to, int lane) const {
#pragma unroll
        for (int t = 0; t < OT; ++t)
#pragma unroll
            for (int i = 0; i < 16; ++i) {
                to[(16 * t + i) * 64 + lane] = dk[t][i];
                to[(16 * (OT + t) + i) * 64 + lane] = dv[t][i];
            }
    }
    __device__ __forceinline__ void take(const CIRCATT_LDS float *from, int lane) {
#pragma unroll
        for (int t = 0; t < OT; ++t)
#pragma unroll
            for (int i = 0; i < 16; ++i) {
                dk[t][i] += from[(16 * t + i) * 64 + lane];
                dv[t][i] += from[(16 * (OT + t) + i) * 64 + lane];
            }
    }
    // Float32 sums to a workspace: the lane's key's channels, dv `apart` floats
    // behind dk
    __device__ __forceinline__ void write(float *w, int apart, int lane) const {
#pragma unroll
        for (int t = 0; t < OT; ++t)
#pragma unroll
            for (int i = 0; i < 16; i += 4) {
                const int d = 32 * t + 2 * i + 4 * (lane >> 5);
                *reinterpret_cast<f4v *>(w + d) = f4v{dk[t][i], dk[t][i + 1], dk[t][i + 2], dk[t][i + 3]};
                *reinterpret_cast<f4v *>(w + apart + d) = f4v{dv[t][i], dv[t][i + 1], dv[t][i + 2], dv[t][i + 3]};
            }
    }
};

// A head of keys and its group of queries' heads.
template <typename T>
struct HeadGroup {
    int b, hk, n, rows;
    const T *k, *v, *q, *dy;
    const float *lse, *dsum;
    __device__ HeadGroup(const SlidingProblem &pr, int64_t unit)
        : HeadGroup(pr, unit, uniform(signal_length(pr, (int)(unit / pr.Hk)))) {}
    __device__ HeadGroup(const SlidingProblem &pr, int64_t unit, int length) {
        b = (int)(unit / pr.Hk);
        hk = (int)(unit - (int64_t)b * pr.Hk);
        n = length;
        rows = n * pr.G;
        const int64_t head = (int64_t)hk * pr.D;
        k = static_cast<const T *>(pr.k) + b * pr.k_batch + head;
        v = static_cast<const T *>(pr.v) + b * pr.v_batch + head;
        q = static_cast<const T *>(pr.q) + b * pr.q_batch + head * pr.G;
        dy = static_cast<const T *>(pr.dy) + b * pr.dy_batch + head * pr.G;
        const int64_t stat = unit * pr.L * pr.G;
        lse = pr.lse + stat;
        dsum = pr.work + stat;
    }
    // whether the statistics of one of the packed rows [r0, r1) are not finite
    __device__ bool bad_rows(int r0, int r1) const {
        bool bad = false;
#pragma unroll 4
        for (int r = r0 + lane_again(); r < r1; r += 64) bad |= !is_finite(lse[r]) || !is_finite(dsum[r]);
        return __any(bad);
    }
    // The gradients of key j, one of the 32 from j0 on, of which dk (bad_k) or dv
    // (bad_v) are not finite.  A row whose statistics are not finite makes all of
    // dk that of every key that it sees, and a row of dy that is not finite has such
    // statistics.  So dk is formed again if no row that sees the key is one, and
    // dv if a row that the products hid from the key is one: zero times its dy is
    // NaN.  Those lie before the key, behind its window in the last block of 32 rows,
    // and, of a group with the last sinks, anywhere behind.
    __device__ void again(const SlidingProblem &pr, int j, int j0, bool bad_k, bool bad_v) const {
        const int end = j < pr.S || n - j < pr.W ? n : j + pr.W;
        const int64_t last = (int64_t)j0 + 31 + pr.W + (30 + pr.G) / pr.G;
        const bool fix_k = bad_k && !bad_rows(j * pr.G, end * pr.G);
        const bool fix_v = bad_v && (bad_rows(j0 * pr.G, j * pr.G) ||
                                     bad_rows(end * pr.G, (j0 < pr.S || last > n ? n : (int)last) * pr.G));
        if (!fix_k && !fix_v) return;
        const int64_t out = ((int64_t)b * pr.L + j) * pr.Hk * pr.D + (int64_t)hk * pr.D;
        dkdv_row(k + j * pr.k_row, v + j * pr.v_row, q, pr.q_row, dy, pr.dy_row, lse, dsum, static_cast<T *>(pr.dk) + out,
                 static_cast<T *>(pr.dv) + out, fix_k, fix_v, j, n, pr.W, pr.S, pr.G, pr.D, pr.scale * kLog2e, pr.scale);
    }
};

template <typename T, int DP>
__global__ __launch_bounds__(256, sizeof(T) == 4 && DP > 32 ? 1 : 2) void sliding_dkdv_far(SlidingProblem pr, WalkSplit sp) {
    typedef BwdShape<T, DP> Sh;
    typedef Tile<T, DP> Tl;
    // two buffers for each wavefront, but for tiles that are too long for that
    constexpr int BUFS = 16 * Sh::FAR_TILE <= 128 * 1024 ? 2 : 1, STATS = 8 * BUFS * Sh::FAR_TILE;
    constexpr int SUMS = 32 * DP * 2 * 4;
    __shared__ __attribute__((aligned(1024))) char lds_mem[STATS + BUFS * 1024 > SUMS ? STATS + BUFS * 1024 : SUMS];
    const int64_t unit = blockIdx.x / (sp.far * sp.far_parts);
    const int in = (int)(blockIdx.x - unit * (sp.far * sp.far_parts)), k0 = in / sp.far_parts * 32, part = in % sp.far_parts;
    const HeadGroup<T> hg(pr, unit);
    const int lane = threadIdx.x & 63, wave = uniform(threadIdx.x >> 6), j = k0 + (lane & 31);
    const unsigned lds = lds_byte((const CIRCATT_LDS char *)lds_mem) + wave * (2 * BUFS * Sh::FAR_TILE);
    const unsigned st = lds_byte((const CIRCATT_LDS char *)lds_mem) + STATS + wave * BUFS * 256;
    KeySums<T, DP> x;
    // a block of keys in which none is seen from behind its window adds nothing
    const FarRows far(pr, k0, hg.n);
    const int tiles = (far.count + 31) / 32, parts = 4 * sp.far_parts, w = 4 * part + wave;
    const int i0 = (int)((int64_t)tiles * w / parts), i1 = (int)((int64_t)tiles * (w + 1) / parts);
    if (i0 < i1) {
        const int jj = j < hg.n ? j : hg.n - 1;
        x.start(hg.k + jj * pr.k_row, hg.v + jj * pr.v_row, pr.D, lane);
        const unsigned row_at = Tl::row_lane(lane) + lds, col_at = Tl::col_lane(lane) + lds;
        auto fetch = [&](int i) {
            const int r0 = far.first + 32 * i, y = BUFS == 2 ? i & 1 : 0;
            const unsigned to = lds + y * 2 * Sh::FAR_TILE;
            fetch_packed<T, DP, 32, 64>(hg.q, pr.q_row, r0, pr.G, sp.heads, hg.n, pr.D, lane, to);
            fetch_packed<T, DP, 32, 64>(hg.dy, pr.dy_row, r0, pr.G, sp.heads, hg.n, pr.D, lane, to + Sh::FAR_TILE);
            fetch_stats<32>(hg.lse, r0, hg.rows, st + y * 256);
            fetch_stats<32>(hg.dsum, r0, hg.rows, st + y * 256 + 128);
        };
        if (BUFS == 2) fetch(i0);
        for (int i = i0; i < i1; ++i) {
            const int y = BUFS == 2 ? i & 1 : 0;
            dma_wait();  // the tile's DMA, and the reads of the one before
            if (BUFS == 1) {
                fetch(i);
                dma_wait();
            } else if (i + 1 < i1) {
                fetch(i + 1);
            }
            const unsigned to = y * 2 * Sh::FAR_TILE;
            typename KeySums<T, DP>::Weights wt;
            x.weigh(row_at + to, row_at + to + Sh::FAR_TILE, st + y * 256 + 16 * (lane >> 5), 128, k0 + 32 <= pr.S,
                    j < pr.S ? ~0u : 0u, pr.scale * kLog2e, wt);
            x.add(col_at + to, col_at + to + Sh::FAR_TILE, wt);
        }
    } else {
        x.clear();
    }
    // one after another into the first wavefront's
    CIRCATT_LDS float *buf = (CIRCATT_LDS float *)lds_mem;
    for (int y = 1; y < 4; ++y) {
        __syncthreads();
        if (wave == y) x.put(buf, lane);
        __syncthreads();
        if (wave == 0) x.take(buf, lane);
    }
    if (wave == 0) x.put(pr.work + sp.far_at + (int64_t)blockIdx.x * Sh::FAR_PART, lane);
}

// The far sums of `groups` groups of 32 keys from w on, added up in the order of
// their parts into LDS as they lie in memory, by all of THREADS threads.
template <typename T, int DP, int THREADS>
__device__ __forceinline__ void sum_far(const float *w, int groups, int parts, CIRCATT_LDS float *buf) {
    constexpr int SIZE = BwdShape<T, DP>::FAR_PART;
    for (int e = 4 * threadIdx.x; e < groups * SIZE; e += 4 * THREADS) {
        const float *we = w + (int64_t)(e / SIZE) * parts * SIZE + e % SIZE;
        f4v sum = f4v{};
#pragma unroll 8
        for (int y = 0; y < parts; ++y) sum += *reinterpret_cast<const f4v *>(we + (int64_t)y * SIZE);
        *(CIRCATT_LDS f4v *)(buf + e) = sum;
    }
}

template <typename T, int DP>
__global__ __launch_bounds__((256 * BwdShape<T, DP>::NG), (sizeof(T) == 2 && DP <= 64 ? 2 : 1))
void sliding_dkdv(SlidingProblem pr, WalkSplit sp) {
    typedef BwdShape<T, DP> Sh;
    typedef Tile<T, DP> Tl;
    constexpr int QT = Sh::QT, NG = Sh::NG;
    __shared__ __attribute__((aligned(1024))) char lds_mem[NG * (4 * Sh::TILE + 16 * QT)];
    // workgroups of one unit: its blocks, part by part, on one XCD
    const int64_t id = (int64_t)(blockIdx.x & 7) * (gridDim.x >> 3) + (blockIdx.x >> 3);
    const int64_t unit = id / (sp.blocks * sp.parts);
    if (unit >= (int64_t)pr.B * pr.Hk) return;
    const int in = (int)(id - unit * (sp.blocks * sp.parts)), kb = in / sp.parts, part = in - kb * sp.parts;
    const HeadGroup<T> hg(pr, unit);
    const int n = hg.n, lane = threadIdx.x & 63, wave = uniform(threadIdx.x >> 6) & 3, group = uniform(threadIdx.x >> 8);
    const int tid = threadIdx.x & 255;
    // packed query rows of the walk: the block's tokens and W - 1 behind
    const int k0 = kb * 128, kn = k0 + 127 < n - 1 ? k0 + 127 : n - 1, end = n - kn > pr.W ? kn + pr.W : n;
    const int tiles = k0 < n ? ((end - k0) * pr.G + QT - 1) / QT : 0;
    const int i0 = (int)((int64_t)tiles * part / sp.parts), i1 = (int)((int64_t)tiles * (part + 1) / sp.parts);
    const int j0 = k0 + 32 * wave, j = j0 + (lane & 31), jj = j < n ? j : n - 1;
    const unsigned lds = lds_byte((const CIRCATT_LDS char *)lds_mem) + group * 4 * Sh::TILE;
    const unsigned stats = lds_byte((const CIRCATT_LDS char *)lds_mem) + NG * 4 * Sh::TILE + group * 16 * QT;
    const float c = pr.scale * kLog2e;
    KeySums<T, DP> x;
    if (i0 < i1) {
        // a group's turn i: tile i0 + NG i + group
        const int mine = (i1 - i0 - group + NG - 1) / NG, turns = (i1 - i0 + NG - 1) / NG;
        auto first_row = [&](int i) { return k0 * pr.G + (i0 + NG * i + group) * QT; };
        auto fetch = [&](int i) {
            const int r0 = first_row(i);
            const unsigned to = lds + (i & 1) * 2 * Sh::TILE, st = stats + (i & 1) * 8 * QT;
            fetch_packed<T, DP, QT, 256>(hg.q, pr.q_row, r0, pr.G, sp.heads, n, pr.D, tid, to);
            fetch_packed<T, DP, QT, 256>(hg.dy, pr.dy_row, r0, pr.G, sp.heads, n, pr.D, tid, to + Sh::TILE);
            if (wave == 0) fetch_stats<QT>(hg.lse, r0, hg.rows, st);
            if (wave == 1) fetch_stats<QT>(hg.dsum, r0, hg.rows, st + 4 * QT);
        };
        if (mine > 0) fetch(0);
        x.start(hg.k + jj * pr.k_row, hg.v + jj * pr.v_row, pr.D, lane);
        const unsigned row_at = Tl::row_lane(lane) + lds, col_at = Tl::col_lane(lane) + lds;
        // the rows that see key j: from its token on, to its window's end or, of a sink,
        // the walk's (rows behind it in the last tile belong to sliding_dkdv_far)
        const int see0 = j * pr.G, see1 = j < pr.S || end - j < pr.W ? end * pr.G : (j + pr.W) * pr.G;
        // and those that see all of the wavefront's keys, or any
        const int all0 = (j0 + 31) * pr.G, all1 = j0 + 31 < pr.S || end - j0 < pr.W ? end * pr.G : (j0 + pr.W) * pr.G;
        const int any1 = j0 < pr.S || end - (j0 + 31) < pr.W ? end * pr.G : (j0 + 31 + pr.W) * pr.G;
        // (Groups half a block apart, one forming weights while the other adds, took 167
        // us where this takes 112: the weights that wait at the barrier between spill.)
        for (int i = 0; i < turns; ++i) {
            dma_barrier();
            if (i + 1 < mine) fetch(i + 1);
            if (i >= mine || j0 >= n) continue;
            for (int m = 0; m < QT; m += 32) {
                const int r0 = first_row(i) + m;
                if (r0 + 32 <= j0 * pr.G || r0 >= any1) continue;
                const unsigned to = (i & 1) * 2 * Sh::TILE + m * Tl::ROW;
                typename KeySums<T, DP>::Weights w;
                x.weigh(row_at + to, row_at + to + Sh::TILE, stats + (i & 1) * 8 * QT + m * 4 + 16 * (lane >> 5), 4 * QT,
                        r0 >= all0 && r0 + 32 <= all1, bits_between(see0 - r0, see1 - r0) >> (4 * (lane >> 5)), c, w);
                x.add(col_at + to, col_at + to + Sh::TILE, w);
            }
        }
    } else {
        x.clear();
    }
    const int lane_e = lane_again(), j_e = j0 + (lane_e & 31);
    CIRCATT_LDS float *buf = (CIRCATT_LDS float *)lds_mem;
    if (NG == 2) {
        static_assert(NG == 1 || 4 * 4 * Sh::FAR_PART <= (int)sizeof(lds_mem), "four wavefronts' sums");
        __syncthreads();
        if (group == 1) x.put(buf + wave * 64 * DP, lane_e);
        __syncthreads();
        if (group == 0) x.take(buf + wave * 64 * DP, lane_e);
    }
    if (sp.parts == 1 && kb * 4 < sp.far) {
        // the far sums of the block's keys, by everybody, as many groups of 32 keys at a
        // time as the tiles' memory holds: all four, but two of Float32 heads wider than 32
        constexpr int FIT = (int)sizeof(lds_mem) / (4 * Sh::FAR_PART), AT_ONCE = FIT < 4 ? FIT : 4;
        static_assert(FIT >= 1, "");
        const int groups = sp.far - kb * 4 < 4 ? sp.far - kb * 4 : 4;
        const float *from = pr.work + sp.far_at + (unit * sp.far + kb * 4) * sp.far_parts * Sh::FAR_PART;
        for (int g = 0; g < groups; g += AT_ONCE) {
            const int now = groups - g < AT_ONCE ? groups - g : AT_ONCE;
            __syncthreads();
            sum_far<T, DP, 256 * NG>(from + (int64_t)g * sp.far_parts * Sh::FAR_PART, now, sp.far_parts, buf);
            __syncthreads();
            if (group == 0 && wave >= g && wave < g + now) x.take(buf + (wave - g) * 64 * DP, lane_e);
        }
    }
    if (sp.parts > 1) {
        if (group == 0)
            x.write(pr.work + sp.part_at + (unit * sp.blocks * sp.parts + in) * Sh::PART + (32 * wave + (lane_e & 31)) * DP,
                    128 * DP, lane_e);
        return;
    }
    bool bad_k = false, bad_v = false;
    if (group == 0) {
        const int64_t out = ((int64_t)hg.b * pr.L + j_e) * pr.Hk * pr.D + (int64_t)hg.hk * pr.D;
        T *kd = static_cast<T *>(pr.dk) + out, *vd = static_cast<T *>(pr.dv) + out;
        if (j_e < n) {
            bad_k = store_channels(x.dk, kd, pr.D, lane_e, pr.scale);
            bad_v = store_channels(x.dv, vd, pr.D, lane_e, 1.f);
        } else if (j_e < pr.L) {
            zero_channels(kd, pr.D, lane_e);
            zero_channels(vd, pr.D, lane_e);
        }
    }
    share_repairs<4 * NG, true>((CIRCATT_LDS uint32_t *)lds_mem, group == 0 ? wave : -1, 4 * group + wave,
                                rows_of(__ballot(bad_k)), rows_of(__ballot(bad_v)), [&](int i, bool fix_k, bool fix_v) {
                                    const SlidingProblem pe = argument_again<SlidingProblem>();
                                    HeadGroup<T>(pe, unit, n).again(pe, k0 + i, k0 + (i & ~31), fix_k, fix_v);
                                });
}

// The partial sums of 32 keys, the far ones first, in the order of their parts: a
// wavefront a key.
template <typename T, int DP>
__global__ __launch_bounds__(256) void sliding_dkdv_join(SlidingProblem pr, WalkSplit sp) {
    typedef BwdShape<T, DP> Sh;
    __shared__ __attribute__((aligned(16))) float far_mem[Sh::FAR_PART];
    CIRCATT_LDS float *far = (CIRCATT_LDS float *)far_mem;
    const int lane = threadIdx.x & 63, groups = (pr.L + 31) / 32;
    const int64_t unit = blockIdx.x / groups;
    const int group = (int)(blockIdx.x - unit * groups);
    if (group < sp.far) {
        sum_far<T, DP, 256>(pr.work + sp.far_at + (unit * sp.far + group) * sp.far_parts * Sh::FAR_PART, 1, sp.far_parts, far);
        __syncthreads();
    }
    const HeadGroup<T> hg(pr, unit);
    for (int x = threadIdx.x >> 6; x < 32; x += 4) {
        const int j = group * 32 + x;
        if (j >= pr.L) return;
        const int64_t out = ((int64_t)hg.b * pr.L + j) * pr.Hk * pr.D + (int64_t)hg.hk * pr.D;
        Pair k{0.f, 0.f}, v{0.f, 0.f};
        if (j >= hg.n) {
            // behind the signal's length: zeros, though a row that is not finite makes
            // its zero weights' sums NaN
            store_row(static_cast<T *>(pr.dk) + out, lane, pr.D, k);
            store_row(static_cast<T *>(pr.dv) + out, lane, pr.D, v);
            continue;
        }
        if (group < sp.far) {
            // channel d of the key, as a wavefront's registers hold it
            auto place = [&](int d) { return (16 * (d >> 5) + 4 * ((d >> 3) & 3) + (d & 3)) * 64 + x + 8 * (d & 4); };
            if (lane < DP) k.a = far[place(lane)], v.a = far[Sh::FAR_PART / 2 + place(lane)];
            if (lane + 64 < DP) k.b = far[place(lane + 64)], v.b = far[Sh::FAR_PART / 2 + place(lane + 64)];
        }
        const float *w = pr.work + sp.part_at + (unit * sp.blocks + (j >> 7)) * sp.parts * Sh::PART + (j & 127) * DP;
        for (int i = 0; i < sp.parts; ++i, w += Sh::PART) {
            const Pair a = load_row(w, lane, DP), c = load_row(w + Sh::PART / 2, lane, DP);
            k.a += a.a;
            k.b += a.b;
            v.a += c.a;
            v.b += c.b;
        }
        k.a *= pr.scale;
        k.b *= pr.scale;
        store_row(static_cast<T *>(pr.dk) + out, lane, pr.D, k);
        store_row(static_cast<T *>(pr.dv) + out, lane, pr.D, v);
        const bool bad_k = __any(!is_finite(k.a) || !is_finite(k.b)), bad_v = __any(!is_finite(v.a) || !is_finite(v.b));
        if (bad_k || bad_v) {
            __threadfence_block();  // other lanes' stores
            hg.again(pr, j, group * 32, bad_k, bad_v);
        }
    }
}

// Parts: the estimate counts rounds of the chip's 256 compute units at the mean
// walk, or the longest walk alone, and three tiles' time for a workgroup's start
// and end, six where it leaves partial sums.  (The lengths of a padded batch are
// not known here: all signals count as full.)
WalkSplit walk_split(const SlidingProblem &pr) {
    const bool wide = pr.dtype == CIRCATT_F32;
    const int QT = wide ? 32 : 64, DP = (pr.D + 31) / 32 * 32;
    WalkSplit sp;
    sp.heads = make_fastdiv(pr.G);
    sp.blocks = (pr.L + 127) / 128;
    const int64_t units = (int64_t)pr.B * pr.Hk, n = units * sp.blocks;
    auto walk = [&](int64_t k0) {
        const int64_t tokens = pr.L - k0 < 127 + (int64_t)pr.W ? pr.L - k0 : 127 + (int64_t)pr.W;
        return (double)tokens * pr.G / QT;
    };
    double all = 0;
    for (int kb = 0; kb < sp.blocks; ++kb) all += walk(kb * 128);
    const double mean = all / sp.blocks, longest = walk(0);
    double best = 1e300;
    for (int p = 1; p <= 8; ++p) {
        const double rounds = (double)((n * p + 255) / 256), a = rounds * (mean / p), b = longest / p;
        const double cost = (a > b ? a : b) + rounds * (p > 1 ? 6 : 3);
        if (cost < best) best = cost, sp.parts = p;
    }
    // sinks that are seen from behind the window of their block; 4 tiles of 32 rows
    // for each of four wavefronts
    sp.far = 0;
    sp.far_parts = 1;
    const int64_t behind = (int64_t)pr.L - 127 - pr.W;
    if (pr.S > 0 && behind > 0) {
        const int64_t seen = pr.S < behind + 127 ? pr.S : behind + 127;
        sp.far = (int)((seen + 31) / 32);
        // and no more workgroups than fill the chip four times
        const int64_t parts = (behind * pr.G + 511) / 512, most = 2048 / (units * sp.far);
        sp.far_parts = (int)(parts < most ? parts : most < 1 ? 1 : most);
    }
    sp.far_at = ((int64_t)pr.B * pr.L * pr.H + 3) & ~(int64_t)3;
    sp.part_at = sp.far_at + units * sp.far * sp.far_parts * 32 * DP * 2;
    return sp;
}

template <typename T, int DP>
hipError_t forward(const SlidingProblem &pr, hipStream_t s) {
    const int blocks = (pr.L * pr.G + 127) / 128;
    sliding_fwd<T, DP><<<(unsigned)grid8((int64_t)pr.B * pr.Hk * blocks), 256, 0, s>>>(pr, blocks);
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
    sliding_dq<T, DP><<<(unsigned)grid8((int64_t)pr.B * pr.Hk * blocks), 256, 0, s>>>(pr, blocks);
    if (pr.dk != nullptr) {
        const WalkSplit sp = walk_split(pr);
        const int64_t units = (int64_t)pr.B * pr.Hk;
        if (sp.far > 0) sliding_dkdv_far<T, DP><<<(unsigned)(units * sp.far * sp.far_parts), 256, 0, s>>>(pr, sp);
        sliding_dkdv<T, DP><<<(unsigned)grid8(units * sp.blocks * sp.parts), 256 * BwdShape<T, DP>::NG, 0, s>>>(pr, sp);
        if (sp.parts > 1) sliding_dkdv_join<T, DP><<<(unsigned)(units * ((pr.L + 31) / 32)), 256, 0, s>>>(pr, sp);
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
    const int DP = (pr.D + 31) / 32 * 32;
    return sp.part_at + (sp.parts > 1 ? (int64_t)pr.B * pr.Hk * sp.blocks * sp.parts * 128 * DP * 2 : 0);
}

int64_t sliding_threads(const SlidingProblem &pr, bool backward) {
    const int64_t units = (int64_t)pr.B * pr.Hk, rows = 256 * grid8(units * (((int64_t)pr.L * pr.G + 127) / 128));
    if (!backward) return rows;
    const WalkSplit sp = walk_split(pr);
    // 512 threads, but 256 for some Float32 heads
    const int64_t keys = 512 * grid8(units * sp.blocks * sp.parts), far = 256 * units * sp.far * sp.far_parts;
    const int64_t join = sp.parts > 1 ? 256 * units * ((pr.L + 31) / 32) : 0;
    int64_t most = rows;
    for (int64_t n : {keys, far, join}) most = n > most ? n : most;
    return most;
}

hipError_t launch_sliding_fwd(const SlidingProblem &pr, hipStream_t s) {
    return pr.dtype == CIRCATT_F32 ? forward<0>(pr, s) : pr.dtype == CIRCATT_F16 ? forward<2>(pr, s) : forward<3>(pr, s);
}
hipError_t launch_sliding_bwd(const SlidingProblem &pr, hipStream_t s) {
    return pr.dtype == CIRCATT_F32 ? backward<0>(pr, s)
                                   : pr.dtype == CIRCATT_F16 ? backward<2>(pr, s) : backward<3>(pr, s);
}

}  // namespace circatt
