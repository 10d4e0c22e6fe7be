// Causal sliding-window attention with sinks on (batch, length, channels)
// signals, forward and backward, on the matrix cores.  X: the scores' kind, plain
// (sliding.hip) or shaped (shaped.hip, capped.hip).
#pragma once

#include "token_shape.h"

namespace circatt {
namespace {

using namespace tok;

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
// card reaches 1390 (1610 with its second operand transposed).  From windows of 128 (4 tiles a block, 76 us) to none (64 tiles)
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
// Shaped scores add vector instructions, which do not run beside the products here: at 8192
// tokens, 32 heads of 128 over 8, window 4096, bf16, each one a score is 38 us.  Plain
// scores take 445 us there, capped ones 465 (890 TFLOP/s; matrix cores busy 0.44 of a busy
// compute unit's time; they have no running maximum), with slopes 530, under a prefix
// 420; in a training step the sum of the rounded weights (KEPT) is 3% of the pass.
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
inline int64_t grid8(int64_t n) { return (n + 7) / 8 * 8; }

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

// What the rows of one signal see, and how the scores of a lane's row follow from its
// products.
struct PlainSignal {
    __device__ __forceinline__ PlainSignal(const SlidingProblem &, int, int) {}
    __device__ __forceinline__ Sight sight(const SlidingProblem &pr, int, int, int) const { return Sight{pr.W, pr.S}; }
    template <int KT>
    __device__ __forceinline__ TileList<KT> tiles(const SlidingProblem &pr, int lo, int hi) const {
        return TileList<KT>(lo, hi, pr.W, pr.S);
    }
    template <typename T>
    __device__ __forceinline__ PlainScorer scorer(const SlidingProblem &pr, int) const {
        return PlainScorer{pr.scale * kLog2e};
    }
    __device__ __forceinline__ PlainView view(const SlidingProblem &pr, int pos, int) const {
        return PlainView(pos, pr.W, pr.S, pr.scale * kLog2e);
    }
};
template <bool CAP>
struct ShapedSignal {
    const int32_t *places;
    int P;
    __device__ __forceinline__ ShapedSignal(const ShapedSlidingProblem &pr, int b, int n)
        : places(pr.shape.places == nullptr ? nullptr : pr.shape.places + b * pr.shape.places_row),
          P(uniform(clamp_prefix(pr.shape.prefix, b, n))) {}
    // at: of this lane's row (-1: none); lo, hi: of the wavefront's first and last
    __device__ __forceinline__ ShapedSight sight(const ShapedSlidingProblem &pr, int at, int, int) const {
        const int start = at < 0 ? 0 : document_start(places, at);
        return ShapedSight{pr.W, pr.S, P, start, uniform(start), __builtin_amdgcn_readlane(start, 31)};
    }
    template <int KT>
    __device__ __forceinline__ ShapedTiles<KT> tiles(const ShapedSlidingProblem &pr, int lo, int hi) const {
        return ShapedTiles<KT>(lo, hi, pr.W, pr.S, P, uniform(document_start(places, lo)));
    }
    template <typename T>
    __device__ __forceinline__ ShapedScorer<CAP, CAP && sizeof(T) == 4> scorer(const ShapedSlidingProblem &pr, int h) const {
        const bool biased = pr.shape.slopes != nullptr;
        return ShapedScorer<CAP, CAP && sizeof(T) == 4>(pr.scale, pr.shape.curve, biased ? pr.shape.slopes[h] * kLog2e : 0.f,
                                                        biased, __is_same(T, __bf16));
    }
    __device__ __forceinline__ ShapedView view(const ShapedSlidingProblem &pr, int pos, int h) const {
        const float slope = pr.shape.slopes == nullptr ? 0.f : pr.shape.slopes[h] * kLog2e;
        return ShapedView(pos, document_start(places, pos), pr.W, pr.S, P,
                          ShapedScore{pr.shape.curve, pr.scale * kLog2e, slope, CAP});
    }
};
template <typename X>
struct SignalOf {
    typedef ShapedSignal<X::kCap> type;
};
template <>
struct SignalOf<Plain> {
    typedef PlainSignal type;
};

// KEPT: of a training step with shaped scores: y_rest takes y to the output that is
// divided by the sum of the rounded weights (y itself is a call's without gradients).
template <typename X, typename T, int DP, bool KEPT>
__global__ __launch_bounds__(256, sizeof(T) == 4 && DP > 64 ? 1 : 2) void sliding_fwd(typename X::Sliding pr, int blocks) {
    typedef typename X::Sliding Problem;
    typedef typename SignalOf<X>::type Signal;
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
        const Signal sg(pr, b, n);
        const auto see = sg.sight(pr, at, lo, hi);
        const auto tiles = sg.template tiles<KT>(pr, r0 / pr.G, last / pr.G);
        const auto score = sg.template scorer<T>(pr, hk * pr.G + g);
        const float c = score.factor();
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
        auto look = [&](f16v (&s)[NB], int i, bool first) {  // scores of tile i, its keys hidden, and the largest
            const int k0 = tiles.key(i);
            score.shape(s, k0, at, lo, lane);
            if (!see.all(lo, hi, k0, KT)) {
                asm volatile("");
#pragma unroll
                for (int m = 0; m < NB; ++m) hide_keys(s[m], see.bits(at, k0 + 32 * m), lane);
            }
            mx = score.largest(x, s, first);
        };
        auto weigh = [&](const f16v (&s)[NB], V8<T> (&p)[2 * NB]) {
            x.template weigh<NB, KEPT>(s, p, c);
        };
        auto step = [&](const f16v (&s)[NB], f16v (&t)[NB], int i) {
            round(i);
            V8<T> p[2 * NB];
            score.raise(x, mx);
            x.scores(row_at + kp * Rg::TILE, t);
            weigh(s, p);
            x.template add<NB>(col_at + vp * Rg::TILE, p);
            next();
            look(t, i + 1, false);
        };
        f16v sa[NB], sb[NB];
        int i = -1;
        for (; i < (live ? first - 1 : count); ++i, next()) round(i);
        if (live) {
            round(i);
            x.scores(row_at + kp * Rg::TILE, sa);
            look(sa, first, true);
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
            score.raise(x, mx);
            weigh(sa, p);
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
                bad = store_channels(x.o, y + ((int64_t)at * pr.H + g) * pr.D, pr.D, lane, inv, out_of_reach<X::kCap>(l));
                if (rest != nullptr)
                    store_rests(x.o, rest + ((int64_t)at * pr.H + g) * pr.D, pr.D, lane, inv,
                                KEPT ? 1.f / x.total_rounded() : inv);
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
                // (With capped scores they may be for want of a larger reference too.)
                const Problem pe = argument_again<Problem>();
                const SignalKV<T> kv = signal_rows<T>(pe, b, hk);
                auto tile_end = [&](int j) { return (int)((int64_t)j + KT - j % KT < n ? j + KT - j % KT : n); };
                if constexpr (X::kCap) {
                } else if constexpr (X::kShaped) {
                    // Hidden from a row: what its tiles hold before its document and
                    // its window, the tiles of the first document's sinks or of the
                    // prefix, and what lies behind the first row.
                    const Signal sg(pe, b, n);
                    const int t0 = r0 / pe.G, s0 = document_start(sg.places, t0), s1 = document_start(sg.places, hi);
                    const int low = t0 - pe.W + 1 > s0 ? t0 - pe.W + 1 : s0, seen = hi - pe.W + 1 > s1 ? hi - pe.W + 1 : s1;
                    const int top = sg.P > s0 + pe.S ? sg.P : s0 + pe.S;
                    const int behind = lo + 1 > sg.P ? lo + 1 : sg.P;
                    if (!bad_values(kv, low / KT * KT, seen, pe.D) &&
                        !bad_values(kv, behind, tile_end(hi + 1 > sg.P ? hi : sg.P - 1), pe.D) &&
                        !((pe.S > 0 || sg.P > 0) &&
                          (bad_values(kv, s0 / KT * KT, s1 > s0 ? s1 : s0, pe.D) ||
                           bad_values(kv, sg.P > s0 ? sg.P : s0, tile_end(top < n ? top : n - 1), pe.D))))
                        again = 0;
                } else {
                    const int window = r0 / pe.G - pe.W + 1;
                    if (!bad_values(kv, window > 0 ? window / KT * KT : 0, hi - pe.W + 1, pe.D) &&
                        !bad_values(kv, lo + 1, tile_end(hi), pe.D) &&
                        !(pe.S % KT != 0 && bad_values(kv, pe.S, tile_end(pe.S), pe.D)))
                        again = 0;
                }
            }
        }
        // (The list lies in a K tile: the last round, whose barrier is behind all, reads
        // none.)
        share_repairs<4, false>((CIRCATT_LDS uint32_t *)lds, wave, wave, again, 0, [&](int i, bool, bool) {
            const Problem pe = argument_again<Problem>();
            const int aj = (r0 + i) / pe.G, h = hk * pe.G + r0 + i - aj * pe.G;
            const int64_t out = (((int64_t)b * pe.L + aj) * pe.H + h) * pe.D;
            forward_row(static_cast<const T *>(pe.q) + b * pe.q_batch + aj * pe.q_row + (int64_t)h * pe.D,
                        static_cast<T *>(pe.y) + out, pe.y_rest == nullptr ? nullptr : static_cast<T *>(pe.y_rest) + out,
                        signal_rows<T>(pe, b, hk), Signal(pe, b, n).view(pe, aj, h), pe.D);
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
//
// LOW: dS goes into dQ' as two values of the element type, the second what rounding took
// from the first.  Capped scores are large ones, of which few keys carry a row, and dq was
// up to 2.2 times as far off as where its results alone are rounded; with that and the
// forward's sum of rounded weights, 1.2 times.  It is a third more products: of 2 x 4099
// tokens in documents of up to 1200, 12 heads of 80 over 4, cap 30, f16, 87 us have become
// 97.  Scores that are not capped have it where walks are short or that may be (few_keys).
template <typename X, typename T, int DP, bool LOW>
__global__ __launch_bounds__(256, sizeof(T) == 4 && DP > 32 ? 1 : 2) void sliding_dq(typename X::Sliding pr, int blocks) {
    typedef typename SignalOf<X>::type Signal;
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
        const Signal sg(pr, b, n);
        const auto see = sg.sight(pr, at, lo, hi);
        const auto tiles = sg.template tiles<KT>(pr, r0 / pr.G, last / pr.G);
        const auto score = sg.template scorer<T>(pr, hk * pr.G + g);
        const float c = score.unit();
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
                f16v bend = f16v{};
                if constexpr (X::kShaped) {
                    if constexpr (X::kCap) score.caps(s, bend);
                    f16v one[1] = {s};
                    score.exponents(one, k0, at, lo, lane, lse);
                    s = one[0];
                }
#pragma unroll
                for (int x = 0; x < 16; ++x)
                    s[x] = __builtin_amdgcn_exp2f(X::kShaped ? s[x] : fmaf(s[x], c, -lse)) * (dp[x] - d);
                if (!see.all(lo, hi, k0, 32)) {
                    asm volatile("");  // a branch: few tiles need it
                    const uint32_t half = see.bits(at, k0) >> (4 * (lane >> 5));
#pragma unroll
                    for (int x = 0; x < 16; ++x)
                        if (!(half & place_bit(x))) {
                            s[x] = 0.f;
                            if constexpr (X::kCap) bend[x] = 0.f;
                        }
                }
                V8<T> ds[2], low[2];
#pragma unroll
                for (int x = 0; x < 16; ++x) {
                    rest += s[x];  // (of the capped scores: those sum to zero)
                    const float e = X::kCap ? s[x] * bend[x] : s[x];
                    ds[x >> 3][x & 7] = (T)e;
                    if constexpr (LOW) low[x >> 3][x & 7] = (T)(e - (float)ds[x >> 3][x & 7]);
                }
                products<T, 2 * OT, 4>([&](int i) { return Tl::col(kc, 16 * (i & 1), i >> 1); },
                                       [&](int i, V8<T> a) {
                                           o[i >> 1] = mma(a, ds[i & 1], o[i >> 1]);
                                           if constexpr (LOW) o[i >> 1] = mma(a, low[i & 1], o[i >> 1]);
                                       });
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
                       gh + aj * pr.dy_row + (int64_t)gj * pr.D, dq + oj, pr.lse[sj], pr.work + sj, kv,
                       sg.view(pr, aj, hk * pr.G + gj), pr.D, pr.scale);
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
//
// Shaped: 2 x 4096 tokens, 16 heads of 128 over 4, window 1024, slopes, bf16: 200 us,
// waiting 0.50 of the cycles, capped at 50 instead 255 and 0.61; 2 x 4099 in documents of up to 1200, 12 heads of 80 over 4,
// cap 30, f16: 100 us and 13 to add up, walks of some 20 tiles, whose starts and ends are
// most of it.
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
    int each;            // with documents or a prefix, tiles a part: short walks have fewer parts
    __device__ __forceinline__ int of(int tiles) const {
        const int p = (tiles + each / 2) / each;
        return p < 1 ? 1 : p < parts ? p : parts;
    }
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
// The slopes of a head of keys' packed rows, its address in scalar registers (which
// the compiler would form in others).
__device__ __forceinline__ const float *slopes_of(const ShapedSlidingProblem &pr, int hk) {
    const uint64_t p = reinterpret_cast<uint64_t>(pr.row_slopes + (int64_t)hk * pr.L * pr.G);
    return reinterpret_cast<const float *>((uint64_t)(uint32_t)uniform((int)(p >> 32)) << 32 | (uint32_t)uniform((int)p));
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

// Tokens [first, end) whose rows see a key.  The walk of a block of keys is over the
// rows of tokens [A, E).
struct KeyRows {
    int first, end;
};
struct PlainKeys {
    __device__ __forceinline__ PlainKeys(const SlidingProblem &, int, int) {}
    __device__ __forceinline__ static int one_row(int W, int j, int n) { return n - j < W ? n : j + W; }
    // the rows of the keys k0 .. kn: kn's window (rows behind it that see a sink are
    // another walk's)
    __device__ __forceinline__ KeyRows walk(const SlidingProblem &pr, int k0, int kn, int n, int) const {
        return KeyRows{k0, n - kn > pr.W ? kn + pr.W : n};
    }
    __device__ __forceinline__ KeyRows rows(const SlidingProblem &pr, int j, int end) const {
        return KeyRows{j, j < pr.S ? end : one_row(pr.W, j, end)};
    }
    // of the keys j0 .. j0 + 31: rows that see all of them, and any
    __device__ __forceinline__ KeyRows all(const SlidingProblem &pr, int j0, int end, int) const {
        return KeyRows{j0 + 31, j0 + 31 < pr.S ? end : one_row(pr.W, j0, end)};
    }
    __device__ __forceinline__ KeyRows any(const SlidingProblem &pr, int j0, int end, int) const {
        return KeyRows{j0, j0 < pr.S ? end : one_row(pr.W, j0 + 31, end)};
    }
};
__device__ __forceinline__ int wave_most(int x) {
    for (int m = 32; m; m >>= 1) {
        const int o = __shfl_xor(x, m, 64);
        x = o > x ? o : x;
    }
    return uniform(x);
}
// With documents or a prefix (masked) there is no other walk, and a block's own goes as
// far as the rows that see one of its keys.
struct ShapedKeys {
    const int32_t *places, *ends;
    int P;
    bool masked;
    __device__ __forceinline__ ShapedKeys(const ShapedSlidingProblem &pr, int b, int n)
        : places(pr.shape.places == nullptr ? nullptr : pr.shape.places + b * pr.shape.places_row),
          ends(pr.shape.places == nullptr ? nullptr : pr.ends + (int64_t)b * pr.L),
          P(uniform(clamp_prefix(pr.shape.prefix, b, n))),
          masked(pr.shape.places != nullptr || pr.shape.prefix != nullptr) {}
    // key j < n among rows below `end`, the signal's length or a walk's end
    __device__ __forceinline__ KeyRows rows(const ShapedSlidingProblem &pr, int j, int end) const {
        int most = end;
        if (places != nullptr) {
            const int e = ends[j];
            most = e < most ? e : most;
        }
        const bool far = j < P || j - document_start(places, j) < pr.S;
        return KeyRows{j < P ? 0 : j, far || most - j < pr.W ? most : j + pr.W};
    }
    // The block's last key is seen furthest, a sink of its document to the document's end, or
    // of a signal that has or might have had a prefix, and the prefix, to the signal's.
    __device__ __forceinline__ KeyRows walk(const ShapedSlidingProblem &pr, int k0, int kn, int n, int) const {
        int last = n;
        bool far = k0 < P || (masked && k0 < pr.S);
        if (places != nullptr && k0 < n) {
            const int e = ends[kn];
            last = e < n ? e : n;
            far = pr.S > 0 && k0 - document_start(places, kn) < pr.S;
        }
        return KeyRows{k0 < P ? 0 : k0, far || last - kn < pr.W ? last : kn + pr.W};
    }
    // (keys from `end` on: what the walk's last has)
    __device__ __forceinline__ KeyRows one(const ShapedSlidingProblem &pr, int j0, int end, int lane) const {
        const int j = j0 + (lane & 31);
        return rows(pr, j < end ? j : end - 1, end);
    }
    __device__ __forceinline__ KeyRows all(const ShapedSlidingProblem &pr, int j0, int end, int lane) const {
        const KeyRows r = one(pr, j0, end, lane);
        return KeyRows{wave_most(r.first), -wave_most(-r.end)};
    }
    __device__ __forceinline__ KeyRows any(const ShapedSlidingProblem &pr, int j0, int end, int lane) const {
        const KeyRows r = one(pr, j0, end, lane);
        return KeyRows{-wave_most(-r.first), wave_most(r.end)};
    }
};
template <typename X>
struct KeysOf {
    typedef ShapedKeys type;
};
template <>
struct KeysOf<Plain> {
    typedef PlainKeys type;
};

// Scores of a key by its rows, for the row by row form.
struct PlainRowScore {
    float c;
    __device__ __forceinline__ PlainRowScore(const SlidingProblem &pr, int, int) : c(pr.scale * kLog2e) {}
    __device__ __forceinline__ float score(float dot, int, int) const { return c * dot; }
    __device__ __forceinline__ float bend(float) const { return 1.f; }
};
template <bool CAP>
struct ShapedRowScore {
    ShapedScore s;
    const float *slopes;
    int j;
    __device__ __forceinline__ ShapedRowScore(const ShapedSlidingProblem &pr, int hk, int j)
        : s{pr.shape.curve, pr.scale * kLog2e, 0.f, CAP},
          slopes(pr.shape.slopes == nullptr ? nullptr : pr.shape.slopes + (int64_t)hk * pr.G), j(j) {}
    __device__ __forceinline__ float score(float dot, int i, int g) const {
        ShapedScore x = s;
        if (slopes != nullptr) x.slope = slopes[g] * kLog2e;
        return x.at(dot, i - j);
    }
    __device__ __forceinline__ float bend(float dot) const { return s.bend(dot); }
};
template <typename X>
struct RowScoreOf {
    typedef ShapedRowScore<X::kCap> type;
};
template <>
struct RowScoreOf<Plain> {
    typedef PlainRowScore type;
};

// The score of a lane's key by the rows in registers.
struct PlainKeyScore {
    float c;
    __device__ __forceinline__ PlainKeyScore(const SlidingProblem &pr, int) : c(pr.scale * kLog2e) {}
    __device__ __forceinline__ float unit() const { return c; }
};
template <bool CAP, bool FINE>
struct ShapedKeyScore : ShapedScorer<CAP, FINE, ReadCurve<ShapedSlidingProblem>> {
    float token;  // of the key
    __device__ __forceinline__ ShapedKeyScore(const ShapedSlidingProblem &pr, int j)
        : ShapedScorer<CAP, FINE, ReadCurve<ShapedSlidingProblem>>(pr.scale, pr.shape.curve, 0.f,
                                                                   pr.shape.slopes != nullptr, false),
          token((float)j) {}
};
template <typename X, typename T>
struct KeyScoreOf {
    typedef ShapedKeyScore<X::kCap, X::kCap && sizeof(T) == 4> type;
};
template <typename T>
struct KeyScoreOf<Plain, T> {
    typedef PlainKeyScore type;
};

// One wavefront's 32 keys: operands, sums, and 32 query rows' share of them.
// LOW: P and dS as two values of the element type each (the second: what rounding took
// from the first).
template <typename X, typename T, int DP, bool LOW = false>
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
        V8<T> p[2], ds[2], low_p[2], low_ds[2];
    };
    // (and with slopes the rows' slopes and tokens, 2 and 3 strides on)
    typedef typename KeyScoreOf<X, T>::type Score;
    __device__ __forceinline__ void weigh(unsigned qr, unsigned gr, unsigned st, int stride, bool every, uint32_t half,
                                          const Score &score, Weights &w) const {
        f16v s = f16v{}, dp = f16v{};
        products<T, 2 * STEPS, AHEAD - 1>([&](int i) { return Tl::row(i & 1 ? gr : qr, 0, i >> 1); },
                                      [&](int i, V8<T> a) {
                                          if (i & 1) dp = mma(a, v[i >> 1], dp);
                                          else s = mma(a, k[i >> 1], s);
                                      });
        f16v bend = f16v{};
        if constexpr (X::kShaped) {
            if constexpr (X::kCap) score.caps(s, bend);
            score.exponents_of_rows(s, st, stride, score.token);
        }
#pragma unroll
        for (int x = 0; x < 16; x += 4) {
            const f4v ls = X::kShaped ? f4v{} : *(const CIRCATT_LDS f4v *)(st + 8 * x);
            const f4v dd = *(const CIRCATT_LDS f4v *)(st + stride + 8 * x);
#pragma unroll
            for (int y = 0; y < 4; ++y) {
                s[x + y] = __builtin_amdgcn_exp2f(X::kShaped ? s[x + y] : fmaf(s[x + y], score.unit(), -ls[y]));
                dp[x + y] = s[x + y] * (dp[x + y] - dd[y]);
                if constexpr (X::kCap) dp[x + y] *= bend[x + y];
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
            if constexpr (LOW) {
                w.low_p[x >> 3][x & 7] = (T)(s[x] - (float)w.p[x >> 3][x & 7]);
                w.low_ds[x >> 3][x & 7] = (T)(dp[x] - (float)w.ds[x >> 3][x & 7]);
            }
        }
    }
    __device__ __forceinline__ void add(unsigned qc, unsigned gc, const Weights &w) {
        products<T, 4 * OT, AHEAD>([&](int i) { return Tl::col(i & 1 ? qc : gc, 16 * ((i >> 1) & 1), i >> 2); },
                                   [&](int i, V8<T> a) {
                                       if (i & 1) dk[i >> 2] = mma(a, w.ds[(i >> 1) & 1], dk[i >> 2]);
                                       else dv[i >> 2] = mma(a, w.p[(i >> 1) & 1], dv[i >> 2]);
                                       if constexpr (LOW) {
                                           if (i & 1) dk[i >> 2] = mma(a, w.low_ds[(i >> 1) & 1], dk[i >> 2]);
                                           else dv[i >> 2] = mma(a, w.low_p[(i >> 1) & 1], dv[i >> 2]);
                                       }
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
    // (With documents or a prefix: a tile of rows more on either side of those that see
    // one of the 32 keys.)
    template <typename X>
    __device__ void again(const typename X::Sliding &pr, int j, int j0, bool bad_k, bool bad_v) const {
        KeyRows r;
        int64_t from, last;  // packed rows
        if constexpr (X::kShaped) {
            const ShapedKeys keys(pr, b, n);
            r = keys.rows(pr, j, n);
            const KeyRows any = keys.any(pr, j0, n, lane_again());
            from = (int64_t)any.first * pr.G - 64;
            last = (int64_t)any.end * pr.G + 64;
        } else {
            r = KeyRows{j, j < pr.S || n - j < pr.W ? n : j + pr.W};
            const int64_t tokens = (int64_t)j0 + 31 + pr.W + (30 + pr.G) / pr.G;
            from = (int64_t)j0 * pr.G;
            last = (j0 < pr.S ? n : tokens) * pr.G;
        }
        from = from < 0 ? 0 : from;
        last = last > rows ? rows : last;
        const int first = r.first * pr.G, end = r.end * pr.G;
        const bool fix_k = bad_k && !bad_rows(first, end);
        const bool fix_v = bad_v && (bad_rows((int)from, first) || bad_rows(end, (int)last));
        if (!fix_k && !fix_v) return;
        const int64_t out = ((int64_t)b * pr.L + j) * pr.Hk * pr.D + (int64_t)hk * pr.D;
        dkdv_row(k + j * pr.k_row, v + j * pr.v_row, q, pr.q_row, dy, pr.dy_row, lse, dsum, static_cast<T *>(pr.dk) + out,
                 static_cast<T *>(pr.dv) + out, fix_k, fix_v, first, end, pr.G, pr.D,
                 typename RowScoreOf<X>::type(pr, hk, j), pr.scale);
    }
};

template <typename X, typename T, int DP>
__global__ __launch_bounds__(256, sizeof(T) == 4 && DP > 32 ? 1 : 2) void sliding_dkdv_far(typename X::Sliding pr, WalkSplit sp) {
    typedef BwdShape<T, DP> Sh;
    typedef Tile<T, DP> Tl;
    // two buffers for each wavefront, but for tiles that are too long for that
    constexpr int BUFS = 16 * Sh::FAR_TILE <= 128 * 1024 ? 2 : 1, STATS = 8 * BUFS * Sh::FAR_TILE;
    constexpr int SUMS = 32 * DP * 2 * 4, NS = X::kShaped ? 512 : 256;  // bytes of a tile's statistics
    __shared__ __attribute__((aligned(1024))) char lds_mem[STATS + 4 * BUFS * NS > SUMS ? STATS + 4 * BUFS * NS : SUMS];
    const int64_t unit = blockIdx.x / (sp.far * sp.far_parts);
    const int in = (int)(blockIdx.x - unit * (sp.far * sp.far_parts)), k0 = in / sp.far_parts * 32, part = in % sp.far_parts;
    const HeadGroup<T> hg(pr, unit);
    const int lane = threadIdx.x & 63, wave = uniform(threadIdx.x >> 6), j = k0 + (lane & 31);
    const unsigned lds = lds_byte((const CIRCATT_LDS char *)lds_mem) + wave * (2 * BUFS * Sh::FAR_TILE);
    const unsigned st = lds_byte((const CIRCATT_LDS char *)lds_mem) + STATS + wave * BUFS * NS;
    KeySums<X, T, DP> x;
    // a block of keys in which none is seen from behind its window adds nothing
    const FarRows far(pr, k0, hg.n);
    const int tiles = (far.count + 31) / 32, parts = 4 * sp.far_parts, w = 4 * part + wave;
    const int i0 = (int)((int64_t)tiles * w / parts), i1 = (int)((int64_t)tiles * (w + 1) / parts);
    if (i0 < i1) {
        const int jj = j < hg.n ? j : hg.n - 1;
        x.start(hg.k + jj * pr.k_row, hg.v + jj * pr.v_row, pr.D, lane);
        const unsigned row_at = Tl::row_lane(lane) + lds, col_at = Tl::col_lane(lane) + lds;
        const typename KeyScoreOf<X, T>::type score(pr, j);
        auto fetch = [&](int i) {
            const int r0 = far.first + 32 * i, y = BUFS == 2 ? i & 1 : 0;
            const unsigned to = lds + y * 2 * Sh::FAR_TILE;
            fetch_packed<T, DP, 32, 64>(hg.q, pr.q_row, r0, pr.G, sp.heads, hg.n, pr.D, lane, to);
            fetch_packed<T, DP, 32, 64>(hg.dy, pr.dy_row, r0, pr.G, sp.heads, hg.n, pr.D, lane, to + Sh::FAR_TILE);
            fetch_stats<32>(hg.lse, r0, hg.rows, st + y * NS);
            fetch_stats<32>(hg.dsum, r0, hg.rows, st + y * NS + 128);
            if constexpr (X::kShaped) {
                if (score.biased) {
                    fetch_stats<32>(slopes_of(pr, hg.hk), r0, hg.rows, st + y * NS + 256);
                    fetch_stats<32>(pr.row_tokens, r0, hg.rows, st + y * NS + 384);
                }
            }
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
            typename KeySums<X, T, DP>::Weights wt;
            x.weigh(row_at + to, row_at + to + Sh::FAR_TILE, st + y * NS + 16 * (lane >> 5), 128, k0 + 32 <= pr.S,
                    j < pr.S ? ~0u : 0u, score, wt);
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

template <typename X, typename T, int DP, bool LOW>
__global__ __launch_bounds__((256 * BwdShape<T, DP>::NG), (sizeof(T) == 2 && DP <= 64 ? 2 : 1))
void sliding_dkdv(typename X::Sliding pr, WalkSplit sp) {
    typedef typename X::Sliding Problem;
    typedef BwdShape<T, DP> Sh;
    typedef Tile<T, DP> Tl;
    constexpr int QT = Sh::QT, NG = Sh::NG, NS = (X::kShaped ? 16 : 8) * QT;  // bytes of a tile's statistics
    __shared__ __attribute__((aligned(1024))) char lds_mem[NG * (4 * Sh::TILE + 2 * NS)];
    // workgroups of one unit: its blocks, part by part, on one XCD
    // (shaped: all blocks' last parts, which long walks alone have, then those before:
    // the long walks begin first, and no idle workgroups lie at every other place, as
    // workgroups go to the chip's engines in turn and would leave engines without work)
    int64_t unit;
    int kb, part;
    if constexpr (X::kShaped) {
        const int per = (gridDim.x >> 3) / sp.parts, at = blockIdx.x >> 3;
        part = sp.parts - 1 - at / per;
        const int64_t id = (int64_t)(blockIdx.x & 7) * per + at % per;
        unit = id / sp.blocks;
        if (unit >= (int64_t)pr.B * pr.Hk) return;
        kb = (int)(id - unit * sp.blocks);
    } else {
        const int64_t id = (int64_t)(blockIdx.x & 7) * (gridDim.x >> 3) + (blockIdx.x >> 3);
        unit = id / (sp.blocks * sp.parts);
        if (unit >= (int64_t)pr.B * pr.Hk) return;
        const int in = (int)(id - unit * (sp.blocks * sp.parts));
        kb = in / sp.parts;
        part = in - kb * sp.parts;
    }
    const HeadGroup<T> hg(pr, unit);
    const int n = hg.n, lane = threadIdx.x & 63, wave = uniform(threadIdx.x >> 6) & 3, group = uniform(threadIdx.x >> 8);
    const int tid = threadIdx.x & 255;
    // packed query rows of the walk: the block's tokens and W - 1 behind
    const int k0 = kb * 128, kn = k0 + 127 < n - 1 ? k0 + 127 : n - 1;
    const typename KeysOf<X>::type keys(pr, hg.b, n);
    const KeyRows walk = keys.walk(pr, k0, kn, n, lane);
    const int begin = X::kShaped ? uniform(walk.first) : walk.first, end = X::kShaped ? uniform(walk.end) : walk.end;
    const int tiles = k0 < n ? ((end - begin) * pr.G + QT - 1) / QT : 0;
    int parts = sp.parts;
    if constexpr (X::kShaped) {
        if (keys.masked) parts = uniform(sp.of(tiles));
        if (part >= parts) return;
    }
    const int i0 = (int)((int64_t)tiles * part / parts), i1 = (int)((int64_t)tiles * (part + 1) / parts);
    const int j0 = k0 + 32 * wave, j = j0 + (lane & 31), jj = j < n ? j : n - 1;
    const unsigned lds = lds_byte((const CIRCATT_LDS char *)lds_mem) + group * 4 * Sh::TILE;
    const unsigned stats = lds_byte((const CIRCATT_LDS char *)lds_mem) + NG * 4 * Sh::TILE + group * 2 * NS;
    const typename KeyScoreOf<X, T>::type score(pr, j);
    KeySums<X, T, DP, LOW> x;
    if (i0 < i1) {
        // a group's turn i: tile i0 + NG i + group
        const int mine = (i1 - i0 - group + NG - 1) / NG, turns = (i1 - i0 + NG - 1) / NG;
        auto first_row = [&](int i) { return begin * pr.G + (i0 + NG * i + group) * QT; };
        auto fetch = [&](int i) {
            const int r0 = first_row(i);
            const unsigned to = lds + (i & 1) * 2 * Sh::TILE, st = stats + (i & 1) * NS;
            fetch_packed<T, DP, QT, 256>(hg.q, pr.q_row, r0, pr.G, sp.heads, n, pr.D, tid, to);
            fetch_packed<T, DP, QT, 256>(hg.dy, pr.dy_row, r0, pr.G, sp.heads, n, pr.D, tid, to + Sh::TILE);
            if (wave == 0) fetch_stats<QT>(hg.lse, r0, hg.rows, st);
            if (wave == 1) fetch_stats<QT>(hg.dsum, r0, hg.rows, st + 4 * QT);
            if constexpr (X::kShaped) {
                if (score.biased && wave == 2)
                    fetch_stats<QT>(slopes_of(pr, hg.hk), r0, hg.rows, st + 8 * QT);
                if (score.biased && wave == 3) fetch_stats<QT>(pr.row_tokens, r0, hg.rows, st + 12 * QT);
            }
        };
        if (mine > 0) fetch(0);
        x.start(hg.k + jj * pr.k_row, hg.v + jj * pr.v_row, pr.D, lane);
        const unsigned row_at = Tl::row_lane(lane) + lds, col_at = Tl::col_lane(lane) + lds;
        // the rows that see key j: from its token on, to its window's end or, of a sink,
        // the walk's (rows behind it in the last tile belong to sliding_dkdv_far)
        const KeyRows mine_rows = keys.rows(pr, X::kShaped ? jj : j, end);
        const int see0 = mine_rows.first * pr.G, see1 = mine_rows.end * pr.G;
        // and those that see all of the wavefront's keys, or any
        const KeyRows all_rows = keys.all(pr, j0, X::kShaped ? n : end, lane);
        const KeyRows any_rows = keys.any(pr, j0, X::kShaped ? n : end, lane);
        const int all0 = all_rows.first * pr.G, all1 = (all_rows.end < end ? all_rows.end : end) * pr.G;
        const int any0 = any_rows.first * pr.G, any1 = (any_rows.end < end ? any_rows.end : end) * pr.G;
        // (Groups half a block apart, one forming weights while the other adds, took 167
        // us where this takes 112: the weights that wait at the barrier between spill.)
        for (int i = 0; i < turns; ++i) {
            dma_barrier();
            if (i + 1 < mine) fetch(i + 1);
            if (i >= mine || j0 >= n) continue;
            for (int m = 0; m < QT; m += 32) {
                const int r0 = first_row(i) + m;
                if (r0 + 32 <= any0 || r0 >= any1) continue;
                const unsigned to = (i & 1) * 2 * Sh::TILE + m * Tl::ROW;
                typename KeySums<X, T, DP, LOW>::Weights w;
                x.weigh(row_at + to, row_at + to + Sh::TILE, stats + (i & 1) * NS + m * 4 + 16 * (lane >> 5), 4 * QT,
                        r0 >= all0 && r0 + 32 <= all1, bits_between(see0 - r0, see1 - r0) >> (4 * (lane >> 5)), score, w);
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
    if (parts == 1 && kb * 4 < sp.far) {
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
    if (parts > 1) {
        if (group == 0)
            x.write(pr.work + sp.part_at + ((unit * sp.blocks + kb) * sp.parts + part) * Sh::PART + (32 * wave + (lane_e & 31)) * DP,
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
                                    const Problem pe = argument_again<Problem>();
                                    HeadGroup<T>(pe, unit, n).template again<X>(pe, k0 + i, k0 + (i & ~31), fix_k, fix_v);
                                });
}

// The partial sums of 32 keys, the far ones first, in the order of their parts: a
// wavefront a key.
template <typename X, typename T, int DP>
__global__ __launch_bounds__(256) void sliding_dkdv_join(typename X::Sliding pr, WalkSplit sp) {
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
    int parts = sp.parts;
    if constexpr (X::kShaped) {
        const ShapedKeys keys(pr, hg.b, hg.n);
        if (keys.masked) {
            const int k0 = group / 4 * 128, kn = k0 + 127 < hg.n - 1 ? k0 + 127 : hg.n - 1;
            const KeyRows walk = keys.walk(pr, k0, kn, hg.n, lane);
            parts = uniform(sp.of(k0 < hg.n ? ((walk.end - walk.first) * pr.G + Sh::QT - 1) / Sh::QT : 0));
            if (parts == 1) return;  // the block's gradients are written
        }
    }
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
        for (int i = 0; i < parts; ++i, w += Sh::PART) {
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
            hg.template again<X>(pr, j, group * 32, bad_k, bad_v);
        }
    }
}

// Parts: the estimate counts rounds of the chip's 256 compute units at the mean
// walk, or the longest walk alone, and three tiles' time for a workgroup's start
// and end, six where it leaves partial sums.  (The lengths of a padded batch are
// not known here: all signals count as full.)
// With documents or a prefix walks leave no rows behind, and where there is a prefix
// the first block's is all rows: parts are for those, and the kernels give short walks
// fewer (of).  2 x 4096 tokens, 16 heads of 128 over 4, window 1024, prefixes of 64: 280
// us and 22 to add up, in one part 520; all walks in four parts 305 and 28.  2 x 4099
// tokens in documents of up to 1200, 12 heads of 80 over 4: 105 and 13, all walks in four
// parts 108 and 22.
inline WalkSplit walk_split(const SlidingProblem &pr, int masked = kUnmasked) {
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
    const double mean = all / sp.blocks, longest = masked == kPrefix ? (double)pr.L * pr.G / QT : walk(0);
    double best = 1e300;
    for (int p = 1; p <= 8; ++p) {
        const double rounds = (double)((n * p + 255) / 256), a = rounds * (mean / p), b = longest / p;
        const double cost = (a > b ? a : b) + rounds * (p == 1 ? 3 : masked == kUnmasked ? 6 : 12);
        if (cost < best) best = cost, sp.parts = p;
    }
    // what a part is worth: half of the longest walk's, but 32 tiles
    sp.each = (int)(longest / (2 * sp.parts));
    sp.each = sp.each > 32 ? sp.each : 32;
    // sinks that are seen from behind the window of their block; 4 tiles of 32 rows
    // for each of four wavefronts
    sp.far = 0;
    sp.far_parts = 1;
    const int64_t behind = (int64_t)pr.L - 127 - pr.W;
    if (masked == kUnmasked && pr.S > 0 && behind > 0) {
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

inline int64_t bwd_floats(const SlidingProblem &pr, const WalkSplit &sp) {
    const int DP = (pr.D + 31) / 32 * 32;
    return sp.part_at + (sp.parts > 1 ? (int64_t)pr.B * pr.Hk * sp.blocks * sp.parts * 128 * DP * 2 : 0);
}

template <typename X, typename T, int DP>
hipError_t forward(const typename X::Sliding &pr, hipStream_t s) {
    const int blocks = (pr.L * pr.G + 127) / 128;
    const unsigned grid = (unsigned)grid8((int64_t)pr.B * pr.Hk * blocks);
    if constexpr (X::kShaped && sizeof(T) == 2)
        if (pr.y_rest != nullptr) {
            sliding_fwd<X, T, DP, true><<<grid, 256, 0, s>>>(pr, blocks);
            return hipGetLastError();
        }
    sliding_fwd<X, T, DP, false><<<grid, 256, 0, s>>>(pr, blocks);
    return hipGetLastError();
}
// Whether dS of scores that are not capped goes into dq as two values.  Errors of dq as
// multiples of rounded results', one value and two, by the window of 1280 tokens: 2 keys 1.51 and
// 1.12, 8 1.47 and 1.06, 16 and more 1.45 and 1.04; heads of 8 channels 1.55 and 1.06 at any
// window.  Cost of two, 2 x 4096 tokens, 16 heads over 4, bf16: up to windows of 128 keys none that
// shows in a call (60 us from Python), 10% of the pass at 512, 16% at 1024 (128 channels), 7% at 1024
// (32).  So windows below 64 keys and heads of up to 32 channels have them.  Documents have them for the short ones that
// may be among them, whose lengths the device alone knows (of 4 tokens 1.50 and 1.10; of 600
// 1.45 and 1.03, at 12%).
inline bool few_keys(const SlidingProblem &pr) { return (pr.W < pr.L ? pr.W : pr.L) < 64; }
inline bool few_keys(const ShapedSlidingProblem &pr) {
    return pr.shape.places != nullptr || pr.D <= 32 || few_keys(static_cast<const SlidingProblem &>(pr));
}
template <typename X, typename T, int DP>
hipError_t backward(const typename X::Sliding &pr, const WalkSplit &sp, hipStream_t s) {
    const int blocks = (pr.L * pr.G + 127) / 128;
    const unsigned grid = (unsigned)grid8((int64_t)pr.B * pr.Hk * blocks);
    constexpr bool HALF = X::kShaped && sizeof(T) == 2;
    if (HALF && (X::kCap || few_keys(pr))) sliding_dq<X, T, DP, HALF><<<grid, 256, 0, s>>>(pr, blocks);
    else sliding_dq<X, T, DP, HALF && X::kCap><<<grid, 256, 0, s>>>(pr, blocks);
    if (pr.dk != nullptr) {
        const int64_t units = (int64_t)pr.B * pr.Hk;
        if (sp.far > 0) sliding_dkdv_far<X, T, DP><<<(unsigned)(units * sp.far * sp.far_parts), 256, 0, s>>>(pr, sp);
        const int64_t walks = X::kShaped ? grid8(units * sp.blocks) * sp.parts : grid8(units * sp.blocks * sp.parts);
        // A signal of one block of keys: P and dS in two values (KeySums).  Its gradients are
        // sums of few terms, and rounded ones gave some a dk 1.8 times as far off as where
        // results alone are rounded, where longer signals have 1.45; a launch's time hides it.
        if (HALF && pr.L <= 128) sliding_dkdv<X, T, DP, HALF><<<(unsigned)walks, 256 * BwdShape<T, DP>::NG, 0, s>>>(pr, sp);
        else sliding_dkdv<X, T, DP, false><<<(unsigned)walks, 256 * BwdShape<T, DP>::NG, 0, s>>>(pr, sp);
        if (sp.parts > 1) sliding_dkdv_join<X, T, DP><<<(unsigned)(units * ((pr.L + 31) / 32)), 256, 0, s>>>(pr, sp);
    }
    return hipGetLastError();
}
template <typename X, int DT>
hipError_t forward_type(const typename X::Sliding &pr, hipStream_t s) {
    typedef typename Elem<DT>::T T;
    return pr.D <= 32 ? forward<X, T, 32>(pr, s)
                      : pr.D <= 64 ? forward<X, T, 64>(pr, s)
                                   : pr.D <= 96 ? forward<X, T, 96>(pr, s) : forward<X, T, 128>(pr, s);
}
template <typename X, int DT>
hipError_t backward_type(const typename X::Sliding &pr, const WalkSplit &sp, hipStream_t s) {
    typedef typename Elem<DT>::T T;
    return pr.D <= 32 ? backward<X, T, 32>(pr, sp, s)
                      : pr.D <= 64 ? backward<X, T, 64>(pr, sp, s)
                                   : pr.D <= 96 ? backward<X, T, 96>(pr, sp, s) : backward<X, T, 128>(pr, sp, s);
}
template <typename X>
hipError_t forward_of(const typename X::Sliding &pr, hipStream_t s) {
    return pr.dtype == CIRCATT_F32 ? forward_type<X, 0>(pr, s)
                                   : pr.dtype == CIRCATT_F16 ? forward_type<X, 2>(pr, s) : forward_type<X, 3>(pr, s);
}
template <typename X>
hipError_t backward_of(const typename X::Sliding &pr, const WalkSplit &sp, hipStream_t s) {
    return pr.dtype == CIRCATT_F32 ? backward_type<X, 0>(pr, sp, s)
                                   : pr.dtype == CIRCATT_F16 ? backward_type<X, 2>(pr, sp, s) : backward_type<X, 3>(pr, sp, s);
}
inline int64_t threads_of(const SlidingProblem &pr, const WalkSplit &sp, bool backward) {
    const int64_t units = (int64_t)pr.B * pr.Hk, rows = 256 * grid8(units * (((int64_t)pr.L * pr.G + 127) / 128));
    if (!backward) return rows;
    // 512 threads, but 256 for some Float32 heads
    const int64_t keys = 512 * grid8(units * sp.blocks) * sp.parts, far = 256 * units * sp.far * sp.far_parts;
    const int64_t join = sp.parts > 1 ? 256 * units * ((pr.L + 31) / 32) : 0;
    int64_t most = rows;
    for (int64_t n : {keys, far, join}) most = n > most ? n : most;
    return most;
}

}  // namespace
}  // namespace circatt
