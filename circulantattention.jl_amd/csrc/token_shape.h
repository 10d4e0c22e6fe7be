// What a row of token attention sees, and how a score follows from a product
// <q, k>.  Two kinds: plain (a causal window with sinks, scores proportional to the
// products), and shaped, which adds
//   a cap:       x -> cap tanh(x / cap), x = scale <q, k>
//   slopes:      - slope_h |i - j| for the query at i and the key at j, behind the cap
//   documents:   row i sees nothing before the first token of its document, whose
//                sinks are the first tokens of it
//   a prefix:    the first tokens of a signal are seen by all of its rows
// Kernels take the kind as a template argument; the plain one adds nothing to them.
//
// Scores count in powers of two (log2(e) times as much), as the exponentials do.
#pragma once

#include "token_tile.h"

namespace circatt {
namespace tok {

constexpr float kLog2e = 1.4426950408889634f;

// The tangent from a product.  With E = exp(2 x d) and r = 1 / (1 + E) it is 1 - 2 r, off
// by some 2^-23 of the cap throughout, at one exponential, one reciprocal and three
// other instructions.  Where no product of a tile passes 0.7 / x, as in a model that
// keeps its scores well below the cap, a series of five terms with the same error takes
// six multiplications instead, and where none passes 0.3 / x one of three terms four.
// Of caps above 256 the series are for scores of the size that those arguments have under
// 256: a series then puts a score off by 1e-4 at most.
// Float32, and caps above 256 outside the series' range, ask for more:
// there arguments below 0.35 take the power series up to the eleventh term, whose next
// is 2^-26 of it.
__device__ __forceinline__ float curve_rest(const Curve &c, float dot) {
    return __builtin_amdgcn_rcpf(__builtin_amdgcn_exp2f(dot * c.u) + 1.f);
}
__device__ __forceinline__ float curve_power(float a) {
    const float b = a * a;
    float p = -1382.f / 155925.f;
    p = fmaf(p, b, 62.f / 2835.f);
    p = fmaf(p, b, -17.f / 315.f);
    p = fmaf(p, b, 2.f / 15.f);
    p = fmaf(p, b, -1.f / 3.f);
    return fmaf(a * b, p, a);
}
__device__ __forceinline__ float curve_fine(const Curve &c, float dot) {
    const float a = dot * c.x, small = curve_power(a);
    return fabsf(a) < 0.35f ? small : fmaf(-2.f, curve_rest(c, dot), 1.f);
}
// A tangent with its derivative 1 - t^2 by the argument.  Formed of t that would be what
// t's rounding left (off by a third of a per cent at 7, by all of it at 9); with r of |d|
// it is 4 r (1 - r), as exact as r wherever t lies.
struct Bent {
    float t, bend;
};
__device__ __forceinline__ Bent curve_bent(const Curve &c, float dot) {
    const float twice = 2.f * curve_rest(c, fabsf(dot)), t = 1.f - twice;
    return Bent{copysignf(t, dot), fmaf(twice, t, twice)};
}
__device__ __forceinline__ Bent curve_fine_bent(const Curve &c, float dot) {
    const float a = dot * c.x, small = curve_power(a);
    const Bent far = curve_bent(c, dot);
    return Bent{fabsf(a) < 0.35f ? small : far.t, far.bend};
}
template <int N>
__device__ __forceinline__ float curve_series(const float (&p)[N], float dot) {
    const float b = dot * dot;
    float t = p[N - 1];
#pragma unroll
    for (int i = N - 2; i >= 0; --i) t = fmaf(t, b, p[i]);
    return dot * t;
}

// ---------------------------------------------------------------------------
// One row, and the rows of one key, for the row by row forms.
struct PlainView {
    int begin, head, lo, end;  // keys [begin, head) and [lo, end) are looked at
    float c;
    __device__ __forceinline__ PlainView(int pos, int W, int S, float c)
        : begin(0), head(S), lo(pos - W + 1 > 0 ? pos - W + 1 : 0), end(pos + 1), c(c) {}
    __device__ __forceinline__ bool sees(int j) const { return j < end && (j < head || j >= lo); }
    __device__ __forceinline__ float score(float dot, int) const { return c * dot; }
    __device__ __forceinline__ float bend(float) const { return 1.f; }
};

// A product's score at a distance, and its derivative by the uncapped one.
struct ShapedScore {
    Curve curve;
    float c, slope;  // slope: of the head, times log2(e)
    bool cap;
    __device__ __forceinline__ float at(float dot, int back) const {
        const float s = cap ? curve.C * curve_fine(curve, dot) : c * dot;
        return fmaf(-slope, fabsf((float)back), s);
    }
    __device__ __forceinline__ float bend(float dot) const { return cap ? curve_bent(curve, dot).bend : 1.f; }
};
struct ShapedView {
    int pos, start, begin, head, lo, end, S, P;
    ShapedScore s;
    __device__ __forceinline__ ShapedView(int pos, int start, int W, int S, int P, const ShapedScore &s)
        : pos(pos), start(start), begin(P > 0 ? 0 : start), S(S), P(P), s(s) {
        head = start + S > P ? start + S : P;
        lo = pos - W + 1 > start ? pos - W + 1 : start;
        end = pos + 1 > P ? pos + 1 : P;
    }
    __device__ __forceinline__ bool sees(int j) const {
        return j < P || (j <= pos && j >= start && (j < start + S || j >= lo));
    }
    __device__ __forceinline__ float score(float dot, int j) const { return s.at(dot, pos - j); }
    __device__ __forceinline__ float bend(float dot) const { return s.bend(dot); }
};

// ---------------------------------------------------------------------------
// What rows see, by tiles of keys.  Rows of documents have their own first key
// (start; slo and shi: the first and the last row's, which ascend).
struct ShapedSight {
    int W, S, P, start, slo, shi;
    // of the keys k0 .. k0 + 31, a bit each
    __device__ __forceinline__ uint32_t bits(int at, int k0) const {
        const int end = at + 1 - k0, first = start - k0;
        const int low = end - W > first ? end - W : first, sinks = first + S;
        return bits_between(low, end) | bits_between(first, end < sinks ? end : sinks) |
               (at >= 0 ? bits_between(0, P - k0) : 0u);
    }
    // (The sinks of documents that begin among the rows lie in their windows' tiles.)
    __device__ __forceinline__ bool none(int lo, int hi, int k0, int n) const {
        return k0 >= P && (k0 > hi || k0 + n <= slo || (k0 + n - 1 <= lo - W && k0 >= slo + S));
    }
    __device__ __forceinline__ bool all(int lo, int hi, int k0, int n) const {
        return k0 + n <= P || (k0 + n - 1 <= lo && k0 >= shi && (k0 > hi - W || k0 + n <= slo + S));
    }
};

// The tiles of KT keys that rows at [lo, hi] see, in order: those of the prefix or
// of the sinks of the first row's document, which begins at s0, then the window's.
template <int KT>
struct ShapedTiles {
    int from, sinks, first, count;
    __device__ ShapedTiles(int lo, int hi, int W, int S, int P, int s0) {
        const int low = lo - W + 1 > s0 ? lo - W + 1 : s0, top = s0 + S > P ? s0 + S : P;
        const int w = low > 0 ? low / KT : 0, e = (hi + 1 > P ? hi + 1 : P) - 1;
        from = P > 0 ? 0 : s0 / KT;
        const int s = S > 0 || P > 0 ? (top + KT - 1) / KT : 0, to = s < w ? s : w;
        sinks = to > from ? to - from : 0;
        first = w;
        count = hi < 0 ? 0 : sinks + e / KT + 1 - w;
    }
    __device__ __forceinline__ int key(int i) const { return (i < sinks ? from + i : first + i - sinks) * KT; }
};

// ---------------------------------------------------------------------------
// Scores of 32 rows, one a lane, over blocks of 32 keys: registers hold the
// products and then the scores.
// Where the sum l of a row's weights is small, as it may be under a fixed reference
// (ShapedScorer), weighted values below 2^-126 are lost, n 2^-126 of n keys' sum at most.
// Channels whose sum is below this become NaN, as those are marked that are formed again:
// 2^-13 of one could be lost of 8192 keys.  (All such rows formed again: 2048 tokens, 32 heads of
// 128 over 8, cap 60 and scores about -40, 5.9 ms instead of 0.08.)
template <bool CAP>
__device__ __forceinline__ float out_of_reach(float l) {
    return CAP && l < 0x1p-20f ? 0x1p-100f : 0.f;
}

struct PlainScorer {
    float c;
    __device__ __forceinline__ float factor() const { return c; }
    __device__ __forceinline__ float unit() const { return c; }
    // The rows' largest scores of a tile (first: the first that is looked at), and what
    // follows of them for the reference of the exponentials.
    template <int NB, typename R>
    __device__ __forceinline__ float largest(R &x, const f16v (&s)[NB], bool) const {
        return x.largest(s) * c;
    }
    template <typename R>
    __device__ __forceinline__ void raise(R &x, float most) const {
        x.raise(most);
    }
    template <int NB>
    __device__ __forceinline__ void shape(f16v (&)[NB], int, int, int, int) const {}
    template <int NB, typename R>
    __device__ __forceinline__ void lowered(const R &, f16v (&)[NB], int, int, int, int) const {}
    template <int NB, typename R, typename P>
    __device__ __forceinline__ void weigh(R &x, f16v (&s)[NB], P &p, bool) const {
        x.raise(x.largest(s) * c);
        x.weigh(s, p, c);
    }
};
// ANEW: the kernel's first argument, from which the curve is read for every tile where
// its numbers would take more scalar registers through a loop than there are; or void.
struct KeptCurve {
    Curve kept;
    __device__ __forceinline__ explicit KeptCurve(const Curve &c) : kept(c) {}
    __device__ __forceinline__ Curve get() const { return kept; }
};
template <typename P>
struct ReadCurve {
    __device__ __forceinline__ explicit ReadCurve(const Curve &) {}
    __device__ __forceinline__ Curve get() const { return argument_again<P>().shape.curve; }
};
template <bool CAP, bool FINE, typename From = KeptCurve>
struct ShapedScorer {
    From from;
    float c, C, slope;
    bool biased;
    // Scores lie below the cap, and a row's own token's, which no bias takes anything off,
    // above its negative.  Where probabilities are rounded to BFloat16, the largest score of
    // the first tile alone is the softmax's reference then, or C - 100 if that is more:
    // weights stay below 2^100, their sum below 2^124, and that of the row's own token, or
    // of the first tile's best, above 2^(100 - 2 C).  (Rows whose sums of values pass Float32
    // so, or of values too small for their weights, are formed again: out_of_reach.  Float16 does
    // not hold such weights, and exponents of some 100 are off by 2^-18, ten times the rest of
    // a Float32 signal's error.)  `wide`: that type, and rows that all see their own token.
    bool bounded;
    __device__ __forceinline__ ShapedScorer(float scale, const Curve &curve, float slope, bool biased, bool wide)
        : from(curve), c(scale * kLog2e), C(curve.C), slope(slope), biased(biased),
          bounded(CAP && wide && curve.C <= 90.f && __all(slope >= 0.f)) {}
    template <int NB, typename R>
    __device__ __forceinline__ float largest(R &x, const f16v (&s)[NB], bool first) const {
        if (CAP && bounded && !first) return 0.f;
        const float most = x.largest(s) * factor();
        if (CAP && bounded) x.m = fmaxf(most, C - 100.f);
        return most;
    }
    template <typename R>
    __device__ __forceinline__ void raise(R &x, float most) const {
        if (!(CAP && bounded)) x.raise(most);
    }
    // What the registers still lack to scores in powers of two: they hold products, or
    // tangents of capped ones, and where there are slopes the scores themselves.
    __device__ __forceinline__ float unit() const { return CAP ? C : c; }
    __device__ __forceinline__ float factor() const { return biased ? 1.f : unit(); }
    // Tangents in the place of products: all by the series, or all by the exponential.
    // (The products pass through an empty asm on each side, or the compiler forms all
    // sides before the branch.)
    template <int NB, typename F>
    __device__ __forceinline__ static void each(f16v (&s)[NB], F f) {
#pragma unroll
        for (int n = 0; n < NB; ++n) asm volatile("" : "+v"(s[n]));
#pragma unroll
        for (int n = 0; n < NB; ++n)
#pragma unroll
            for (int i = 0; i < 16; ++i) s[n][i] = f(s[n][i], (float)(32 * n + 8 * (i >> 2) + (i & 3)));
    }
    template <int NB>
    __device__ __forceinline__ void caps(f16v (&s)[NB]) const {
        if constexpr (!CAP) return;
        const Curve curve = from.get();
        if constexpr (CAP && FINE) {
            each(s, [&](float d, float) { return curve_fine(curve, d); });
        } else if constexpr (CAP) {
            float most = 0.f;
#pragma unroll
            for (int n = 0; n < NB; ++n)
#pragma unroll
                for (int i = 0; i < 16; ++i) most = fmaxf(most, fabsf(s[n][i]));
            if (!__any(most > curve.near)) each(s, [&](float d, float) { return curve_series(curve.few, d); });
            else if (!__any(most > curve.far)) each(s, [&](float d, float) { return curve_series(curve.more, d); });
            else if (curve.fine) each(s, [&](float d, float) { return curve_fine(curve, d); });
            else each(s, [&](float d, float) { return fmaf(-2.f, curve_rest(curve, d), 1.f); });
        }
    }
    // The same, with the tangents' derivatives by their arguments.
    template <typename F>
    __device__ __forceinline__ static void each_bent(f16v &s, f16v &bend, F f) {
        asm volatile("" : "+v"(s));
#pragma unroll
        for (int i = 0; i < 16; ++i) {
            const Bent b = f(s[i]);
            s[i] = b.t;
            bend[i] = b.bend;
        }
    }
    template <int N>
    __device__ __forceinline__ static Bent series_bent(const float (&p)[N], float d) {
        const float t = curve_series(p, d);
        return Bent{t, fmaf(-t, t, 1.f)};
    }
    __device__ __forceinline__ void caps(f16v &s, f16v &bend) const {
        const Curve curve = from.get();
        if constexpr (FINE) {
            each_bent(s, bend, [&](float d) { return curve_fine_bent(curve, d); });
        } else {
            float most = 0.f;
#pragma unroll
            for (int i = 0; i < 16; ++i) most = fmaxf(most, fabsf(s[i]));
            if (!__any(most > curve.near)) each_bent(s, bend, [&](float d) { return series_bent(curve.few, d); });
            else if (!__any(most > curve.far)) each_bent(s, bend, [&](float d) { return series_bent(curve.more, d); });
            else if (curve.fine) each_bent(s, bend, [&](float d) { return curve_fine_bent(curve, d); });
            else each_bent(s, bend, [&](float d) { return curve_bent(curve, d); });
        }
    }
    // Register i of block n is key k0 + 32 n + 8 (i / 4) + 4 half + i % 4; lo: the
    // first row's position, behind which a key's distance may count the other way.
    template <int NB>
    __device__ __forceinline__ void biases(f16v (&s)[NB], int k0, int at, int lo, int lane) const {
        if (biased) bias(s, k0 + 4 * (lane >> 5) - at, k0 + 32 * NB - 1 <= lo);
    }
    template <int NB>
    __device__ __forceinline__ void bias(f16v (&s)[NB], int ahead, bool before) const {
        const float f = unit();
        if (before) {  // distances as they are: keys do not lie behind their rows
            const float b = slope * (float)ahead;
#pragma unroll
            for (int n = 0; n < NB; ++n)
#pragma unroll
                for (int i = 0; i < 16; ++i)
                    s[n][i] = fmaf(s[n][i], f, fmaf(slope, (float)(32 * n + 8 * (i >> 2) + (i & 3)), b));
        } else {
            const float d = (float)ahead;
#pragma unroll
            for (int n = 0; n < NB; ++n)
#pragma unroll
                for (int i = 0; i < 16; ++i)
                    s[n][i] = fmaf(-slope, fabsf(d + (float)(32 * n + 8 * (i >> 2) + (i & 3))), s[n][i] * f);
        }
    }
    template <int NB>
    __device__ __forceinline__ void shape(f16v (&s)[NB], int k0, int at, int lo, int lane) const {
        caps(s);
        biases(s, k0, at, lo, lane);
    }
    // Exponents: the scores less `by`, which costs nothing behind a bias.
    template <int NB>
    __device__ __forceinline__ void exponents(f16v (&s)[NB], int k0, int at, int lo, int lane, float by) const {
        const float f = unit(), ahead = (float)(k0 + 4 * (lane >> 5) - at);
        if (!biased) {
            each(s, [&](float d, float) { return fmaf(d, f, -by); });
        } else if (k0 + 32 * NB - 1 <= lo) {
            const float b = fmaf(slope, ahead, -by);
            each(s, [&](float d, float k) { return fmaf(d, f, fmaf(slope, k, b)); });
        } else {
            each(s, [&](float d, float k) { return fmaf(-slope, fabsf(ahead + k), fmaf(d, f, -by)); });
        }
    }
    // A tile's products to what its weights are formed from, hidden ones -inf by then, and
    // those to weights; first: of the first tile that is looked at.  Capped scores go by
    // exponents: chunks with cap, slopes and prefixes 167 us, 146 so.  Others have no
    // reason to (128 us instead of 124), and in sliding_fwd, which has a tile more in
    // registers, exponents spill (8192 tokens 563 us instead of 483).
    template <int NB, typename R>
    __device__ __forceinline__ void lowered(const R &x, f16v (&s)[NB], int k0, int at, int lo, int lane) const {
        caps(s);
        if constexpr (CAP) exponents(s, k0, at, lo, lane, x.reference());
        else biases(s, k0, at, lo, lane);
    }
    template <int NB, typename R>
    __device__ __forceinline__ float largest_lowered(R &x, f16v (&s)[NB], bool first) const {
        if (bounded && !first) return 0.f;
        const float most = x.largest(s);
        if (bounded) {
            x.m = fmaxf(most, C - 100.f);
            x.lower(s, x.m);
        }
        return most;
    }
    template <int NB, typename R, typename P>
    __device__ __forceinline__ void weigh(R &x, f16v (&s)[NB], P &p, bool first) const {
        if constexpr (CAP) {
            const float most = largest_lowered(x, s, first);
            if (!bounded) x.raise(s, most);
            x.weigh(s, p);
        } else {
            x.raise(largest(x, s, first));
            x.weigh(s, p, factor());
        }
    }
    // Exponents of one key's products (or tangents) with 32 rows, a row a register: the rows'
    // logarithms of sums lie at LDS byte st, their slopes and tokens 2 and 3 strides behind.
    __device__ __forceinline__ void exponents_of_rows(f16v &s, unsigned st, int stride, float token) const {
        const float f = unit();
#pragma unroll
        for (int i = 0; i < 16; i += 4) {
            const f4v ls = *(const CIRCATT_LDS f4v *)(st + 8 * i);
#pragma unroll
            for (int y = 0; y < 4; ++y) s[i + y] = fmaf(s[i + y], f, -ls[y]);
        }
        if (!biased) return;
#pragma unroll
        for (int i = 0; i < 16; i += 4) {
            const f4v sl = *(const CIRCATT_LDS f4v *)(st + 2 * stride + 8 * i);
            const f4v at = *(const CIRCATT_LDS f4v *)(st + 3 * stride + 8 * i);
#pragma unroll
            for (int y = 0; y < 4; ++y) s[i + y] = fmaf(-sl[y], fabsf(at[y] - token), s[i + y]);
        }
    }
};

// ---------------------------------------------------------------------------
// The kinds.
struct Plain {
    typedef SlidingProblem Sliding;
    typedef PagedProblem Paged;
    static constexpr bool kShaped = false, kCap = false;
};
template <bool CAP>
struct Shaped {
    typedef ShapedSlidingProblem Sliding;
    typedef ShapedPagedProblem Paged;
    static constexpr bool kShaped = true, kCap = CAP;
};

__device__ __forceinline__ int clamp_prefix(const int32_t *prefix, int b, int n) {
    const int p = prefix == nullptr ? 0 : prefix[b];
    return p < 0 ? 0 : p < n ? p : n;
}
// The first token of token t's document, from its place in it.
__device__ __forceinline__ int document_start(const int32_t *places, int t) {
    if (places == nullptr) return 0;
    const int p = places[t];
    return p <= 0 ? t : p < t ? t - p : 0;
}

}  // namespace tok
}  // namespace circatt
