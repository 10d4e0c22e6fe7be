// Token attention row by row: one wavefront forms one row of an output from
// the rows that it sees and reads no other.  They are taken 64 at a time: every
// lane forms the scores of one of them by itself, and the sums run over the 64 with
// lane l holding channels l and l + 64 of the output.  All sums are Float32.
//
// These are for rows that the matrix products have spoilt, a few in a call: zero
// weights times values that are not finite, and score gradients that Float16 cannot
// hold.  They write the channels alone that are not finite as they stand, and end
// as soon as every one of those has met a value that makes it so: what is left
// cannot take that back.  (Which of the infinities or NaN a channel is that sees
// several of them may then hang on the first ones alone.)  A training step of 4096
// tokens, 8 heads of 64 over 4, Float16, no window, takes 0.26 ms, with dy NaN
// throughout 0.53, with one infinity in it 2.6: the chain of 64 rows' loads that the
// keys beside that row's tiles walk.
#pragma once

#include "token_kernels.h"

namespace circatt {
namespace tok {

template <int DT>
struct Elem;
template <>
struct Elem<0> {
    typedef float T;
};
template <>
struct Elem<2> {
    typedef _Float16 T;
};
template <>
struct Elem<3> {
    typedef __bf16 T;
};

template <typename T>
using V8 = T __attribute__((ext_vector_type(8)));
typedef float f4v __attribute__((ext_vector_type(4)));

// Eight channels from global memory, zero from channel D on (D a multiple of 8).
template <typename T>
__device__ __forceinline__ V8<T> load8(const T *p, int d, int D) {
    V8<T> v{};
    if (d < D) {
        if constexpr (sizeof(T) == 2) {
            v = *reinterpret_cast<const V8<T> *>(p + d);
        } else {
            const f4v a = *reinterpret_cast<const f4v *>(p + d), b = *reinterpret_cast<const f4v *>(p + d + 4);
            v = V8<T>{a[0], a[1], a[2], a[3], b[0], b[1], b[2], b[3]};
        }
    }
    return v;
}

__device__ __forceinline__ bool is_finite(float x) { return fabsf(x) < INFINITY; }

// The lane's number formed anew, for what follows a loop whose registers are full: no
// address that hangs on it is kept through the loop.
__device__ __forceinline__ int lane_again() {
    int lane = __builtin_amdgcn_mbcnt_hi(~0u, __builtin_amdgcn_mbcnt_lo(~0u, 0u));
    asm volatile("" : "+v"(lane));
    return lane;
}

struct Pair {
    float a, b;
};
template <typename T>
__device__ __forceinline__ Pair load_row(const T *p, int lane, int D) {
    return Pair{lane < D ? (float)p[lane] : 0.f, lane + 64 < D ? (float)p[lane + 64] : 0.f};
}
template <typename T>
__device__ __forceinline__ void store_row(T *p, int lane, int D, Pair v) {
    if (lane < D) p[lane] = (T)v.a;
    if (lane + 64 < D) p[lane + 64] = (T)v.b;
}

// The channels of an output's row that are not finite as they stand.
struct Lacks {
    bool a, b;
    template <typename T>
    __device__ __forceinline__ Lacks(const T *p, int lane, int D) {
        const Pair v = load_row(p, lane, D);
        a = !is_finite(v.a);
        b = !is_finite(v.b);
    }
    __device__ __forceinline__ bool open(Pair sum) const { return (a && is_finite(sum.a)) || (b && is_finite(sum.b)); }
    template <typename T>
    __device__ __forceinline__ void store(T *p, int lane, Pair v) const {
        if (a) p[lane] = (T)v.a;
        if (b) p[lane + 64] = (T)v.b;
    }
};
// What x (to `exact`, a value nearer to the one meant) lacks when rounded to T, 0 where
// that is not finite.
template <typename T>
__device__ __forceinline__ T rounding_rest(float x, float exact) {
    const float e = exact - (float)(T)x;
    return fabsf(e) < INFINITY ? (T)e : (T)0.f;
}
template <typename T>
__device__ __forceinline__ T rounding_rest(float x) {
    return rounding_rest<T>(x, x);
}
__device__ __forceinline__ float wave_sum(float x) {
    for (int m = 32; m; m >>= 1) x += __shfl_xor(x, m, 64);
    return x;
}
__device__ __forceinline__ float wave_max(float x) {
    for (int m = 32; m; m >>= 1) x = fmaxf(x, __shfl_xor(x, m, 64));
    return x;
}
__device__ __forceinline__ float dot(Pair x, Pair y) { return wave_sum(x.a * y.a + x.b * y.b); }
__device__ __forceinline__ float lane_of(float x, int lane) {
    return __builtin_bit_cast(float, __builtin_amdgcn_readlane(__builtin_bit_cast(int, x), lane));
}
#define CIRCATT_GLOBAL __attribute__((address_space(1)))
template <typename T>
__device__ __forceinline__ const CIRCATT_GLOBAL T *lane_of(const T *p, int lane) {
    const uint64_t x = reinterpret_cast<uint64_t>(p);
    const uint32_t lo = __builtin_amdgcn_readlane((int)(uint32_t)x, lane), hi = __builtin_amdgcn_readlane((int)(x >> 32), lane);
    return reinterpret_cast<const CIRCATT_GLOBAL T *>((uint64_t)hi << 32 | lo);
}
// Loads below are under no condition, which would make each wait for itself: what
// is not there reads something else in its place.
//
// <p, x> of every lane's own row p and one row x that the wavefront holds.  For whole
// wavefronts: under a condition, a lane that is left out has no part of x to read.
template <typename T>
__device__ __forceinline__ float lane_dot(const T *p, Pair x, int D) {
    constexpr int N = 4;
    float s = 0.f;
    for (int d = 0; d < D; d += 8 * N) {
        V8<T> v[N];
#pragma unroll
        for (int n = 0; n < N; ++n) v[n] = load8(p + (d + 8 * n < D ? d + 8 * n : 0), 0, 8);
#pragma unroll
        for (int n = 0; n < N; ++n)
            if (d + 8 * n < D) {
                const float xs = d < 64 ? x.a : x.b;
#pragma unroll
                for (int e = 0; e < 8; ++e) s = fmaf((float)v[n][e], lane_of(xs, (d & 63) + 8 * n + e), s);
                __builtin_amdgcn_sched_barrier(0);  // no more scalars at a time
            }
    }
    return s;
}
// o += sum over the lanes of their weight w times their row p (lanes without one: 0
// and zero_row, so that what o holds stays as it is).
__device__ const float kZeroRow[128] = {};
template <typename T>
__device__ __forceinline__ const T *zero_row() {
    return reinterpret_cast<const T *>(kZeroRow);
}
template <typename T>
__device__ __forceinline__ void add_rows(Pair &o, const T *p, float w, int lane, int D) {
    const int a = lane < D ? lane : D - 1, b = lane + 64 < D ? lane + 64 : D - 1;
#pragma unroll 8
    for (int i = 0; i < 64; ++i) {
        const CIRCATT_GLOBAL T *row = lane_of(p, i);
        const float wi = lane_of(w, i);
        o.a = fmaf(wi, (float)row[a], o.a);
        o.b = fmaf(wi, (float)row[b], o.b);
    }
}
// Whether one of the values that kv has for the keys [j0, j1) is not finite.
template <typename KV>
__device__ __forceinline__ bool bad_values(const KV &kv, int j0, int j1, int D) {
    bool bad = false;
    for (int j = j0 + lane_again(); j < j1; j += 64) {
        typename KV::Ptr kp, vp;
        if (!kv.row(j, kp, vp)) continue;
        for (int d = 0; d < D; d += 8) {
            const auto x = load8(vp, d, D);
#pragma unroll
            for (int e = 0; e < 8; ++e) bad |= !is_finite((float)x[e]);
        }
    }
    return __any(bad);
}

// Whether a row sees one of the keys that kv has.  (see, here and below: which keys the
// row sees, and their scores from the products: PlainView or ShapedView.)
template <typename KV, typename V>
__device__ __forceinline__ bool sees_any(const KV &kv, const V &see) {
    for (int j0 = see.begin; j0 < see.end; j0 += 64) {
        if (j0 >= see.head && j0 < see.lo) j0 = see.lo;
        const int j = j0 + lane_again();
        typename KV::Ptr kp, vp;
        if (__any(see.sees(j) && kv.row(j, kp, vp))) return true;
    }
    return false;
}

// y = sum_j softmax_j(score_j) v_j in base 2 over the keys that the row sees.
// kv.row(j): whether key j is there, and its rows.
// rest: what y's rounding took, or NULL.
template <typename T, typename KV, typename V>
__device__ void forward_row(const T *q, T *y, T *rest, const KV &kv, const V &see, int D) {
    const int lane = lane_again();
    const Pair qr = load_row(q, lane, D);
    const Lacks lacks(y, lane, D);
    float m = -INFINITY, l = 0.f;
    Pair o{0.f, 0.f};
    for (int j0 = see.begin; j0 < see.end; j0 += 64) {
        if (j0 >= see.head && j0 < see.lo) j0 = see.lo;
        const int j = j0 + lane;
        const T *kp = q, *vp = q;
        const bool sees = see.sees(j) && kv.row(j, kp, vp);
        if (!sees) kp = q, vp = zero_row<T>();
        const float score = see.score(lane_dot(kp, qr, D), j), t = sees ? score : -INFINITY;
        const float mn = fmaxf(m, wave_max(t)), mu = mn == -INFINITY ? 0.f : mn;
        const float r = __builtin_amdgcn_exp2f(m - mu), p = sees ? __builtin_amdgcn_exp2f(t - mu) : 0.f;
        l = l * r + wave_sum(p);
        o.a *= r;
        o.b *= r;
        m = mn;
        add_rows(o, vp, p, lane, D);
        if (!__any(lacks.open(o))) break;
    }
    const float inv = 1.f / l;
    lacks.store(y, lane, Pair{o.a * inv, o.b * inv});
    if (rest != nullptr)
        lacks.store(rest, lane, Pair{(float)rounding_rest<T>(o.a * inv), (float)rounding_rest<T>(o.b * inv)});
}

// The gradient of row i's query: dq = scale sum_j p_j (<dy, v_j> - d) k_j with
// p_j = exp2(score_j - lse) and d = <dy, y + rest> (rest may be NULL), which is
// stored too; capped scores bring their derivative.
template <typename T, typename KV, typename V>
__device__ void dq_row(const T *q, const T *y, const T *rest, const T *dy, T *dq, float lse, float *dsum, const KV &kv,
                       const V &see, int D, float scale) {
    const int lane = lane_again();
    const Pair qr = load_row(q, lane, D), gr = load_row(dy, lane, D);
    const Lacks lacks(dq, lane, D);
    Pair yr = load_row(y, lane, D);
    if (rest != nullptr) {
        const Pair e = load_row(rest, lane, D);
        yr.a += e.a;
        yr.b += e.b;
    }
    const float d = dot(gr, yr);
    if (lane == 0) *dsum = d;
    Pair o{0.f, 0.f};
    for (int j0 = see.begin; j0 < see.end; j0 += 64) {
        if (j0 >= see.head && j0 < see.lo) j0 = see.lo;
        const int j = j0 + lane;
        const T *kp = q, *vp = q;
        const bool sees = see.sees(j) && kv.row(j, kp, vp);
        if (!sees) kp = vp = zero_row<T>();
        const float x = lane_dot(kp, qr, D), p = __builtin_amdgcn_exp2f(see.score(x, j) - lse);
        const float ds = p * (lane_dot(vp, gr, D) - d) * see.bend(x);
        add_rows(o, kp, sees ? ds : 0.f, lane, D);
        if (!__any(lacks.open(o))) break;
    }
    lacks.store(dq, lane, Pair{o.a * scale, o.b * scale});
}

// The gradients of key j and value j (fix_k, fix_v: which) over the packed rows
// [first, end), G heads a token: q and dy point at head 0 of token 0 of the group, lse
// and dsum at its row 0.  see.score and see.bend as above, by row.
template <typename T, typename V>
__device__ void dkdv_row(const T *k, const T *v, const T *q, int64_t q_row, const T *dy, int64_t dy_row,
                         const float *lse, const float *dsum, T *dk, T *dv, bool fix_k, bool fix_v, int first, int end,
                         int G, int D, const V &see, float scale) {
    const int lane = lane_again();
    const Pair kr = load_row(k, lane, D), vr = load_row(v, lane, D);
    Lacks lk(dk, lane, D), lv(dv, lane, D);
    lk.a &= fix_k, lk.b &= fix_k;
    lv.a &= fix_v, lv.b &= fix_v;
    Pair ok{0.f, 0.f}, ov{0.f, 0.f};
    for (int r0 = first; r0 < end; r0 += 64) {
        const bool in = r0 + lane < end;
        const int r = in ? r0 + lane : end - 1, i = r / G, g = r - i * G;
        const T *qp = q + i * q_row + g * D, *gp = dy + i * dy_row + g * D;
        const float x = lane_dot(qp, kr, D), p = __builtin_amdgcn_exp2f(see.score(x, i, g) - lse[r]);
        const float ds = p * (lane_dot(gp, vr, D) - dsum[r]) * see.bend(x);
        if (fix_v) add_rows(ov, in ? gp : zero_row<T>(), in ? p : 0.f, lane, D);
        if (fix_k) add_rows(ok, in ? qp : zero_row<T>(), in ? ds : 0.f, lane, D);
        if (!__any(lk.open(ok) || lv.open(ov))) break;
    }
    lk.store(dk, lane, Pair{ok.a * scale, ok.b * scale});
    lv.store(dv, lane, ov);
}

// Keys and values of a contiguous signal, and of a paged cache (page numbers
// outside the cache are never read: their tokens are hidden).
template <typename T>
struct SignalKV {
    typedef const T *Ptr;
    const T *k, *v;
    int64_t k_row, v_row;
    __device__ __forceinline__ bool row(int j, const T *&kp, const T *&vp) const {
        kp = k + j * k_row;
        vp = v + j * v_row;
        return true;
    }
};
template <typename T>
struct PagedKV {
    typedef const T *Ptr;
    const T *k, *v;
    int64_t page_stride, row_stride;
    const int32_t *pages;  // of one sequence
    int npages, page_log2;
    __device__ __forceinline__ bool row(int j, const T *&kp, const T *&vp) const {
        const int pg = pages[j >> page_log2];
        const int64_t at = pg * page_stride + (j & ((1 << page_log2) - 1)) * row_stride;
        kp = k + at;
        vp = v + at;
        return (unsigned)pg < (unsigned)npages;
    }
};

}  // namespace tok
}  // namespace circatt
