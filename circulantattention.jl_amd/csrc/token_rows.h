// Token attention row by row: one wavefront forms one row of an output from
// the rows that it sees and reads no other, lane l holding channels l and
// l + 64.  Every visible key is one step of the running softmax; all sums are
// Float32.
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
// x minus x rounded to T, 0 where that is not finite.
template <typename T>
__device__ __forceinline__ T rounding_rest(float x) {
    const float e = x - (float)(T)x;
    return fabsf(e) < INFINITY ? (T)e : (T)0.f;
}
__device__ __forceinline__ float wave_sum(float x) {
    for (int m = 32; m; m >>= 1) x += __shfl_xor(x, m, 64);
    return x;
}
__device__ __forceinline__ float dot(Pair x, Pair y) { return wave_sum(x.a * y.a + x.b * y.b); }

// y = sum_j softmax_j(c q.k_j) v_j in base 2 over [0, min(S, lo)) and [lo, pos],
// lo = max(0, pos - W + 1).  kv.row(j): whether key j is there, and its rows.
// rest: what y's rounding took, or NULL.
template <typename T, typename KV>
__device__ void forward_row(const T *q, T *y, T *rest, const KV &kv, int pos, int W, int S, int D,
                            float c) {
    const int lane = threadIdx.x & 63;
    const Pair qr = load_row(q, lane, D);
    const int lo = pos - W + 1 > 0 ? pos - W + 1 : 0;
    float m = -INFINITY, l = 0.f;
    Pair o{0.f, 0.f};
    for (int j = 0; j <= pos; ++j) {
        if (j >= S && j < lo) j = lo;
        const T *kp, *vp;
        if (!kv.row(j, kp, vp)) continue;
        const float t = c * dot(qr, load_row(kp, lane, D));
        const float mn = fmaxf(m, t), mu = mn == -INFINITY ? 0.f : mn;
        const float r = __builtin_amdgcn_exp2f(m - mu), p = __builtin_amdgcn_exp2f(t - mu);
        const Pair vr = load_row(vp, lane, D);
        l = l * r + p;
        o.a = o.a * r + p * vr.a;
        o.b = o.b * r + p * vr.b;
        m = mn;
    }
    const float inv = l == 0.f ? 0.f : 1.f / l;
    store_row(y, lane, D, Pair{o.a * inv, o.b * inv});
    if (rest != nullptr)
        store_row(rest, lane, D, Pair{(float)rounding_rest<T>(o.a * inv), (float)rounding_rest<T>(o.b * inv)});
}

// The gradient of row i's query: dq = scale sum_j p_j (<dy, v_j> - d) k_j with
// p_j = exp2(c q.k_j - lse) and d = <dy, y + rest> (rest may be NULL), which is
// stored too.
template <typename T, typename KV>
__device__ void dq_row(const T *q, const T *y, const T *rest, const T *dy, T *dq, float lse, float *dsum, const KV &kv,
                       int pos, int W, int S, int D, float c, float scale) {
    const int lane = threadIdx.x & 63;
    const Pair qr = load_row(q, lane, D), gr = load_row(dy, lane, D);
    Pair yr = load_row(y, lane, D);
    if (rest != nullptr) {
        const Pair e = load_row(rest, lane, D);
        yr.a += e.a;
        yr.b += e.b;
    }
    const float d = dot(gr, yr);
    if (lane == 0) *dsum = d;
    const int lo = pos - W + 1 > 0 ? pos - W + 1 : 0;
    Pair o{0.f, 0.f};
    for (int j = 0; j <= pos; ++j) {
        if (j >= S && j < lo) j = lo;
        const T *kp, *vp;
        if (!kv.row(j, kp, vp)) continue;
        const Pair kr = load_row(kp, lane, D);
        const float p = __builtin_amdgcn_exp2f(c * dot(qr, kr) - lse);
        const float ds = p * (dot(gr, load_row(vp, lane, D)) - d);
        o.a += ds * kr.a;
        o.b += ds * kr.b;
    }
    store_row(dq, lane, D, Pair{o.a * scale, o.b * scale});
}

// The gradients of key j and value j over the queries i of [j, j + W) (j < S:
// all from j on) below n, and the G heads of each: q and dy point at head 0 of
// query 0 of the group, lse and dsum at its row 0.
template <typename T>
__device__ void dkdv_row(const T *k, const T *v, const T *q, int64_t q_row, const T *dy, int64_t dy_row,
                         const float *lse, const float *dsum, T *dk, T *dv, int j, int n, int W, int S, int G,
                         int D, float c, float scale) {
    const int lane = threadIdx.x & 63;
    const Pair kr = load_row(k, lane, D), vr = load_row(v, lane, D);
    const int end = j < S || n - j < W ? n : j + W;
    Pair ok{0.f, 0.f}, ov{0.f, 0.f};
    for (int i = j; i < end; ++i)
        for (int g = 0; g < G; ++g) {
            const Pair qr = load_row(q + i * q_row + g * D, lane, D), gr = load_row(dy + i * dy_row + g * D, lane, D);
            const int64_t r = (int64_t)i * G + g;
            const float p = __builtin_amdgcn_exp2f(c * dot(qr, kr) - lse[r]);
            const float ds = p * (dot(gr, vr) - dsum[r]);
            ov.a += p * gr.a;
            ov.b += p * gr.b;
            ok.a += ds * qr.a;
            ok.b += ds * qr.b;
        }
    store_row(dk, lane, D, Pair{ok.a * scale, ok.b * scale});
    store_row(dv, lane, D, ov);
}

// Keys and values of a contiguous signal, and of a paged cache (page numbers
// outside the cache are never read: their tokens are hidden).
template <typename T>
struct SignalKV {
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
