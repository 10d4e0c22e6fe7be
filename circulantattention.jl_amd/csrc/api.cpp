// C-ABI layer of libcircatt: host-side validation (the reference's @assert
// checks, src/circulant.jl:65,87, src/similarity.jl:43-44,
// src/attention.jl:54,73, src/array.jl:133,142,180) and kernel dispatch.
// No entry point allocates device memory.
#include <hip/hip_runtime.h>

#include <atomic>
#include <cmath>
#include <cstdarg>
#include <cstdio>
#include <cstring>
#include <initializer_list>
#include <mutex>
#include <string>

#include "circatt.h"
#include "circatt_kernels.h"
#include "token_kernels.h"

using namespace circatt;

namespace circatt {
namespace {
std::atomic<int> g_math{CIRCATT_MATH_SPLIT_F16};
}
int math_mode() { return g_math.load(std::memory_order_relaxed); }
}  // namespace circatt

namespace {

thread_local std::string g_last_error;

int fail(int code, const char *fmt, ...) {
    char buf[512];
    va_list ap;
    va_start(ap, fmt);
    vsnprintf(buf, sizeof(buf), fmt, ap);
    va_end(ap);
    g_last_error = buf;
    return code;
}

int ok() {
    g_last_error.clear();
    return CIRCATT_OK;
}

int hip_result(hipError_t e, const char *what) {
    if (e == hipSuccess) return ok();
    if (e == hipErrorNotSupported)
        return fail(CIRCATT_ERR_UNSUPPORTED, "%s: shape not supported by the HIP kernels", what);
    return fail(CIRCATT_ERR_HIP, "%s: HIP error %d (%s)", what, (int)e, hipGetErrorString(e));
}

hipStream_t as_stream(void *s) { return reinterpret_cast<hipStream_t>(s); }

// Validates (nsp, n1, n2, ws) and fills g.  Returns 0 or an error code.
int check_geom(int nsp, int64_t n1, int64_t n2, int32_t ws, Geom &g) {
    if (nsp != 1 && nsp != 2) return fail(CIRCATT_ERR_INVALID, "nsp=%d must be 1 or 2", nsp);
    if (ws < 1 || ws % 2 != 1) return fail(CIRCATT_ERR_INVALID, "filter size M=%d must be odd.", ws);
    if (n1 < 1 || n1 > INT32_MAX) return fail(CIRCATT_ERR_INVALID, "invalid spatial size n1=%lld", (long long)n1);
    if (nsp == 2 && (n2 < 1 || n2 > INT32_MAX))
        return fail(CIRCATT_ERR_INVALID, "invalid spatial size n2=%lld", (long long)n2);
    if (nsp == 2 && (int64_t)ws * ws > INT32_MAX)
        return fail(CIRCATT_ERR_INVALID, "window %d too large", ws);
    g = make_geom(nsp, (int)n1, nsp == 2 ? (int)n2 : 1, ws);
    // colVal / rowPtr are Int32 (src/circulant.jl:64,86): P*K+1 must fit.
    if (g.P * (int64_t)g.K + 1 > INT32_MAX)
        return fail(CIRCATT_ERR_INVALID, "P*K = %lld exceeds the Int32 index range",
                    (long long)(g.P * (int64_t)g.K));
    return CIRCATT_OK;
}

int check_dtype(int dtype) {
    if (dtype != CIRCATT_F32 && dtype != CIRCATT_C32)
        return fail(CIRCATT_ERR_UNSUPPORTED, "dtype %d not supported (Float32 or ComplexF32)", dtype);
    return CIRCATT_OK;
}

int check_kind(int kind) {
    if (kind != CIRCATT_DOT && kind != CIRCATT_DISTANCE)
        return fail(CIRCATT_ERR_INVALID, "unknown similarity kind %d", kind);
    return CIRCATT_OK;
}

#define CIRCATT_TRY(expr)            \
    do {                             \
        int _rc = (expr);            \
        if (_rc != CIRCATT_OK) return _rc; \
    } while (0)

#define CIRCATT_NONNULL(p)                                                  \
    do {                                                                    \
        if ((p) == nullptr) return fail(CIRCATT_ERR_INVALID, "%s is NULL", #p); \
    } while (0)

}  // namespace

extern "C" {

int circatt_version(void) { return 10200; }

int circatt_set_math(int mode) {
    if (mode != CIRCATT_MATH_SPLIT_F16 && mode != CIRCATT_MATH_F32)
        return fail(CIRCATT_ERR_INVALID, "unknown math mode %d", mode);
    g_math.store(mode, std::memory_order_relaxed);
    return ok();
}

int circatt_get_math(void) { return math_mode(); }

const char *circatt_last_error(void) { return g_last_error.c_str(); }

int circatt_pattern(int nsp, int64_t n1, int64_t n2, int32_t ws, int64_t nb, int32_t *rowptr,
                    int32_t *colval, void *stream) {
    Geom g;
    CIRCATT_TRY(check_geom(nsp, n1, n2, ws, g));
    if (nb < 1) return fail(CIRCATT_ERR_INVALID, "nb=%lld must be >= 1", (long long)nb);
    CIRCATT_NONNULL(rowptr);
    CIRCATT_NONNULL(colval);
    return hip_result(launch_pattern(g, nb, rowptr, colval, as_stream(stream)), "circatt_pattern");
}

int circatt_similarity(int kind, int dtype, int nsp, int64_t n1, int64_t n2, int32_t ws,
                       int64_t C, int64_t nb, float scale, const void *x, const void *y,
                       float *nzval, void *stream) {
    Geom g;
    CIRCATT_TRY(check_kind(kind));
    CIRCATT_TRY(check_dtype(dtype));
    CIRCATT_TRY(check_geom(nsp, n1, n2, ws, g));
    if (C < 1 || C > INT32_MAX) return fail(CIRCATT_ERR_INVALID, "invalid channel count %lld", (long long)C);
    if (nb < 1) return fail(CIRCATT_ERR_INVALID, "nb=%lld must be >= 1", (long long)nb);
    CIRCATT_NONNULL(x);
    CIRCATT_NONNULL(y);
    CIRCATT_NONNULL(nzval);
    const int ncomp = dtype == CIRCATT_C32 ? 2 : 1;
    FusedProblem pr{};
    pr.g = g;
    pr.kind = kind;
    pr.ncomp = ncomp;
    pr.dh = (int)C;
    pr.nunits = nb;
    pr.scale = scale;
    pr.q = static_cast<const float *>(x);
    pr.k = static_cast<const float *>(y);
    pr.nz = nzval;
    // 2D windows of 17 to 33: scores in registers; up to 15 wide: the row
    // kernel (faster than the matrix-core kernel at every measured size); wider
    // windows, 1D or 2D, and every Distance similarity those do not take: the
    // sub-row kernel (all three form -|x - y|^2 / 2 from the differences, as the
    // reference does, where the matrix-core kernel expands it); otherwise the
    // matrix-core kernel
    if (sim_mx_supported(kind == CIRCATT_DISTANCE, g, (int)C, ncomp, nb))
        return hip_result(launch_sim_mx(kind == CIRCATT_DISTANCE, ncomp, g, (int)C, nb, scale,
                                        pr.q, pr.k, nzval, as_stream(stream)),
                          "circatt_similarity");
    const bool rows_ok = sim_rows_supported(g, (int)C, ncomp, nb);
    const bool mfma_ok = fused_supported(MODE_SIM, pr);
    if (!rows_ok && (g.ws > 15 || kind == CIRCATT_DISTANCE) &&
        sim_wide_supported(g, (int)C, ncomp, nb))
        return hip_result(launch_sim_wide(kind == CIRCATT_DISTANCE, ncomp, g, (int)C, nb, scale,
                                          pr.q, pr.k, nzval, as_stream(stream)),
                          "circatt_similarity");
    if (rows_ok)
        return hip_result(launch_sim_rows(kind == CIRCATT_DISTANCE, ncomp, g, (int)C, nb, scale,
                                          pr.q, pr.k, nzval, as_stream(stream)),
                          "circatt_similarity");
    if (mfma_ok)
        return hip_result(launch_fused(MODE_SIM, pr, as_stream(stream)), "circatt_similarity");
    return hip_result(launch_similarity(kind == CIRCATT_DISTANCE, ncomp, g, (int)C, nb, scale,
                                        pr.q, pr.k, nzval, as_stream(stream)),
                      "circatt_similarity");
}

int circatt_softmax(int64_t K, int64_t rows, const float *in, float *out, void *stream) {
    if (K < 1 || K > INT32_MAX) return fail(CIRCATT_ERR_INVALID, "invalid K=%lld", (long long)K);
    if (rows < 0) return fail(CIRCATT_ERR_INVALID, "invalid rows=%lld", (long long)rows);
    if (rows == 0) return ok();
    CIRCATT_NONNULL(in);
    CIRCATT_NONNULL(out);
    return hip_result(launch_softmax((int)K, rows, in, out, as_stream(stream)), "circatt_softmax");
}

int circatt_softmax_bwd(int64_t K, int64_t rows, const float *A, const float *dA, float *dS,
                        void *stream) {
    if (K < 1 || K > INT32_MAX) return fail(CIRCATT_ERR_INVALID, "invalid K=%lld", (long long)K);
    if (rows < 0) return fail(CIRCATT_ERR_INVALID, "invalid rows=%lld", (long long)rows);
    if (rows == 0) return ok();
    CIRCATT_NONNULL(A);
    CIRCATT_NONNULL(dA);
    CIRCATT_NONNULL(dS);
    return hip_result(launch_softmax_bwd((int)K, rows, A, dA, dS, as_stream(stream)),
                      "circatt_softmax_bwd");
}

int circatt_apply(int trans, int dtype, int nsp, int64_t n1, int64_t n2, int32_t ws, int64_t C,
                  int64_t nb, const float *nzval, const void *x, void *y, void *stream) {
    Geom g;
    CIRCATT_TRY(check_dtype(dtype));
    CIRCATT_TRY(check_geom(nsp, n1, n2, ws, g));
    if (trans != 0 && trans != 1) return fail(CIRCATT_ERR_INVALID, "trans=%d must be 0 or 1", trans);
    if (C < 1 || C > INT32_MAX) return fail(CIRCATT_ERR_INVALID, "invalid channel count %lld", (long long)C);
    if (nb < 1) return fail(CIRCATT_ERR_INVALID, "nb=%lld must be >= 1", (long long)nb);
    CIRCATT_NONNULL(nzval);
    CIRCATT_NONNULL(x);
    CIRCATT_NONNULL(y);
    if (x == y) return fail(CIRCATT_ERR_INVALID, "x and y must not alias");
    return hip_result(launch_apply(trans == 1, false, dtype == CIRCATT_C32 ? 2 : 1, g, (int)C, nb,
                                   1.f, nzval, static_cast<const float *>(x), nullptr,
                                   static_cast<float *>(y), as_stream(stream)),
                      "circatt_apply");
}

int circatt_similarity_bwd(int kind, int dtype, int nsp, int64_t n1, int64_t n2, int32_t ws,
                           int64_t C, int64_t nb, float scale, const float *dS, const void *x,
                           const void *y, void *dx, void *dy, void *stream) {
    Geom g;
    CIRCATT_TRY(check_kind(kind));
    CIRCATT_TRY(check_dtype(dtype));
    CIRCATT_TRY(check_geom(nsp, n1, n2, ws, g));
    if (C < 1 || C > INT32_MAX) return fail(CIRCATT_ERR_INVALID, "invalid channel count %lld", (long long)C);
    if (nb < 1) return fail(CIRCATT_ERR_INVALID, "nb=%lld must be >= 1", (long long)nb);
    CIRCATT_NONNULL(dS);
    CIRCATT_NONNULL(x);
    CIRCATT_NONNULL(y);
    const int ncomp = dtype == CIRCATT_C32 ? 2 : 1;
    const bool dist = kind == CIRCATT_DISTANCE;
    const float *xf = static_cast<const float *>(x);
    const float *yf = static_cast<const float *>(y);
    const bool mx = apply_mx_supported(g, (int)C, ncomp, nb, 2);
    if (dx && dy && (mx || apply_pair_supported(g, (int)C, ncomp, nb))) {
        // both products in one grid
        if (dx == x || dx == y) return fail(CIRCATT_ERR_INVALID, "dx must not alias x or y");
        if (dy == x || dy == y) return fail(CIRCATT_ERR_INVALID, "dy must not alias x or y");
        return hip_result((mx ? launch_apply_mx_pair : launch_apply_pair)(
                              dist, ncomp, g, (int)C, nb, scale, dS, xf, yf, static_cast<float *>(dx),
                              static_cast<float *>(dy), as_stream(stream)),
                          "circatt_similarity_bwd");
    }
    if (dx) {
        if (dx == x || dx == y) return fail(CIRCATT_ERR_INVALID, "dx must not alias x or y");
        hipError_t e = launch_apply(false, dist, ncomp, g, (int)C, nb, scale, dS, yf, xf,
                                    static_cast<float *>(dx), as_stream(stream));
        if (e != hipSuccess) return hip_result(e, "circatt_similarity_bwd");
    }
    if (dy) {
        if (dy == x || dy == y) return fail(CIRCATT_ERR_INVALID, "dy must not alias x or y");
        hipError_t e = launch_apply(true, dist, ncomp, g, (int)C, nb, scale, dS, xf, yf,
                                    static_cast<float *>(dy), as_stream(stream));
        if (e != hipSuccess) return hip_result(e, "circatt_similarity_bwd");
    }
    return ok();
}

static int sum_impl(bool col, int nsp, int64_t n1, int64_t n2, int32_t ws, int64_t nb,
                    const float *nzval, float *out, void *stream, const char *name) {
    Geom g;
    CIRCATT_TRY(check_geom(nsp, n1, n2, ws, g));
    if (nb < 1) return fail(CIRCATT_ERR_INVALID, "nb=%lld must be >= 1", (long long)nb);
    CIRCATT_NONNULL(nzval);
    CIRCATT_NONNULL(out);
    return hip_result(launch_sum(col, g, nb, nzval, out, as_stream(stream)), name);
}

int circatt_rowsum(int nsp, int64_t n1, int64_t n2, int32_t ws, int64_t nb, const float *nzval,
                   float *out, void *stream) {
    return sum_impl(false, nsp, n1, n2, ws, nb, nzval, out, stream, "circatt_rowsum");
}

int circatt_colsum(int nsp, int64_t n1, int64_t n2, int32_t ws, int64_t nb, const float *nzval,
                   float *out, void *stream) {
    return sum_impl(true, nsp, n1, n2, ws, nb, nzval, out, stream, "circatt_colsum");
}

int circatt_axpby(int64_t nnz, int64_t nb, const float *alpha, float alpha0, const float *X,
                  const float *beta, float beta0, const float *Y, float *Z, void *stream) {
    if (nnz < 0 || nb < 1) return fail(CIRCATT_ERR_INVALID, "invalid nnz=%lld / nb=%lld", (long long)nnz, (long long)nb);
    if (nnz == 0) return ok();
    CIRCATT_NONNULL(X);
    CIRCATT_NONNULL(Z);
    return hip_result(launch_axpby(nnz, nb, alpha, alpha0, X, beta, beta0, Y, Z, as_stream(stream)),
                      "circatt_axpby");
}

int64_t circatt_batch_dot_workspace_bytes(int64_t nnz, int64_t nb) {
    if (nnz < 0 || nb < 1) return -1;
    return nb * (int64_t)batch_dot_chunks(nnz) * (int64_t)sizeof(double);
}

int circatt_batch_dot(int64_t nnz, int64_t nb, const float *X, const float *Y, float *out,
                      void *workspace, int64_t workspace_bytes, void *stream) {
    if (nnz < 0 || nb < 1)
        return fail(CIRCATT_ERR_INVALID, "invalid nnz=%lld / nb=%lld", (long long)nnz, (long long)nb);
    CIRCATT_NONNULL(X);
    CIRCATT_NONNULL(out);
    CIRCATT_NONNULL(workspace);
    const int64_t need = circatt_batch_dot_workspace_bytes(nnz, nb);
    if (workspace_bytes < need)
        return fail(CIRCATT_ERR_INVALID, "workspace of %lld bytes, %lld needed",
                    (long long)workspace_bytes, (long long)need);
    if (out == X || out == Y || workspace == X || workspace == Y || workspace == out)
        return fail(CIRCATT_ERR_INVALID, "out and workspace must not alias X or Y");
    return hip_result(launch_batch_dot(nnz, nb, X, Y, out, workspace, as_stream(stream)),
                      "circatt_batch_dot");
}

static int fused_problem(int kind, int dtype, int nsp, int64_t n1, int64_t n2, int32_t ws,
                         int64_t C, int64_t nheads, int64_t B, FusedProblem &pr) {
    Geom g;
    const int cl = (dtype & CIRCATT_CHANNELS_LAST) ? 1 : 0;
    dtype &= ~CIRCATT_CHANNELS_LAST;
    CIRCATT_TRY(check_kind(kind));
    CIRCATT_TRY(check_dtype(dtype));
    CIRCATT_TRY(check_geom(nsp, n1, n2, ws, g));
    if (nheads < 1 || C < 1 || C % nheads != 0)
        return fail(CIRCATT_ERR_INVALID, "channels (%lld) must be divisible by nheads (%lld)",
                    (long long)C, (long long)nheads);
    if (B < 1) return fail(CIRCATT_ERR_INVALID, "batch B=%lld must be >= 1", (long long)B);
    pr = FusedProblem{};
    pr.g = g;
    pr.kind = kind;
    pr.ncomp = dtype == CIRCATT_C32 ? 2 : 1;
    pr.dh = (int)(C / nheads);
    pr.nunits = nheads * B;
    pr.cl = cl;
    pr.nheads = (int)nheads;
    if (cl && g.P * C * pr.ncomp * 4 >= (int64_t)INT32_MAX)
        return fail(CIRCATT_ERR_UNSUPPORTED,
                    "channels-last image of %lld floats exceeds the kernels' 32-bit offsets",
                    (long long)(g.P * C * pr.ncomp));
    // q ./ sqrt(tau), k ./ sqrt(tau), tau = sqrt(channels per head)
    // (src/attention.jl:20-21) scale the similarity by 1/sqrt(dh).
    pr.scale = (float)(1.0 / std::sqrt((double)pr.dh));
    return CIRCATT_OK;
}

int circatt_fused_fwd(int kind, int dtype, int nsp, int64_t n1, int64_t n2, int32_t ws,
                      int64_t C, int64_t nheads, int64_t B, const void *q, const void *k,
                      const void *v, void *y, float *lse, void *stream) {
    FusedProblem pr;
    CIRCATT_TRY(fused_problem(kind, dtype, nsp, n1, n2, ws, C, nheads, B, pr));
    CIRCATT_NONNULL(q);
    CIRCATT_NONNULL(k);
    CIRCATT_NONNULL(v);
    CIRCATT_NONNULL(y);
    CIRCATT_NONNULL(lse);
    if (y == q || y == k || y == v) return fail(CIRCATT_ERR_INVALID, "y must not alias q, k or v");
    pr.q = static_cast<const float *>(q);
    pr.k = static_cast<const float *>(k);
    pr.v = static_cast<const float *>(v);
    pr.yout = static_cast<float *>(y);
    pr.lse_out = lse;
    if (!fused_supported(MODE_FWD, pr))
        return fail(CIRCATT_ERR_UNSUPPORTED,
                    "circatt_fused_fwd: window ws=%d with %d real components per head is outside "
                    "the fused kernels' range", pr.g.ws, pr.dh * pr.ncomp);
    return hip_result(launch_fused(MODE_FWD, pr, as_stream(stream)), "circatt_fused_fwd");
}

int64_t circatt_fused_bwd_workspace_bytes(int nsp, int64_t n1, int64_t n2, int64_t nheads,
                                          int64_t B) {
    if ((nsp != 1 && nsp != 2) || n1 < 1 || (nsp == 2 && n2 < 1) || nheads < 1 || B < 1) return -1;
    const int64_t P = nsp == 1 ? n1 : n1 * n2;
    return P * nheads * B * (int64_t)sizeof(float);
}

namespace {

enum BwdParts { BWD_DQ = 1, BWD_DKDV = 2 };

int fused_bwd_impl(int parts, int kind, int dtype, int nsp, int64_t n1, int64_t n2, int32_t ws,
                   int64_t C, int64_t nheads, int64_t B, const void *q, const void *k,
                   const void *v, const void *y, const void *dy, const float *lse, void *dq,
                   void *dk, void *dv, const void *workspace, int64_t workspace_bytes,
                   void *stream, const char *name) {
    FusedProblem pr;
    CIRCATT_TRY(fused_problem(kind, dtype, nsp, n1, n2, ws, C, nheads, B, pr));
    CIRCATT_NONNULL(q);
    CIRCATT_NONNULL(k);
    CIRCATT_NONNULL(v);
    CIRCATT_NONNULL(dy);
    CIRCATT_NONNULL(lse);
    CIRCATT_NONNULL(workspace);
    if (parts & BWD_DQ) {
        CIRCATT_NONNULL(y);
        CIRCATT_NONNULL(dq);
    }
    if (parts & BWD_DKDV) {
        CIRCATT_NONNULL(dk);
        CIRCATT_NONNULL(dv);
    }
    const int64_t need = circatt_fused_bwd_workspace_bytes(nsp, n1, n2, nheads, B);
    if (workspace_bytes < need)
        return fail(CIRCATT_ERR_INVALID, "workspace of %lld bytes, %lld needed",
                    (long long)workspace_bytes, (long long)need);
    for (const void *out : {dq, dk, dv}) {
        if (out == nullptr) continue;
        for (const void *in : {q, k, v, y, dy, static_cast<const void *>(lse), workspace})
            if (out == in) return fail(CIRCATT_ERR_INVALID, "gradient outputs must not alias inputs");
    }
    pr.q = static_cast<const float *>(q);
    pr.k = static_cast<const float *>(k);
    pr.v = static_cast<const float *>(v);
    pr.y = static_cast<const float *>(y);
    pr.dy = static_cast<const float *>(dy);
    pr.lse = lse;
    pr.dq = static_cast<float *>(dq);
    pr.dk = static_cast<float *>(dk);
    pr.dv = static_cast<float *>(dv);
    pr.dbuf = static_cast<float *>(const_cast<void *>(workspace));
    if (!fused_supported(MODE_BWDQ, pr) || !fused_supported(MODE_BWDKV, pr))
        return fail(CIRCATT_ERR_UNSUPPORTED,
                    "%s: window ws=%d with %d real components per head is outside the fused "
                    "kernels' range", name, pr.g.ws, pr.dh * pr.ncomp);
    if (parts & BWD_DQ) {
        hipError_t e = launch_fused(MODE_BWDQ, pr, as_stream(stream));
        if (e != hipSuccess) return hip_result(e, name);
    }
    if (parts & BWD_DKDV) {
        hipError_t e = launch_fused(MODE_BWDKV, pr, as_stream(stream));
        if (e != hipSuccess) return hip_result(e, name);
    }
    return ok();
}

}  // namespace

int circatt_fused_bwd(int kind, int dtype, int nsp, int64_t n1, int64_t n2, int32_t ws,
                      int64_t C, int64_t nheads, int64_t B, const void *q, const void *k,
                      const void *v, const void *y, const void *dy, const float *lse, void *dq,
                      void *dk, void *dv, void *workspace, int64_t workspace_bytes,
                      void *stream) {
    return fused_bwd_impl(BWD_DQ | BWD_DKDV, kind, dtype, nsp, n1, n2, ws, C, nheads, B, q, k,
                          v, y, dy, lse, dq, dk, dv, workspace, workspace_bytes, stream,
                          "circatt_fused_bwd");
}

int circatt_fused_bwd_dq(int kind, int dtype, int nsp, int64_t n1, int64_t n2, int32_t ws,
                         int64_t C, int64_t nheads, int64_t B, const void *q, const void *k,
                         const void *v, const void *y, const void *dy, const float *lse,
                         void *dq, void *workspace, int64_t workspace_bytes, void *stream) {
    return fused_bwd_impl(BWD_DQ, kind, dtype, nsp, n1, n2, ws, C, nheads, B, q, k, v, y, dy,
                          lse, dq, nullptr, nullptr, workspace, workspace_bytes, stream,
                          "circatt_fused_bwd_dq");
}

int circatt_fused_bwd_dkdv(int kind, int dtype, int nsp, int64_t n1, int64_t n2, int32_t ws,
                           int64_t C, int64_t nheads, int64_t B, const void *q, const void *k,
                           const void *v, const void *dy, const float *lse, void *dk, void *dv,
                           const void *workspace, int64_t workspace_bytes, void *stream) {
    return fused_bwd_impl(BWD_DKDV, kind, dtype, nsp, n1, n2, ws, C, nheads, B, q, k, v,
                          nullptr, dy, lse, nullptr, dk, dv, workspace, workspace_bytes, stream,
                          "circatt_fused_bwd_dkdv");
}

}  // extern "C"

// ---------------------------------------------------------------------------
// Fused backward without a workspace argument: the per-row D = <dy, y> lives
// in `scratch`, a file-scope device array of fixed size.  Each GPU the
// library runs on holds its own copy until the process ends; its device
// address is looked up once per device (hipGetSymbolAddress) and kept.
// ---------------------------------------------------------------------------
namespace {

constexpr int64_t kScratchBytes = int64_t(16) << 20;  // 4M rows of D
constexpr int kMaxDevices = 64;

static __device__ __align__(256) float scratch[kScratchBytes / sizeof(float)];

std::mutex g_scratch_mu;
void *g_scratch_ptr[kMaxDevices] = {};

// Device address of this device's `scratch` (looked up on its first use).
int scratch_address(void **out, const char *name) {
    int dev = -1;
    hipError_t e = hipGetDevice(&dev);
    if (e != hipSuccess) return hip_result(e, name);
    if (dev < 0 || dev >= kMaxDevices)
        return fail(CIRCATT_ERR_UNSUPPORTED, "%s: device %d beyond the %d supported", name, dev,
                    kMaxDevices);
    std::lock_guard<std::mutex> lock(g_scratch_mu);
    if (g_scratch_ptr[dev] == nullptr) {
        void *p = nullptr;
        e = hipGetSymbolAddress(&p, HIP_SYMBOL(scratch));
        if (e != hipSuccess) return hip_result(e, name);
        if (p == nullptr) return fail(CIRCATT_ERR_HIP, "%s: no device address for scratch", name);
        g_scratch_ptr[dev] = p;
    }
    *out = g_scratch_ptr[dev];
    return CIRCATT_OK;
}

}  // namespace

extern "C" {

int64_t circatt_fused_bwd_noalloc_max_rows(void) {
    return kScratchBytes / (int64_t)sizeof(float);
}

int circatt_fused_bwd_noalloc(int kind, int dtype, int nsp, int64_t n1, int64_t n2, int32_t ws,
                              int64_t C, int64_t nheads, int64_t B, const void *q,
                              const void *k, const void *v, const void *y, const void *dy,
                              const float *lse, void *dq, void *dk, void *dv, void *stream) {
    const char *name = "circatt_fused_bwd_noalloc";
    const int64_t need = circatt_fused_bwd_workspace_bytes(nsp, n1, n2, nheads, B);
    if (need < 0) return fail(CIRCATT_ERR_INVALID, "%s: invalid shape", name);
    if (need > kScratchBytes)
        return fail(CIRCATT_ERR_INVALID,
                    "%s: %lld rows of D (P*nheads*B) exceed the static scratch of %lld rows; "
                    "use circatt_fused_bwd with a workspace",
                    name, (long long)(need / 4), (long long)(kScratchBytes / 4));
    FusedProblem pr;
    CIRCATT_TRY(fused_problem(kind, dtype, nsp, n1, n2, ws, C, nheads, B, pr));
    CIRCATT_NONNULL(q);
    CIRCATT_NONNULL(k);
    CIRCATT_NONNULL(v);
    CIRCATT_NONNULL(y);
    CIRCATT_NONNULL(dy);
    CIRCATT_NONNULL(lse);
    CIRCATT_NONNULL(dq);
    CIRCATT_NONNULL(dk);
    CIRCATT_NONNULL(dv);
    void *work = nullptr;
    CIRCATT_TRY(scratch_address(&work, name));
    return fused_bwd_impl(BWD_DQ | BWD_DKDV, kind, dtype, nsp, n1, n2, ws, C, nheads, B, q, k,
                          v, y, dy, lse, dq, dk, dv, work, need, stream, name);
}

int circatt_malloc(void **ptr, int64_t bytes) {
    CIRCATT_NONNULL(ptr);
    if (bytes < 0) return fail(CIRCATT_ERR_INVALID, "negative size");
    return hip_result(hipMalloc(ptr, (size_t)bytes), "circatt_malloc");
}

int circatt_free(void *ptr) { return hip_result(hipFree(ptr), "circatt_free"); }

int circatt_fill(float *dst, int64_t n, float value, void *stream) {
    if (n < 0) return fail(CIRCATT_ERR_INVALID, "n=%lld must be >= 0", (long long)n);
    if (n == 0) return ok();
    CIRCATT_NONNULL(dst);
    uint32_t bits;
    std::memcpy(&bits, &value, 4);
    return hip_result(launch_fill(reinterpret_cast<uint32_t *>(dst), n, bits, as_stream(stream)),
                      "circatt_fill");
}

int circatt_copy_blocks(void *dst, const void *src, int64_t block_bytes, int64_t ninner,
                        int64_t dst_stride_inner, int64_t src_stride_inner, int64_t nouter,
                        int64_t dst_stride_outer, int64_t src_stride_outer, void *stream) {
    if (block_bytes < 0 || ninner < 0 || nouter < 0)
        return fail(CIRCATT_ERR_INVALID, "negative block size or count");
    if (dst_stride_inner < 0 || src_stride_inner < 0 || dst_stride_outer < 0 || src_stride_outer < 0)
        return fail(CIRCATT_ERR_INVALID, "negative stride");
    if (block_bytes == 0 || ninner == 0 || nouter == 0) return ok();
    CIRCATT_NONNULL(dst);
    CIRCATT_NONNULL(src);
    // the destination blocks must not overlap (a destination byte written
    // twice would depend on the order of the writes)
    if ((ninner > 1 && dst_stride_inner < block_bytes) ||
        (nouter > 1 && dst_stride_outer < (ninner - 1) * dst_stride_inner + block_bytes))
        return fail(CIRCATT_ERR_INVALID, "destination blocks overlap");
    const int64_t dst_end = (nouter - 1) * dst_stride_outer + (ninner - 1) * dst_stride_inner + block_bytes;
    const int64_t src_end = (nouter - 1) * src_stride_outer + (ninner - 1) * src_stride_inner + block_bytes;
    const char *d0 = static_cast<const char *>(dst), *s0 = static_cast<const char *>(src);
    if (d0 < s0 + src_end && s0 < d0 + dst_end)
        return fail(CIRCATT_ERR_INVALID, "source and destination ranges overlap");
    return hip_result(launch_copy_blocks(dst, src, block_bytes, ninner, dst_stride_inner,
                                         src_stride_inner, nouter, dst_stride_outer,
                                         src_stride_outer, as_stream(stream)),
                      "circatt_copy_blocks");
}

int circatt_sum_middle(const float *src, float *dst, int64_t inner, int64_t nsum, int64_t outer,
                       void *stream) {
    if (inner < 0 || nsum < 0 || outer < 0) return fail(CIRCATT_ERR_INVALID, "negative size");
    if (inner == 0 || outer == 0) return ok();
    if (nsum == 0) return circatt_fill(dst, inner * outer, 0.f, stream);
    CIRCATT_NONNULL(src);
    CIRCATT_NONNULL(dst);
    if (dst < src + inner * nsum * outer && src < dst + inner * outer)
        return fail(CIRCATT_ERR_INVALID, "src and dst overlap");
    return hip_result(launch_sum_middle(src, dst, inner, nsum, outer, as_stream(stream)),
                      "circatt_sum_middle");
}

int circatt_count_unequal(int kind, int64_t n, const void *a, const void *b, int64_t *count,
                          void *stream) {
    if (kind != 0 && kind != 1) return fail(CIRCATT_ERR_INVALID, "kind=%d must be 0 or 1", kind);
    if (n < 0) return fail(CIRCATT_ERR_INVALID, "n=%lld must be >= 0", (long long)n);
    CIRCATT_NONNULL(count);
    if (n > 0) {
        CIRCATT_NONNULL(a);
        CIRCATT_NONNULL(b);
    }
    return hip_result(launch_count_unequal(kind == 1, n, static_cast<const uint32_t *>(a),
                                           static_cast<const uint32_t *>(b), count,
                                           as_stream(stream)),
                      "circatt_count_unequal");
}

// ---------------------------------------------------------------------------
// Token operators.

namespace {

int check_token_dtype(int dtype) {
    if (dtype != CIRCATT_F32 && dtype != CIRCATT_F16 && dtype != CIRCATT_BF16)
        return fail(CIRCATT_ERR_UNSUPPORTED, "dtype %d not supported (Float32, Float16 or BFloat16)", dtype);
    return CIRCATT_OK;
}
int esize_of(int dtype) { return dtype == CIRCATT_F32 ? 4 : 2; }

// Heads of one call: nheads of queries over kv_heads of keys and values.
int check_heads(int64_t nheads, int64_t kv_heads, int64_t dh) {
    if (nheads < 1 || kv_heads < 1 || nheads > 32768)
        return fail(CIRCATT_ERR_INVALID, "invalid head counts %lld, %lld", (long long)nheads, (long long)kv_heads);
    if (nheads % kv_heads != 0)
        return fail(CIRCATT_ERR_INVALID, "nheads (%lld) must be divisible by kv_heads (%lld)", (long long)nheads,
                    (long long)kv_heads);
    if (dh < 1) return fail(CIRCATT_ERR_INVALID, "invalid channels per head %lld", (long long)dh);
    if (dh > 128 || dh % 8 != 0)
        return fail(CIRCATT_ERR_UNSUPPORTED, "channels per head (%lld) must be a multiple of 8 up to 128", (long long)dh);
    return CIRCATT_OK;
}
int check_window(int64_t window, int64_t sinks, float scale) {
    if (window < 1) return fail(CIRCATT_ERR_INVALID, "window W=%lld must be >= 1", (long long)window);
    if (sinks < 0) return fail(CIRCATT_ERR_INVALID, "sinks=%lld must be >= 0", (long long)sinks);
    if (!(scale > 0.f) || !std::isfinite(scale))
        return fail(CIRCATT_ERR_INVALID, "scale=%g must be positive and finite", (double)scale);
    return CIRCATT_OK;
}
// Rows of a token signal: channels adjacent, 16-byte aligned, row over row.
int check_rows(const char *name, const void *p, int64_t row, int64_t batch, int64_t channels, int esize) {
    if (p == nullptr) return fail(CIRCATT_ERR_INVALID, "%s is NULL", name);
    if (row < channels || batch < 0 || row > (int64_t)1 << 22)
        return fail(CIRCATT_ERR_INVALID, "%s: strides %lld, %lld do not fit rows of %lld channels", name,
                    (long long)row, (long long)batch, (long long)channels);
    if (reinterpret_cast<uintptr_t>(p) % 16 != 0 || row * esize % 16 != 0 || batch * esize % 16 != 0)
        return fail(CIRCATT_ERR_INVALID, "%s must have 16-byte aligned rows", name);
    return CIRCATT_OK;
}

// A launch holds less than 2^32 threads along an axis.
int check_threads(int64_t threads) {
    if (threads > UINT32_MAX)
        return fail(CIRCATT_ERR_UNSUPPORTED, "a launch of %lld threads, at most 2^32 - 1 are supported", (long long)threads);
    return CIRCATT_OK;
}

int sliding_problem(int dtype, int64_t L, int64_t B, int64_t nheads, int64_t kv_heads, int64_t dh, int64_t window,
                    int64_t sinks, float scale, SlidingProblem &pr) {
    CIRCATT_TRY(check_token_dtype(dtype));
    CIRCATT_TRY(check_heads(nheads, kv_heads, dh));
    CIRCATT_TRY(check_window(window, sinks, scale));
    if (L < 0 || B < 0 || L > INT32_MAX / 2 || B > INT32_MAX || L * nheads > INT32_MAX / 2)
        return fail(CIRCATT_ERR_INVALID, "invalid signal size L=%lld, B=%lld", (long long)L, (long long)B);
    if (B > 0 && L * nheads > (int64_t)INT32_MAX / B)
        return fail(CIRCATT_ERR_UNSUPPORTED, "B*L*nheads = %lld * %lld exceeds 2^31", (long long)B, (long long)(L * nheads));
    pr = SlidingProblem{};
    pr.dtype = dtype;
    pr.B = (int)B;
    pr.L = (int)L;
    pr.H = (int)nheads;
    pr.Hk = (int)kv_heads;
    pr.G = (int)(nheads / kv_heads);
    pr.D = (int)dh;
    // a window that holds every token leaves no sinks outside it
    pr.W = (int)(window < L ? window : L);
    pr.S = window >= L ? 0 : (int)(sinks < L ? sinks : L);
    pr.scale = scale;
    return CIRCATT_OK;
}

int paged_table(int64_t B, int64_t npages, int64_t page_size, int64_t page_stride, int64_t row_stride, int64_t channels,
                const int32_t *pages, int64_t pages_row, int64_t maxp, const int32_t *lengths, const void *cache_k,
                const void *cache_v, int esize, int &log2) {
    if (B < 1 || B > INT32_MAX / 2) return fail(CIRCATT_ERR_INVALID, "invalid sequence count %lld", (long long)B);
    if (page_size < 1 || page_size > 65536 || (page_size & (page_size - 1)) != 0)
        return fail(CIRCATT_ERR_UNSUPPORTED, "page size %lld must be a power of two up to 65536", (long long)page_size);
    for (log2 = 0; (1 << log2) < page_size;) ++log2;
    if (npages < 1 || npages > INT32_MAX / page_size)
        return fail(CIRCATT_ERR_INVALID, "a cache of %lld pages of %lld tokens", (long long)npages, (long long)page_size);
    if (maxp < 1 || pages_row < maxp || maxp > (int64_t)1 << (30 - log2))
        return fail(CIRCATT_ERR_INVALID, "a page table of %lld pages, rows of %lld", (long long)maxp, (long long)pages_row);
    CIRCATT_NONNULL(pages);
    CIRCATT_NONNULL(lengths);
    if (row_stride < channels || page_stride < 0 || (npages > 1 && page_stride < row_stride))
        return fail(CIRCATT_ERR_INVALID, "cache strides %lld, %lld do not fit rows of %lld channels",
                    (long long)page_stride, (long long)row_stride, (long long)channels);
    // rows are addressed in units of 16 bytes, in 32 bits
    if (row_stride > (int64_t)1 << 24 || page_stride > (int64_t)1 << 36 ||
        ((npages - 1) * (double)page_stride + (page_size - 1) * (double)row_stride + channels) * esize > 6.8e10)
        return fail(CIRCATT_ERR_UNSUPPORTED, "a cache of more than 63 GiB from end to end");
    for (const void *p : {cache_k, cache_v}) {
        if (p == nullptr) return fail(CIRCATT_ERR_INVALID, "cache is NULL");
        if (reinterpret_cast<uintptr_t>(p) % 16 != 0 || row_stride * esize % 16 != 0 || page_stride * esize % 16 != 0)
            return fail(CIRCATT_ERR_INVALID, "the cache must have 16-byte aligned rows");
    }
    return CIRCATT_OK;
}

int paged_problem(int dtype, int64_t T, int64_t B, int64_t nheads, int64_t kv_heads, int64_t dh, int64_t window,
                  int64_t sinks, float scale, int64_t page_size, int64_t maxp, PagedProblem &pr) {
    CIRCATT_TRY(check_token_dtype(dtype));
    CIRCATT_TRY(check_heads(nheads, kv_heads, dh));
    CIRCATT_TRY(check_window(window, sinks, scale));
    if (T < 0 || B < 1 || B > 65535 || T > INT32_MAX / 2 / nheads)
        return fail(CIRCATT_ERR_INVALID, "invalid sizes T=%lld, B=%lld", (long long)T, (long long)B);
    if (maxp < 1 || page_size < 1 || maxp > ((int64_t)1 << 30) / page_size)
        return fail(CIRCATT_ERR_INVALID, "a page table of %lld pages of %lld tokens", (long long)maxp, (long long)page_size);
    pr = PagedProblem{};
    pr.dtype = dtype;
    pr.T = T;
    pr.B = (int)B;
    pr.H = (int)nheads;
    pr.Hk = (int)kv_heads;
    pr.G = (int)(nheads / kv_heads);
    pr.D = (int)dh;
    const int64_t most = maxp * page_size;
    pr.W = (int)(window < most ? window : most);
    pr.S = window >= most ? 0 : (int)(sinks < most ? sinks : most);
    pr.scale = scale;
    pr.page = (int)page_size;
    pr.maxp = (int)maxp;
    return T == 0 ? CIRCATT_OK : check_threads(paged_threads(pr));
}

bool overlap(const void *a, int64_t na, const void *b, int64_t nb) {
    const uintptr_t x = reinterpret_cast<uintptr_t>(a), y = reinterpret_cast<uintptr_t>(b);
    return x < y ? y - x < (uintptr_t)na : x - y < (uintptr_t)nb;
}

// Memory of a call, from end to end of its strides (NULL: none).
struct Span {
    const char *name;
    const void *p;
    int64_t bytes;
};
Span span(const char *name, const void *p, int64_t n1, int64_t s1, int64_t n2, int64_t s2, int64_t width, int esize) {
    return Span{name, p, ((n1 - 1) * s1 + (n2 - 1) * s2 + width) * esize};
}
// Results are written while other workgroups still read the arguments.
int check_apart(std::initializer_list<Span> results, std::initializer_list<Span> arguments) {
    for (const Span *r = results.begin(); r != results.end(); ++r) {
        if (r->p == nullptr) continue;
        for (const Span &a : arguments)
            if (a.p != nullptr && overlap(r->p, r->bytes, a.p, a.bytes))
                return fail(CIRCATT_ERR_INVALID, "%s must not overlap %s", r->name, a.name);
        for (const Span *o = results.begin(); o != r; ++o)
            if (o->p != nullptr && overlap(r->p, r->bytes, o->p, o->bytes))
                return fail(CIRCATT_ERR_INVALID, "%s must not overlap %s", r->name, o->name);
    }
    return CIRCATT_OK;
}

int check_rests(const void *rest, const void *y, int64_t bytes, int dtype) {
    if (dtype == CIRCATT_F32) return fail(CIRCATT_ERR_INVALID, "y_rest belongs to the 16-bit types");
    if (reinterpret_cast<uintptr_t>(rest) % 16 != 0) return fail(CIRCATT_ERR_INVALID, "y_rest must be 16-byte aligned");
    if (overlap(rest, bytes, y, bytes)) return fail(CIRCATT_ERR_INVALID, "y_rest must not overlap y");
    return CIRCATT_OK;
}

}  // namespace

namespace {

// What scores are shaped by, for signals of up to `tokens` tokens.
int check_shape(int dtype, float scale, float cap, const float *slopes, const int32_t *prefix, const int32_t *places,
                int64_t places_row, int64_t tokens, ScoreShape &sh) {
    // the kernels form scale / cap and multiples of it and of the cap in Float32
    if (!(cap >= 0.f) || !(cap <= 1e30f) || (cap > 0.f && (!(scale / cap >= 1e-30f) || !(scale / cap <= 1e30f))))
        return fail(CIRCATT_ERR_INVALID, "cap=%g must be 0 or positive, and scale / cap within 1e-30 .. 1e30", (double)cap);
    if (prefix != nullptr && places != nullptr)
        return fail(CIRCATT_ERR_INVALID, "prefix and places do not go together");
    if (places != nullptr && places_row < 0) return fail(CIRCATT_ERR_INVALID, "negative stride");
    if (slopes != nullptr && tokens > (int64_t)1 << 24)
        return fail(CIRCATT_ERR_UNSUPPORTED, "slopes for %lld tokens, at most 2^24 are supported", (long long)tokens);
    sh.cap = cap;
    sh.curve = make_curve(cap, scale, dtype);
    sh.slopes = slopes;
    sh.prefix = prefix;
    sh.places = places;
    sh.places_row = places_row;
    return CIRCATT_OK;
}

// Arrays of a call's shape, which its results must not overlap.
struct ShapeSpans {
    Span slopes{"slopes", nullptr, 0}, prefix{"prefix", nullptr, 0}, places{"places", nullptr, 0};
    ShapeSpans() = default;
    ShapeSpans(const ScoreShape &sh, int64_t B, int64_t L, int64_t H)
        : slopes{"slopes", sh.slopes, 4 * H}, prefix{"prefix", sh.prefix, 4 * B},
          places{"places", sh.places, 4 * ((B - 1) * sh.places_row + L)} {}
};

int sliding_fwd_arguments(int dtype, int64_t L, int64_t B, int64_t nheads, int64_t kv_heads, int64_t dh, const void *q,
                          int64_t q_row, int64_t q_batch, const void *k, int64_t k_row, int64_t k_batch, const void *v,
                          int64_t v_row, int64_t v_batch, const int32_t *lengths, void *y, void *y_rest, float *lse,
                          const ShapeSpans &sh, SlidingProblem &pr) {
    const int es = esize_of(dtype);
    CIRCATT_TRY(check_rows("q", q, q_row, q_batch, nheads * dh, es));
    CIRCATT_TRY(check_rows("k", k, k_row, k_batch, kv_heads * dh, es));
    CIRCATT_TRY(check_rows("v", v, v_row, v_batch, kv_heads * dh, es));
    CIRCATT_TRY(check_rows("y", y, nheads * dh, 0, nheads * dh, es));
    pr.q = q, pr.q_row = q_row, pr.q_batch = q_batch;
    pr.k = k, pr.k_row = k_row, pr.k_batch = k_batch;
    pr.v = v, pr.v_row = v_row, pr.v_batch = v_batch;
    pr.lengths = lengths;
    if (y_rest != nullptr) CIRCATT_TRY(check_rests(y_rest, y, L * B * nheads * dh * es, dtype));
    pr.y = y;
    pr.y_rest = y_rest;
    pr.lse = lse;
    const int64_t C = nheads * dh, Ck = kv_heads * dh;
    return check_apart({span("y", y, B, L * C, L, C, C, es), span("y_rest", y_rest, B, L * C, L, C, C, es),
                        span("lse", lse, 1, 0, 1, 0, B * L * nheads, 4)},
                       {span("q", q, B, q_batch, L, q_row, C, es), span("k", k, B, k_batch, L, k_row, Ck, es),
                        span("v", v, B, v_batch, L, v_row, Ck, es), sh.slopes, sh.prefix, sh.places});
}

int sliding_bwd_arguments(int dtype, int64_t L, int64_t B, int64_t nheads, int64_t kv_heads, int64_t dh, const void *q,
                          int64_t q_row, int64_t q_batch, const void *k, int64_t k_row, int64_t k_batch, const void *v,
                          int64_t v_row, int64_t v_batch, const int32_t *lengths, const void *y, const void *y_rest,
                          const float *lse, const void *dy, int64_t dy_row, int64_t dy_batch, void *dq, void *dk, void *dv,
                          void *workspace, int64_t workspace_bytes, int64_t need, const ShapeSpans &sh, SlidingProblem &pr) {
    const int es = esize_of(dtype);
    CIRCATT_TRY(check_rows("q", q, q_row, q_batch, nheads * dh, es));
    CIRCATT_TRY(check_rows("k", k, k_row, k_batch, kv_heads * dh, es));
    CIRCATT_TRY(check_rows("v", v, v_row, v_batch, kv_heads * dh, es));
    CIRCATT_TRY(check_rows("y", y, nheads * dh, 0, nheads * dh, es));
    CIRCATT_TRY(check_rows("dy", dy, dy_row, dy_batch, nheads * dh, es));
    CIRCATT_TRY(check_rows("dq", dq, nheads * dh, 0, nheads * dh, es));
    CIRCATT_NONNULL(lse);
    if ((dk == nullptr) != (dv == nullptr)) return fail(CIRCATT_ERR_INVALID, "dk and dv go together");
    if (dk != nullptr) {
        CIRCATT_TRY(check_rows("dk", dk, kv_heads * dh, 0, kv_heads * dh, es));
        CIRCATT_TRY(check_rows("dv", dv, kv_heads * dh, 0, kv_heads * dh, es));
    }
    CIRCATT_NONNULL(workspace);
    if (workspace_bytes < need)
        return fail(CIRCATT_ERR_INVALID, "workspace of %lld bytes, %lld needed", (long long)workspace_bytes, (long long)need);
    if (reinterpret_cast<uintptr_t>(workspace) % 16 != 0) return fail(CIRCATT_ERR_INVALID, "workspace must be 16-byte aligned");
    pr.q = q, pr.q_row = q_row, pr.q_batch = q_batch;
    pr.k = k, pr.k_row = k_row, pr.k_batch = k_batch;
    pr.v = v, pr.v_row = v_row, pr.v_batch = v_batch;
    pr.lengths = lengths;
    if (y_rest != nullptr) CIRCATT_TRY(check_rests(y_rest, y, L * B * nheads * dh * es, dtype));
    pr.y = const_cast<void *>(y);
    pr.y_rest = const_cast<void *>(y_rest);
    pr.lse = const_cast<float *>(lse);
    pr.dy = dy, pr.dy_row = dy_row, pr.dy_batch = dy_batch;
    pr.dq = dq, pr.dk = dk, pr.dv = dv;
    pr.work = static_cast<float *>(workspace);
    const int64_t C = nheads * dh, Ck = kv_heads * dh;
    return check_apart(
        {span("dq", dq, B, L * C, L, C, C, es), span("dk", dk, B, L * Ck, L, Ck, Ck, es),
         span("dv", dv, B, L * Ck, L, Ck, Ck, es), span("workspace", workspace, 1, 0, 1, 0, need, 1)},
        {span("q", q, B, q_batch, L, q_row, C, es), span("k", k, B, k_batch, L, k_row, Ck, es),
         span("v", v, B, v_batch, L, v_row, Ck, es), span("y", y, B, L * C, L, C, C, es),
         span("y_rest", y_rest, B, L * C, L, C, C, es), span("lse", lse, 1, 0, 1, 0, B * L * nheads, 4),
         span("dy", dy, B, dy_batch, L, dy_row, C, es), sh.slopes, sh.prefix, sh.places});
}

}  // namespace

int circatt_sliding_fwd(int dtype, int64_t L, int64_t B, int64_t nheads, int64_t kv_heads, int64_t dh, int64_t window,
                        int64_t sinks, float scale, const void *q, int64_t q_row, int64_t q_batch, const void *k,
                        int64_t k_row, int64_t k_batch, const void *v, int64_t v_row, int64_t v_batch,
                        const int32_t *lengths, void *y, void *y_rest, float *lse, void *stream) {
    SlidingProblem pr;
    CIRCATT_TRY(sliding_problem(dtype, L, B, nheads, kv_heads, dh, window, sinks, scale, pr));
    if (L == 0 || B == 0) return ok();
    CIRCATT_TRY(check_threads(sliding_threads(pr, lse != nullptr)));  // lse: a backward will follow
    CIRCATT_TRY(sliding_fwd_arguments(dtype, L, B, nheads, kv_heads, dh, q, q_row, q_batch, k, k_row, k_batch, v, v_row,
                                      v_batch, lengths, y, y_rest, lse, ShapeSpans(), pr));
    return hip_result(launch_sliding_fwd(pr, as_stream(stream)), "circatt_sliding_fwd");
}

int64_t circatt_sliding_bwd_workspace_bytes(int dtype, int64_t L, int64_t B, int64_t nheads, int64_t kv_heads,
                                            int64_t dh, int64_t window, int64_t sinks) {
    SlidingProblem pr;
    if (sliding_problem(dtype, L, B, nheads, kv_heads, dh, window, sinks, 1.f, pr) != CIRCATT_OK) return -1;
    if (L == 0 || B == 0) return 0;
    return check_threads(sliding_threads(pr, true)) == CIRCATT_OK ? 4 * sliding_bwd_workspace_floats(pr) : -1;
}

int circatt_sliding_bwd(int dtype, int64_t L, int64_t B, int64_t nheads, int64_t kv_heads, int64_t dh, int64_t window,
                        int64_t sinks, float scale, const void *q, int64_t q_row, int64_t q_batch, const void *k,
                        int64_t k_row, int64_t k_batch, const void *v, int64_t v_row, int64_t v_batch,
                        const int32_t *lengths, const void *y, const void *y_rest, const float *lse, const void *dy,
                        int64_t dy_row, int64_t dy_batch, void *dq, void *dk, void *dv, void *workspace, int64_t workspace_bytes,
                        void *stream) {
    SlidingProblem pr;
    CIRCATT_TRY(sliding_problem(dtype, L, B, nheads, kv_heads, dh, window, sinks, scale, pr));
    if (L == 0 || B == 0) return ok();
    CIRCATT_TRY(check_threads(sliding_threads(pr, true)));
    CIRCATT_TRY(sliding_bwd_arguments(dtype, L, B, nheads, kv_heads, dh, q, q_row, q_batch, k, k_row, k_batch, v, v_row,
                                      v_batch, lengths, y, y_rest, lse, dy, dy_row, dy_batch, dq, dk, dv, workspace,
                                      workspace_bytes, 4 * sliding_bwd_workspace_floats(pr), ShapeSpans(), pr));
    return hip_result(launch_sliding_bwd(pr, as_stream(stream)), "circatt_sliding_bwd");
}

int circatt_shaped_fwd(int dtype, int64_t L, int64_t B, int64_t nheads, int64_t kv_heads, int64_t dh, int64_t window,
                       int64_t sinks, float scale, float cap, const float *slopes, const int32_t *prefix,
                       const int32_t *places, int64_t places_row, const void *q, int64_t q_row, int64_t q_batch,
                       const void *k, int64_t k_row, int64_t k_batch, const void *v, int64_t v_row, int64_t v_batch,
                       const int32_t *lengths, void *y, void *y_rest, float *lse, void *stream) {
    ShapedSlidingProblem pr{};
    CIRCATT_TRY(sliding_problem(dtype, L, B, nheads, kv_heads, dh, window, sinks, scale, pr));
    CIRCATT_TRY(check_shape(dtype, scale, cap, slopes, prefix, places, places_row, L, pr.shape));
    if (L == 0 || B == 0) return ok();
    CIRCATT_TRY(check_threads(shaped_sliding_threads(pr, masked_by(pr.shape), lse != nullptr)));
    CIRCATT_TRY(sliding_fwd_arguments(dtype, L, B, nheads, kv_heads, dh, q, q_row, q_batch, k, k_row, k_batch, v, v_row,
                                      v_batch, lengths, y, y_rest, lse, ShapeSpans(pr.shape, B, L, nheads), pr));
    return hip_result(launch_shaped_fwd(pr, as_stream(stream)), "circatt_shaped_fwd");
}

int64_t circatt_shaped_bwd_workspace_bytes(int dtype, int64_t L, int64_t B, int64_t nheads, int64_t kv_heads, int64_t dh,
                                           int64_t window, int64_t sinks, int biased, int masked) {
    SlidingProblem pr;
    if (sliding_problem(dtype, L, B, nheads, kv_heads, dh, window, sinks, 1.f, pr) != CIRCATT_OK) return -1;
    if (masked < kUnmasked || masked > kPrefix) {
        fail(CIRCATT_ERR_INVALID, "masked=%d must be 0, 1 or 2", masked);
        return -1;
    }
    if (L == 0 || B == 0) return 0;
    return check_threads(shaped_sliding_threads(pr, masked, true)) == CIRCATT_OK
               ? 4 * shaped_bwd_workspace_floats(pr, biased != 0, masked)
               : -1;
}

int circatt_shaped_bwd(int dtype, int64_t L, int64_t B, int64_t nheads, int64_t kv_heads, int64_t dh, int64_t window,
                       int64_t sinks, float scale, float cap, const float *slopes, const int32_t *prefix,
                       const int32_t *places, int64_t places_row, const void *q, int64_t q_row, int64_t q_batch,
                       const void *k, int64_t k_row, int64_t k_batch, const void *v, int64_t v_row, int64_t v_batch,
                       const int32_t *lengths, const void *y, const void *y_rest, const float *lse, const void *dy,
                       int64_t dy_row, int64_t dy_batch, void *dq, void *dk, void *dv, void *workspace,
                       int64_t workspace_bytes, void *stream) {
    ShapedSlidingProblem pr{};
    CIRCATT_TRY(sliding_problem(dtype, L, B, nheads, kv_heads, dh, window, sinks, scale, pr));
    CIRCATT_TRY(check_shape(dtype, scale, cap, slopes, prefix, places, places_row, L, pr.shape));
    if (L == 0 || B == 0) return ok();
    const int masked = masked_by(pr.shape);
    CIRCATT_TRY(check_threads(shaped_sliding_threads(pr, masked, true)));
    CIRCATT_TRY(sliding_bwd_arguments(dtype, L, B, nheads, kv_heads, dh, q, q_row, q_batch, k, k_row, k_batch, v, v_row,
                                      v_batch, lengths, y, y_rest, lse, dy, dy_row, dy_batch, dq, dk, dv, workspace,
                                      workspace_bytes, 4 * shaped_bwd_workspace_floats(pr, slopes != nullptr, masked),
                                      ShapeSpans(pr.shape, B, L, nheads), pr));
    return hip_result(launch_shaped_bwd(pr, as_stream(stream)), "circatt_shaped_bwd");
}

int64_t circatt_paged_workspace_bytes(int dtype, int64_t T, int64_t B, int64_t nheads, int64_t kv_heads, int64_t dh,
                                      int64_t window, int64_t sinks, int64_t page_size, int64_t max_pages) {
    PagedProblem pr;
    if (paged_problem(dtype, T, B, nheads, kv_heads, dh, window, sinks, 1.f, page_size, max_pages, pr) != CIRCATT_OK)
        return -1;
    return T == 0 ? 0 : 4 * paged_workspace_floats(pr);
}

int64_t circatt_shaped_paged_workspace_bytes(int dtype, int64_t T, int64_t B, int64_t nheads, int64_t kv_heads, int64_t dh,
                                             int64_t window, int64_t sinks, int64_t page_size, int64_t max_pages,
                                             int prefixed) {
    PagedProblem pr;
    if (paged_problem(dtype, T, B, nheads, kv_heads, dh, window, sinks, 1.f, page_size, max_pages, pr) != CIRCATT_OK)
        return -1;
    return T == 0 ? 0 : 4 * paged_workspace_floats(pr, prefixed != 0);
}

namespace {

// Everything of a call over a paged cache but the kinds of its scores and the launch; done: nothing to launch.
int paged_arguments(int dtype, int64_t T, int64_t B, int64_t nheads, int64_t kv_heads, int64_t dh, int64_t window,
                    int64_t sinks, float scale, const void *q, int64_t q_row, const void *cache_k, const void *cache_v,
                    int64_t npages, int64_t page_size, int64_t page_stride, int64_t row_stride, const int32_t *pages,
                    int64_t pages_row, int64_t max_pages, const int32_t *lengths, const int32_t *offsets, void *y,
                    int zero_tail, void *workspace, int64_t workspace_bytes, PagedProblem &pr) {
    CIRCATT_TRY(paged_problem(dtype, T, B, nheads, kv_heads, dh, window, sinks, scale, page_size, max_pages, pr));
    const int es = esize_of(dtype);
    CIRCATT_TRY(paged_table(B, npages, page_size, page_stride, row_stride, kv_heads * dh, pages, pages_row, max_pages,
                            lengths, cache_k, cache_v, es, pr.page_log2));
    if (offsets == nullptr && T != B)
        return fail(CIRCATT_ERR_INVALID, "without offsets q has one row for each sequence: %lld rows, %lld sequences",
                    (long long)T, (long long)B);
    if (T == 0) return CIRCATT_OK;
    CIRCATT_TRY(check_rows("q", q, q_row, 0, nheads * dh, es));
    CIRCATT_TRY(check_rows("y", y, nheads * dh, 0, nheads * dh, es));
    const int64_t need = 4 * paged_workspace_floats(pr);
    if (need > 0) {
        CIRCATT_NONNULL(workspace);
        if (workspace_bytes < need)
            return fail(CIRCATT_ERR_INVALID, "workspace of %lld bytes, %lld needed", (long long)workspace_bytes,
                        (long long)need);
        if (reinterpret_cast<uintptr_t>(workspace) % 16 != 0)
            return fail(CIRCATT_ERR_INVALID, "workspace must be 16-byte aligned");
    }
    // a block writes rows that others still read of the cache, and splits read q again
    const int64_t y_bytes = T * nheads * dh * es, q_bytes = ((T - 1) * q_row + nheads * dh) * es;
    const int64_t cache_bytes = ((npages - 1) * page_stride + (page_size - 1) * row_stride + kv_heads * dh) * es;
    if (overlap(y, y_bytes, q, q_bytes) || overlap(y, y_bytes, cache_k, cache_bytes) ||
        overlap(y, y_bytes, cache_v, cache_bytes))
        return fail(CIRCATT_ERR_INVALID, "y must not overlap q or the caches");
    pr.q = q, pr.q_row = q_row;
    pr.k = cache_k, pr.v = cache_v;
    pr.npages = (int)npages;
    pr.page_stride = page_stride, pr.row_stride = row_stride;
    pr.pages = pages, pr.pages_row = pages_row;
    pr.lengths = lengths, pr.offsets = offsets;
    pr.y = y;
    pr.zero_tail = zero_tail != 0;
    pr.work = static_cast<float *>(workspace);
    return CIRCATT_OK;
}

}  // namespace

int circatt_paged_attention(int dtype, int64_t T, int64_t B, int64_t nheads, int64_t kv_heads, int64_t dh,
                            int64_t window, int64_t sinks, float scale, const void *q, int64_t q_row,
                            const void *cache_k, const void *cache_v, int64_t npages, int64_t page_size,
                            int64_t page_stride, int64_t row_stride, const int32_t *pages, int64_t pages_row,
                            int64_t max_pages, const int32_t *lengths, const int32_t *offsets, void *y, int zero_tail,
                            void *workspace, int64_t workspace_bytes, void *stream) {
    PagedProblem pr;
    CIRCATT_TRY(paged_arguments(dtype, T, B, nheads, kv_heads, dh, window, sinks, scale, q, q_row, cache_k, cache_v, npages,
                                page_size, page_stride, row_stride, pages, pages_row, max_pages, lengths, offsets, y,
                                zero_tail, workspace, workspace_bytes, pr));
    if (T == 0) return ok();
    return hip_result(launch_paged(pr, as_stream(stream)), "circatt_paged_attention");
}

int circatt_shaped_paged(int dtype, int64_t T, int64_t B, int64_t nheads, int64_t kv_heads, int64_t dh, int64_t window,
                         int64_t sinks, float scale, float cap, const float *slopes, const int32_t *prefix, const void *q,
                         int64_t q_row, const void *cache_k, const void *cache_v, int64_t npages, int64_t page_size,
                         int64_t page_stride, int64_t row_stride, const int32_t *pages, int64_t pages_row,
                         int64_t max_pages, const int32_t *lengths, const int32_t *offsets, void *y, int zero_tail,
                         void *workspace, int64_t workspace_bytes, void *stream) {
    ShapedPagedProblem pr{};
    CIRCATT_TRY(paged_arguments(dtype, T, B, nheads, kv_heads, dh, window, sinks, scale, q, q_row, cache_k, cache_v, npages,
                                page_size, page_stride, row_stride, pages, pages_row, max_pages, lengths, offsets, y,
                                zero_tail, workspace, workspace_bytes, pr));
    CIRCATT_TRY(check_shape(dtype, scale, cap, slopes, prefix, nullptr, 0, max_pages * page_size, pr.shape));
    if (T == 0) return ok();
    const ShapeSpans sh(pr.shape, B, 0, nheads);
    CIRCATT_TRY(check_apart({span("y", y, 1, 0, T, nheads * dh, nheads * dh, esize_of(dtype))}, {sh.slopes, sh.prefix}));
    // the plan for prefixes where the workspace holds what it leaves, which may be more than
    // was asked for above
    const bool whole = prefix != nullptr && (workspace != nullptr ? workspace_bytes : 0) >= 4 * paged_workspace_floats(pr, true) &&
                       reinterpret_cast<uintptr_t>(workspace) % 16 == 0;
    return hip_result(launch_shaped_paged(pr, whole, as_stream(stream)), "circatt_shaped_paged");
}

int circatt_paged_append(int dtype, int64_t T, int64_t B, int64_t channels, const void *k, int64_t k_row, const void *v,
                         int64_t v_row, void *cache_k, void *cache_v, int64_t npages, int64_t page_size,
                         int64_t page_stride, int64_t row_stride, const int32_t *pages, int64_t pages_row,
                         int64_t max_pages, const int32_t *lengths, const int32_t *offsets, void *stream) {
    AppendProblem pr{};
    CIRCATT_TRY(check_token_dtype(dtype));
    if (T < 0 || T > INT32_MAX / 2) return fail(CIRCATT_ERR_INVALID, "invalid token count %lld", (long long)T);
    if (channels < 1 || channels > 1 << 24) return fail(CIRCATT_ERR_INVALID, "invalid channel count %lld", (long long)channels);
    pr.esize = esize_of(dtype);
    CIRCATT_TRY(paged_table(B, npages, page_size, page_stride, row_stride, channels, pages, pages_row, max_pages,
                            lengths, cache_k, cache_v, pr.esize, pr.page_log2));
    if (offsets == nullptr && T != B)
        return fail(CIRCATT_ERR_INVALID, "without offsets there is one row for each sequence: %lld rows, %lld sequences",
                    (long long)T, (long long)B);
    if (T == 0) return ok();
    CIRCATT_NONNULL(k);
    CIRCATT_NONNULL(v);
    if (k_row < 0 || v_row < 0) return fail(CIRCATT_ERR_INVALID, "negative stride");
    pr.T = T;
    pr.B = (int)B;
    pr.C = channels;
    pr.k = k, pr.k_row = k_row, pr.v = v, pr.v_row = v_row;
    pr.cache_k = cache_k, pr.cache_v = cache_v;
    pr.page_stride = page_stride, pr.row_stride = row_stride;
    pr.npages = (int)npages;
    pr.pages = pages, pr.pages_row = pages_row, pr.maxp = (int)max_pages;
    pr.lengths = lengths, pr.offsets = offsets;
    CIRCATT_TRY(check_threads(append_threads(pr)));
    return hip_result(launch_append(pr, as_stream(stream)), "circatt_paged_append");
}

namespace {

// The sequences of a cache and what they hold; outputs are contiguous and apart from
// everything that is read.
int page_table(int64_t B, int64_t maxp, int64_t npages, int64_t page_size, const int32_t *pages, int64_t pages_row,
               PageTable &pr) {
    if (B < 1 || B > 65535) return fail(CIRCATT_ERR_INVALID, "invalid sequence count %lld", (long long)B);
    if (page_size < 1 || page_size > 65536 || (page_size & (page_size - 1)) != 0)
        return fail(CIRCATT_ERR_UNSUPPORTED, "page size %lld must be a power of two up to 65536", (long long)page_size);
    if (npages < 1 || npages > INT32_MAX / page_size)
        return fail(CIRCATT_ERR_INVALID, "a cache of %lld pages of %lld tokens", (long long)npages, (long long)page_size);
    for (pr.page_log2 = 0; (1 << pr.page_log2) < page_size;) ++pr.page_log2;
    if (maxp < 1 || pages_row < maxp || maxp > (int64_t)1 << (30 - pr.page_log2))
        return fail(CIRCATT_ERR_INVALID, "a page table of %lld pages, rows of %lld", (long long)maxp, (long long)pages_row);
    if (maxp + 1 > INT32_MAX / B)  // pages that all sequences may ask for are counted in 32 bits
        return fail(CIRCATT_ERR_UNSUPPORTED, "a table of %lld sequences with %lld pages", (long long)B, (long long)maxp);
    CIRCATT_NONNULL(pages);
    pr.B = (int)B;
    pr.maxp = (int)maxp;
    pr.npages = (int)npages;
    pr.pages = pages, pr.pages_row = pages_row;
    return CIRCATT_OK;
}
Span ints(const char *name, const void *p, int64_t n) { return Span{name, p, 4 * n}; }

int page_shape(int dtype, int64_t channels, int64_t B, int64_t npages, int64_t page_size, int64_t page_stride,
               int64_t row_stride, const int32_t *pages, int64_t pages_row, int64_t maxp, const int32_t *lengths,
               void *cache_k, void *cache_v, PageShape &sh) {
    CIRCATT_TRY(check_token_dtype(dtype));
    if (channels < 1 || channels > 1 << 24) return fail(CIRCATT_ERR_INVALID, "invalid channel count %lld", (long long)channels);
    int log2;
    CIRCATT_TRY(paged_table(B, npages, page_size, page_stride, row_stride, channels, pages, pages_row, maxp, lengths,
                            cache_k, cache_v, esize_of(dtype), log2));
    if (page_size * channels > INT32_MAX)
        return fail(CIRCATT_ERR_UNSUPPORTED, "a page of %lld values", (long long)(page_size * channels));
    // tokens move: rows that lie in one another would be written twice
    if ((page_size > 1 && row_stride < channels) || (npages > 1 && page_stride < (page_size - 1) * row_stride + channels))
        return fail(CIRCATT_ERR_INVALID, "the cache's pages must not overlap");
    sh.esize = esize_of(dtype);
    sh.C = channels;
    sh.cache_k = cache_k, sh.cache_v = cache_v;
    sh.page_stride = page_stride, sh.row_stride = row_stride;
    return CIRCATT_OK;
}
int check_page_workspace(const void *workspace, int64_t bytes, int64_t need) {
    CIRCATT_NONNULL(workspace);
    if (bytes < need)
        return fail(CIRCATT_ERR_INVALID, "workspace of %lld bytes, %lld needed", (long long)bytes, (long long)need);
    if (reinterpret_cast<uintptr_t>(workspace) % 16 != 0) return fail(CIRCATT_ERR_INVALID, "workspace must be 16-byte aligned");
    return CIRCATT_OK;
}

}  // namespace

int circatt_paged_fork(int64_t B, int64_t npages, int64_t page_size, const int32_t *pages, int64_t pages_row,
                       int64_t max_pages, const int32_t *lengths, const int32_t *counts, int64_t N, const int32_t *source,
                       int32_t *out_pages, int32_t *out_lengths, int32_t *out_counts, void *stream) {
    ForkProblem pr{};
    CIRCATT_TRY(page_table(B, max_pages, npages, page_size, pages, pages_row, pr));
    if (N < 0 || N > 65535) return fail(CIRCATT_ERR_INVALID, "invalid sequence count %lld", (long long)N);
    CIRCATT_NONNULL(lengths);
    CIRCATT_NONNULL(counts);
    CIRCATT_NONNULL(out_counts);
    if (N > 0) {
        CIRCATT_NONNULL(source);
        CIRCATT_NONNULL(out_pages);
        CIRCATT_NONNULL(out_lengths);
    }
    CIRCATT_TRY(check_apart({ints("out_pages", out_pages, N * max_pages), ints("out_lengths", out_lengths, N),
                             ints("out_counts", out_counts, npages)},
                            {ints("pages", pages, (B - 1) * pages_row + max_pages), ints("lengths", lengths, B),
                             ints("counts", counts, npages), ints("source", source, N)}));
    pr.lengths = lengths, pr.counts = counts;
    pr.N = (int)N;
    pr.source = source;
    pr.out_pages = out_pages, pr.out_lengths = out_lengths, pr.out_counts = out_counts;
    return hip_result(launch_fork(pr, as_stream(stream)), "circatt_paged_fork");
}

int64_t circatt_paged_resize_workspace_bytes(int64_t B, int64_t npages) {
    if (B < 1 || B > 65535 || npages < 1 || npages > INT32_MAX) return -1;
    return 4 * resize_workspace_ints(B, npages);
}

int circatt_paged_resize(int dtype, int64_t channels, void *cache_k, void *cache_v, int64_t npages, int64_t page_size,
                         int64_t page_stride, int64_t row_stride, int64_t B, const int32_t *pages, int64_t pages_row,
                         int64_t max_pages, const int32_t *lengths, const int32_t *counts, const int32_t *to,
                         int32_t *out_pages, int32_t *out_lengths, int32_t *out_counts, void *workspace,
                         int64_t workspace_bytes, void *stream) {
    ResizeProblem pr{};
    CIRCATT_TRY(page_table(B, max_pages, npages, page_size, pages, pages_row, pr));
    CIRCATT_NONNULL(lengths);
    CIRCATT_TRY(page_shape(dtype, channels, B, npages, page_size, page_stride, row_stride, pages, pages_row, max_pages,
                           lengths, cache_k, cache_v, pr.shape));
    CIRCATT_NONNULL(counts);
    CIRCATT_NONNULL(to);
    CIRCATT_NONNULL(out_pages);
    CIRCATT_NONNULL(out_lengths);
    CIRCATT_NONNULL(out_counts);
    const int64_t need = 4 * resize_workspace_ints(B, npages);
    CIRCATT_TRY(check_page_workspace(workspace, workspace_bytes, need));
    CIRCATT_TRY(check_apart({ints("out_pages", out_pages, B * max_pages), ints("out_lengths", out_lengths, B),
                             ints("out_counts", out_counts, npages), Span{"workspace", workspace, need}},
                            {ints("pages", pages, (B - 1) * pages_row + max_pages), ints("lengths", lengths, B),
                             ints("counts", counts, npages), ints("to", to, B)}));
    pr.lengths = lengths, pr.counts = counts;
    pr.to = to;
    pr.out_pages = out_pages, pr.out_lengths = out_lengths, pr.out_counts = out_counts;
    return hip_result(launch_resize(pr, static_cast<int32_t *>(workspace), as_stream(stream)), "circatt_paged_resize");
}

int64_t circatt_paged_compact_workspace_bytes(int64_t npages) {
    return npages < 1 || npages > INT32_MAX ? -1 : 4 * compact_workspace_ints(npages);
}

int circatt_paged_compact(int dtype, int64_t channels, void *cache_k, void *cache_v, int64_t npages, int64_t page_size,
                          int64_t page_stride, int64_t row_stride, int64_t B, const int32_t *pages, int64_t pages_row,
                          int64_t max_pages, const int32_t *counts, int32_t *out_pages, int32_t *out_counts,
                          void *workspace, int64_t workspace_bytes, void *stream) {
    CompactProblem pr{};
    CIRCATT_TRY(page_table(B, max_pages, npages, page_size, pages, pages_row, pr));
    CIRCATT_TRY(page_shape(dtype, channels, B, npages, page_size, page_stride, row_stride, pages, pages_row, max_pages,
                           pages, cache_k, cache_v, pr.shape));
    CIRCATT_NONNULL(counts);
    CIRCATT_NONNULL(out_pages);
    CIRCATT_NONNULL(out_counts);
    const int64_t need = 4 * compact_workspace_ints(npages);
    CIRCATT_TRY(check_page_workspace(workspace, workspace_bytes, need));
    CIRCATT_TRY(check_apart({ints("out_pages", out_pages, B * max_pages), ints("out_counts", out_counts, npages),
                             Span{"workspace", workspace, need}},
                            {ints("pages", pages, (B - 1) * pages_row + max_pages), ints("counts", counts, npages)}));
    pr.counts = counts;
    pr.out_pages = out_pages, pr.out_counts = out_counts;
    return hip_result(launch_compact(pr, static_cast<int32_t *>(workspace), as_stream(stream)), "circatt_paged_compact");
}

int circatt_axial_rotary(int dtype, int inverse, int interleaved, int naxes, int64_t n1, int64_t n2, int64_t n3,
                         int64_t P, int64_t nb, int64_t nheads, int64_t dh, int32_t p1, int32_t p2, int32_t p3,
                         float base, const void *x, int64_t x_row, const int32_t *positions, int64_t pos_batch,
                         void *y, void *stream) {
    return circatt_axial_rotary_wide(dtype, inverse, interleaved, naxes, n1, n2, n3, P, nb, nheads, dh, p1, p2, p3, base,
                                     0.f, x, x_row, positions, pos_batch, y, stream);
}

int circatt_axial_rotary_wide(int dtype, int inverse, int interleaved, int naxes, int64_t n1, int64_t n2, int64_t n3,
                              int64_t P, int64_t nb, int64_t nheads, int64_t dh, int32_t p1, int32_t p2, int32_t p3,
                              float base, float base_rest, const void *x, int64_t x_row, const int32_t *positions,
                              int64_t pos_batch, void *y, void *stream) {
    CIRCATT_TRY(check_token_dtype(dtype));
    if (naxes < 1 || naxes > 3) return fail(CIRCATT_ERR_INVALID, "naxes=%d must be 1, 2 or 3", naxes);
    if (nheads < 1 || nheads > 65536 || dh < 2 || dh % 2 != 0 || dh > 65536 || nheads * dh > 1 << 24)
        return fail(CIRCATT_ERR_INVALID, "invalid heads: %lld of %lld channels (even)", (long long)nheads, (long long)dh);
    RotaryProblem pr{};
    const int32_t p[3] = {p1, naxes > 1 ? p2 : 0, naxes > 2 ? p3 : 0};
    int64_t total = 0;
    for (int a = 0; a < naxes; ++a) {
        if (p[a] < 1) return fail(CIRCATT_ERR_INVALID, "axis %d has %d pairs: at least one is needed", a + 1, p[a]);
        total += p[a];
    }
    if (2 * total > dh)
        return fail(CIRCATT_ERR_INVALID, "%lld pairs do not fit heads of %lld channels", (long long)total, (long long)dh);
    if (total > kMaxPairs)
        return fail(CIRCATT_ERR_UNSUPPORTED, "%lld pairs: at most %d are supported", (long long)total, kMaxPairs);
    const double whole = (double)base + (double)base_rest;
    if (!(base > 0.f) || !(whole > 0) || !std::isfinite(whole))
        return fail(CIRCATT_ERR_INVALID, "base=%g must be positive and finite", whole);
    if (P < 0 || nb < 0 || P > INT32_MAX / 2 || nb > INT32_MAX || (nb > 0 && P > (int64_t)INT32_MAX / nb))
        return fail(CIRCATT_ERR_INVALID, "invalid sizes P=%lld, nb=%lld", (long long)P, (long long)nb);
    if (positions == nullptr) {
        const int64_t n[3] = {n1, naxes > 1 ? n2 : 1, naxes > 2 ? n3 : 1};
        int64_t prod = 1;
        for (int64_t m : n) {
            if (m < 0 || m > INT32_MAX / 2) return fail(CIRCATT_ERR_INVALID, "invalid grid size %lld", (long long)m);
            prod = m > 0 && prod > INT32_MAX / m ? INT32_MAX : prod * m;
        }
        if (prod != P) return fail(CIRCATT_ERR_INVALID, "a grid of %lld pixels for %lld tokens", (long long)prod, (long long)P);
        pr.n1 = (int)n[0];
        pr.n2 = (int)n[1];
    } else {
        if (pos_batch != 0 && pos_batch < P * naxes)
            return fail(CIRCATT_ERR_INVALID, "positions: images %lld apart hold %lld", (long long)pos_batch, (long long)(P * naxes));
        pr.n1 = pr.n2 = 1;
    }
    if (P == 0 || nb == 0) return ok();
    CIRCATT_NONNULL(x);
    CIRCATT_NONNULL(y);
    if (x_row < nheads * dh)
        return fail(CIRCATT_ERR_INVALID, "x: token stride %lld below %lld channels", (long long)x_row, (long long)(nheads * dh));
    const int es = esize_of(dtype);
    const int64_t C = nheads * dh;
    if (x == y || overlap(y, nb * P * C * es, x, ((nb * P - 1) * x_row + C) * es))
        return fail(CIRCATT_ERR_INVALID, "y must not alias x");
    pr.dtype = dtype;
    pr.inverse = inverse != 0;
    pr.interleaved = interleaved != 0;
    pr.naxes = naxes;
    pr.P = P;
    pr.nb = nb;
    pr.H = (int)nheads;
    pr.D = (int)dh;
    pr.x = x;
    pr.x_row = x_row;
    pr.positions = positions;
    pr.pos_batch = pos_batch;
    pr.y = y;
    pr.npairs = (int)total;
    int at = 0;
    for (int a = 0; a < naxes; ++a) {
        pr.pairs[a] = p[a];
        for (int i = 0; i < p[a]; ++i)
            pr.turns[at++] = std::pow(whole, -(double)i / p[a]) / 6.283185307179586476925;
    }
    CIRCATT_TRY(check_threads(rotary_threads(pr)));
    return hip_result(launch_rotary(pr, as_stream(stream)), "circatt_axial_rotary");
}

int circatt_memcpy(void *dst, const void *src, int64_t bytes, int kind) {
    static const hipMemcpyKind kinds[] = {hipMemcpyHostToDevice, hipMemcpyDeviceToHost,
                                          hipMemcpyDeviceToDevice};
    if (kind < 0 || kind > 2) return fail(CIRCATT_ERR_INVALID, "memcpy kind %d", kind);
    if (bytes < 0) return fail(CIRCATT_ERR_INVALID, "negative size");
    if (bytes == 0) return ok();
    CIRCATT_NONNULL(dst);
    CIRCATT_NONNULL(src);
    return hip_result(hipMemcpy(dst, src, (size_t)bytes, kinds[kind]), "circatt_memcpy");
}

int circatt_stream_synchronize(void *stream) {
    return hip_result(hipStreamSynchronize(as_stream(stream)), "circatt_stream_synchronize");
}

}  // extern "C"
