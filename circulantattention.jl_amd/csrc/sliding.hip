// Causal sliding-window attention with sinks on (batch, length, channels)
// signals, forward and backward: one wavefront a row.
#include "token_rows.h"

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

template <typename T>
__global__ __launch_bounds__(256) void sliding_fwd_rows(SlidingProblem pr) {
    const int64_t r = (int64_t)blockIdx.x * 4 + (threadIdx.x >> 6);
    if (r >= (int64_t)pr.B * pr.L * pr.H) return;
    const Row<T> w(pr, r);
    T *y = static_cast<T *>(pr.y) + ((int64_t)w.b * pr.L + w.i) * pr.H * pr.D + w.channel(pr);
    forward_row(static_cast<const T *>(pr.q) + w.b * pr.q_batch + w.i * pr.q_row + w.channel(pr), y,
                pr.lse ? pr.lse + w.stat : nullptr, w.kv, w.i < w.n ? w.i : -1, pr.W, pr.S, pr.D, pr.scale * kLog2e);
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

template <int DT>
hipError_t forward(const SlidingProblem &pr, hipStream_t s) {
    const int64_t rows = (int64_t)pr.B * pr.L * pr.H;
    sliding_fwd_rows<typename Elem<DT>::T><<<(unsigned)((rows + 3) / 4), 256, 0, s>>>(pr);
    return hipGetLastError();
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
