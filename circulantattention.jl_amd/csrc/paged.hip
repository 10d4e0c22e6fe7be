// Attention of new tokens over a paged cache, and the cache's append.
#include "token_rows.h"

namespace circatt {
namespace {

using namespace tok;
constexpr float kLog2e = 1.4426950408889634f;

// The sequence that row t of the packed new tokens belongs to (B: behind the
// last one), with the token's position and the first row of the sequence.
struct NewToken {
    int b, pos;
};
__device__ __forceinline__ NewToken new_token(const int32_t *offsets, const int32_t *lengths, int B, int64_t t) {
    int b = (int)t;
    if (offsets == nullptr) return NewToken{b, b < B ? lengths[b] - 1 : -1};
    int lo = 0, hi = B;  // the first b with offsets[b + 1] > t
    while (lo < hi) {
        const int mid = (lo + hi) >> 1;
        if (offsets[mid + 1] > t) hi = mid;
        else lo = mid + 1;
    }
    b = lo;
    if (b == B || t < offsets[b]) return NewToken{B, -1};
    return NewToken{b, lengths[b] - offsets[b + 1] + (int)t};
}

template <typename T>
__global__ __launch_bounds__(256) void paged_rows(PagedProblem pr) {
    const int64_t r = (int64_t)blockIdx.x * 4 + (threadIdx.x >> 6);
    if (r >= pr.T * pr.H) return;
    const int64_t t = r / pr.H;
    const int h = (int)(r - t * pr.H);
    NewToken w = new_token(pr.offsets, pr.lengths, pr.B, t);
    if (w.b == pr.B && !pr.zero_tail) return;
    // a position outside the sequence's pages: the row sees nothing
    int64_t held = (int64_t)pr.maxp << pr.page_log2;
    if (w.pos >= held) w.pos = -1;
    const int64_t head = (int64_t)(h / pr.G) * pr.D;
    const PagedKV<T> kv{static_cast<const T *>(pr.k) + head, static_cast<const T *>(pr.v) + head, pr.page_stride,
                        pr.row_stride, pr.pages + (w.b < pr.B ? w.b : 0) * pr.pages_row, pr.npages, pr.page_log2};
    forward_row(static_cast<const T *>(pr.q) + t * pr.q_row + (int64_t)h * pr.D,
                static_cast<T *>(pr.y) + (t * pr.H + h) * pr.D, nullptr, kv, w.pos, pr.W, pr.S, pr.D,
                pr.scale * kLog2e);
}

typedef uint32_t u4 __attribute__((ext_vector_type(4)));

// One wavefront a token: its k, then its v, in units of U.
template <typename U>
__global__ __launch_bounds__(256) void append_rows(AppendProblem pr) {
    const int64_t t = (int64_t)blockIdx.x * 4 + (threadIdx.x >> 6);
    if (t >= pr.T) return;
    const NewToken w = new_token(pr.offsets, pr.lengths, pr.B, t);
    if (w.b == pr.B || w.pos < 0 || (w.pos >> pr.page_log2) >= pr.maxp) return;
    const int pg = pr.pages[w.b * pr.pages_row + (w.pos >> pr.page_log2)];
    if ((unsigned)pg >= (unsigned)pr.npages) return;
    const int64_t at = (pg * pr.page_stride + (w.pos & ((1 << pr.page_log2) - 1)) * pr.row_stride) * pr.esize;
    const int units = (int)(pr.C * pr.esize / (int)sizeof(U));
    const U *k = reinterpret_cast<const U *>(static_cast<const char *>(pr.k) + t * pr.k_row * pr.esize);
    const U *v = reinterpret_cast<const U *>(static_cast<const char *>(pr.v) + t * pr.v_row * pr.esize);
    U *ck = reinterpret_cast<U *>(static_cast<char *>(pr.cache_k) + at);
    U *cv = reinterpret_cast<U *>(static_cast<char *>(pr.cache_v) + at);
    for (int i = threadIdx.x & 63; i < units; i += 64) {
        ck[i] = k[i];
        cv[i] = v[i];
    }
}

}  // namespace

int64_t paged_workspace_floats(const PagedProblem &) { return 0; }

hipError_t launch_paged(const PagedProblem &pr, hipStream_t s) {
    const unsigned blocks = (unsigned)((pr.T * pr.H + 3) / 4);
    if (pr.dtype == CIRCATT_F32) paged_rows<float><<<blocks, 256, 0, s>>>(pr);
    else if (pr.dtype == CIRCATT_F16) paged_rows<_Float16><<<blocks, 256, 0, s>>>(pr);
    else paged_rows<__bf16><<<blocks, 256, 0, s>>>(pr);
    return hipGetLastError();
}

hipError_t launch_append(const AppendProblem &pr, hipStream_t s) {
    const unsigned blocks = (unsigned)((pr.T + 3) / 4);
    // the widest unit that divides every address, row and stride
    const uint64_t all = reinterpret_cast<uint64_t>(pr.k) | reinterpret_cast<uint64_t>(pr.v) |
                         reinterpret_cast<uint64_t>(pr.cache_k) | reinterpret_cast<uint64_t>(pr.cache_v) |
                         (uint64_t)((pr.C | pr.k_row | pr.v_row | pr.page_stride | pr.row_stride) * pr.esize);
    if (all % 16 == 0) append_rows<u4><<<blocks, 256, 0, s>>>(pr);
    else if (all % 4 == 0) append_rows<uint32_t><<<blocks, 256, 0, s>>>(pr);
    else append_rows<uint16_t><<<blocks, 256, 0, s>>>(pr);
    return hipGetLastError();
}

}  // namespace circatt
