// Attention over a paged cache with plain scores (paged_impl.h), and the cache's append.
#include "paged_impl.h"

namespace circatt {
namespace {

// The sequence that row t of the packed new tokens belongs to (B: behind the
// last one), with the token's position and the first row of the sequence.
struct NewToken {
    int b, pos;
};
__device__ __forceinline__ NewToken new_token(const int32_t *offsets, const int32_t *lengths, int B, int64_t t) {
    int b = (int)t;
    if (offsets == nullptr) return NewToken{b, b < B && lengths[b] > 0 ? lengths[b] - 1 : -1};
    int lo = 0, hi = B;  // the first b with offsets[b + 1] > t
    while (lo < hi) {
        const int mid = (lo + hi) >> 1;
        if (offsets[mid + 1] > t) hi = mid;
        else lo = mid + 1;
    }
    b = lo;
    if (b == B || offsets[b] < 0 || t < offsets[b]) return NewToken{B, -1};
    return NewToken{b, (lengths[b] > 0 ? lengths[b] : 0) - offsets[b + 1] + (int)t};
}

// ---------------------------------------------------------------------------
// Append.
typedef uint32_t u4 __attribute__((ext_vector_type(4)));

// One wavefront a token: its k, then its v, in units of U.  Bound by memory: chunks of
// 4 x 4096 tokens of 1024 channels, bf16, 21.7 us with the call, 4.8 TB/s.
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

int64_t paged_workspace_floats(const PagedProblem &pr, bool whole) { return paged_plan(pr, whole).floats; }

int64_t paged_threads(const PagedProblem &pr) {
    const PagedPlan pl = paged_plan(pr);
    // and the workgroups for the rows behind the last sequence
    return 512 * ((int64_t)(pl.chunk ? pl.chunk_grid.blocks : 0) + pl.few_grid.blocks + 8);
}

hipError_t launch_paged(const PagedProblem &pr, hipStream_t s) { return launch_of<Plain>(pr, paged_plan(pr), s); }

int64_t append_threads(const AppendProblem &pr) { return (pr.T + 3) / 4 * 256; }

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
