// The pages of a cache: which sequences hold which, and the tokens in them.
//
//   fork     sequences go on from others and share their pages; counts (of a page's
//            holders) follow.  No token moves.
//   resize   sequences give pages back or get free ones, the lowest numbers first; a
//            sequence that goes on in a part page which others hold gets its own copy.
//   compact  pages that are held move to the lowest numbers.
//
// All of it is whole numbers, and sums of them by atomics do not hang on their order:
// results are the same from call to call.  Nothing is read from or written to pages
// outside the cache, whatever the tables hold.
//
// The tables of a serving batch are some 100 KB, so the time is that of launches and of
// the chain from load to load.  Each call is two launches: a plan by one workgroup, whose
// barriers stand between its steps, and the work of it by many.
#include "token_kernels.h"

namespace circatt {
namespace {

typedef int i4 __attribute__((ext_vector_type(4)));
typedef uint32_t u4 __attribute__((ext_vector_type(4)));

__device__ __forceinline__ bool is_page(int p, int npages) { return (unsigned)p < (unsigned)npages; }
// Pages that n tokens reach, of a table of maxp.
__device__ __forceinline__ int reach(int n, int page_log2, int maxp) {
    const int p = n <= 0 ? 0 : (int)(((int64_t)n + (1 << page_log2) - 1) >> page_log2);
    return p < maxp ? p : maxp;
}

// ---------------------------------------------------------------------------
// Fork.  The first launch writes the new rows and the old counts, the second adds to
// the pages of every old sequence how many have taken it, less itself.
__global__ __launch_bounds__(256) void fork_rows(ForkProblem pr) {
    const int64_t step = (int64_t)gridDim.x * 256, at = (int64_t)blockIdx.x * 256 + threadIdx.x;
    for (int64_t i = at; i < (int64_t)pr.N * pr.maxp; i += step) {
        const int n = (int)(i / pr.maxp), e = (int)(i - (int64_t)n * pr.maxp), b = pr.source[n];
        int p = -1;
        if ((unsigned)b < (unsigned)pr.B && e < reach(pr.lengths[b], pr.page_log2, pr.maxp)) p = pr.pages[b * pr.pages_row + e];
        pr.out_pages[i] = p;
    }
    for (int64_t i = at; i < pr.N; i += step) {
        const int b = pr.source[i];
        pr.out_lengths[i] = (unsigned)b < (unsigned)pr.B ? pr.lengths[b] : 0;
    }
    for (int64_t i = at; i < pr.npages; i += step) pr.out_counts[i] = pr.counts[i];
}
__global__ __launch_bounds__(256) void fork_counts(ForkProblem pr) {
    __shared__ int sums[4];
    const int b = blockIdx.x, lane = threadIdx.x & 63;
    int takers = 0;
    for (int n = threadIdx.x; n < pr.N; n += 256) takers += pr.source[n] == b;
    for (int m = 32; m; m >>= 1) takers += __shfl_xor(takers, m, 64);
    if (lane == 0) sums[threadIdx.x >> 6] = takers;
    __syncthreads();
    const int more = sums[0] + sums[1] + sums[2] + sums[3] - 1;
    if (more == 0) return;
    const int has = reach(pr.lengths[b], pr.page_log2, pr.maxp);
    for (int e = threadIdx.x; e < has; e += 256) {
        const int p = pr.pages[b * pr.pages_row + e];
        if (is_page(p, pr.npages)) atomicAdd(pr.out_counts + p, more);
    }
}

// ---------------------------------------------------------------------------
// One workgroup's sums over its threads in order: the sum before this thread's x, and
// that of all.
constexpr int kPlan = 1024;
struct BlockSum {
    int before, all;
};
__device__ __forceinline__ BlockSum block_sum(int x, int *waves) {
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    int s = x;
#pragma unroll
    for (int m = 1; m < 64; m <<= 1) {
        const int o = __shfl_up(s, m, 64);
        if (lane >= m) s += o;
    }
    __syncthreads();  // (the sums of the call before are read)
    if (lane == 63) waves[wave] = s;
    __syncthreads();
    BlockSum r{s - x, 0};
#pragma unroll
    for (int w = 0; w < kPlan / 64; ++w) {
        const int v = waves[w];
        r.before += w < wave ? v : 0;
        r.all += v;
    }
    return r;
}

// Pages per thread and round of a walk over the counts.
constexpr int kEach = 16;
// The counts of a thread's pages [i0, i0 + kEach), those behind the cache as held.
__device__ __forceinline__ void load_counts(const int32_t *counts, int64_t i0, int npages, int (&c)[kEach]) {
    if (i0 + kEach <= npages && reinterpret_cast<uintptr_t>(counts) % 16 == 0) {
#pragma unroll
        for (int k = 0; k < kEach; k += 4) {
            const i4 v = *reinterpret_cast<const i4 *>(counts + i0 + k);
#pragma unroll
            for (int y = 0; y < 4; ++y) c[k + y] = v[y];
        }
    } else {
#pragma unroll
        for (int k = 0; k < kEach; ++k) c[k] = i0 + k < npages ? counts[i0 + k] : 1;
    }
}

// A sequence's change of size.
struct Change {
    int from, to, has, wants, last;  // tokens, pages; the page that its last token is in
    __device__ __forceinline__ Change(const ResizeProblem &pr, int b) {
        const int64_t held = (int64_t)pr.maxp << pr.page_log2;
        const int n = pr.lengths[b], t = pr.to[b];
        from = n < 0 ? 0 : n < held ? n : (int)held;
        to = t < 0 ? from : t < held ? t : (int)held;
        has = reach(from, pr.page_log2, pr.maxp);
        wants = reach(to, pr.page_log2, pr.maxp);
        last = has > 0 ? pr.pages[b * pr.pages_row + has - 1] : -1;
    }
};

// Resize, plan: the counts less the pages given back, then what every sequence needs
// and where its pages begin in the list of free ones (ranks: -1 for a sequence that
// stays as it is), then that list.
__global__ __launch_bounds__(kPlan) void resize_plan(ResizeProblem pr) {
    __shared__ int waves[kPlan / 64];
    const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
    for (int64_t i = (int64_t)tid; i < pr.npages; i += kPlan) pr.out_counts[i] = pr.counts[i];
    __threadfence();
    __syncthreads();
    // a wavefront a sequence
    for (int b = wave; b < pr.B; b += kPlan / 64) {
        const Change c(pr, b);
        for (int e = c.wants + lane; e < c.has; e += 64) {
            const int p = pr.pages[b * pr.pages_row + e];
            if (is_page(p, pr.npages)) atomicAdd(pr.out_counts + p, -1);
        }
    }
    // the counts are read again from here on, past what this compute unit may hold of them
    __threadfence();
    __syncthreads();
    int64_t asked = 0;
    for (int b0 = 0; b0 < pr.B; b0 += kPlan) {
        const int b = b0 + tid;
        int need = 0, copy = 0;
        if (b < pr.B) {
            const Change c(pr, b);
            copy = c.to > c.from && (c.from & ((1 << pr.page_log2) - 1)) != 0 && is_page(c.last, pr.npages) &&
                   __hip_atomic_load(pr.out_counts + c.last, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT) > 1;
            need = copy + (c.wants > c.has ? c.wants - c.has : 0);
        }
        const BlockSum s = block_sum(need, waves);
        if (b < pr.B) {
            const int64_t first = asked + s.before;
            pr.ranks[b] = (int)(first < INT32_MAX / 2 ? first : INT32_MAX / 2);
            pr.needs[b] = copy ? -need : need;
        }
        asked += s.all;
    }
    int64_t found = 0;
    for (int64_t p0 = 0; p0 < pr.npages && found < asked; p0 += (int64_t)kPlan * kEach) {
        int c[kEach], n = 0;
        const int64_t i0 = p0 + (int64_t)tid * kEach;
        load_counts(pr.out_counts, i0, pr.npages, c);
#pragma unroll
        for (int k = 0; k < kEach; ++k) n += c[k] == 0;
        const BlockSum s = block_sum(n, waves);
        int64_t rank = found + s.before;
#pragma unroll
        for (int k = 0; k < kEach; ++k)
            if (c[k] == 0) pr.free_list[rank++] = (int)(i0 + k);
        found += s.all;
    }
    // (own entries: written by this thread above)
    for (int b = tid; b < pr.B; b += kPlan) {
        const int need = pr.needs[b] < 0 ? -pr.needs[b] : pr.needs[b];
        if (need > 0 && (int64_t)pr.ranks[b] + need > found) pr.ranks[b] = -1;
    }
}

// Rows [0, rows) of page `from` to page `to` of one cache, by `threads` threads.
template <typename U>
__device__ __forceinline__ void copy_rows(char *cache, const PageShape &sh, int from, int to, int rows, int tid, int threads) {
    const int units = (int)(sh.C * sh.esize / (int)sizeof(U));
    const char *s = cache + (int64_t)from * sh.page_stride * sh.esize;
    char *d = cache + (int64_t)to * sh.page_stride * sh.esize;
    const int64_t row = sh.row_stride * sh.esize;
    for (int i = tid; i < rows * units; i += threads) {
        const int r = i / units, u = i - r * units;
        reinterpret_cast<U *>(d + r * row)[u] = reinterpret_cast<const U *>(s + r * row)[u];
    }
}
__device__ __forceinline__ void copy_page(const PageShape &sh, bool v, int from, int to, int rows, int tid, int threads) {
    char *cache = static_cast<char *>(v ? sh.cache_v : sh.cache_k);
    const int64_t width = sh.C * sh.esize;
    if (width % 16 == 0) copy_rows<u4>(cache, sh, from, to, rows, tid, threads);
    else if (width % 4 == 0) copy_rows<uint32_t>(cache, sh, from, to, rows, tid, threads);
    else copy_rows<uint16_t>(cache, sh, from, to, rows, tid, threads);
}

// Resize, work: a workgroup a sequence, and another for the copy of its values.
__global__ __launch_bounds__(256) void resize_apply(ResizeProblem pr) {
    const int b = blockIdx.x, tid = threadIdx.x;
    const Change c(pr, b);
    const int rank = pr.ranks[b], need = pr.needs[b];
    const bool copy = need < 0 && rank >= 0, stays = need != 0 && rank < 0;
    const int wants = stays ? c.has : c.wants, fresh = copy ? pr.free_list[rank] : -1;
    const int rows = c.from & ((1 << pr.page_log2) - 1);
    if (blockIdx.y == 0) {
        const int32_t *row = pr.pages + b * pr.pages_row;
        const int32_t *list = pr.free_list + rank + (copy ? 1 : 0) - c.has;
        for (int e = tid; e < pr.maxp; e += 256) {
            int p = -1;
            if (e < wants) {
                p = e < c.has ? row[e] : list[e];
                if (copy && e == c.has - 1) p = fresh;
                if (e >= c.has || (copy && e == c.has - 1)) pr.out_counts[p] = 1;
            }
            pr.out_pages[(int64_t)b * pr.maxp + e] = p;
        }
        if (tid == 0) {
            pr.out_lengths[b] = stays ? c.from : c.to;
            if (copy) atomicAdd(pr.out_counts + c.last, -1);
        }
    }
    if (copy) copy_page(pr.shape, blockIdx.y != 0, c.last, fresh, rows, tid, 256);
}

// ---------------------------------------------------------------------------
// Compact, plan: `used`, the number of pages held; below it the pages that take each
// place (whence: itself, or the page that moves there), and a moved page's new number
// (whither).  The i-th place that is free below `used` gets the i-th held page behind.
__global__ __launch_bounds__(kPlan) void compact_plan(CompactProblem pr) {
    __shared__ int waves[kPlan / 64];
    const int tid = threadIdx.x;
    int used = 0;
    for (int64_t p0 = 0; p0 < pr.npages; p0 += (int64_t)kPlan * kEach) {
        int c[kEach], n = 0;
        const int64_t i0 = p0 + (int64_t)tid * kEach;
        load_counts(pr.counts, i0, pr.npages, c);
#pragma unroll
        for (int k = 0; k < kEach; ++k) n += i0 + k < pr.npages && c[k] > 0;
        used += block_sum(n, waves).all;
    }
    int holes = 0, movers = 0;
    for (int64_t p0 = 0; p0 < pr.npages; p0 += (int64_t)kPlan * kEach) {
        int c[kEach], h = 0, m = 0;
        const int64_t i0 = p0 + (int64_t)tid * kEach;
        load_counts(pr.counts, i0, pr.npages, c);
#pragma unroll
        for (int k = 0; k < kEach; ++k) {
            h += i0 + k < used && c[k] <= 0;
            m += i0 + k >= used && i0 + k < pr.npages && c[k] > 0;
        }
        const BlockSum sh = block_sum(h, waves), sm = block_sum(m, waves);
        int hr = holes + sh.before, mr = movers + sm.before;
#pragma unroll
        for (int k = 0; k < kEach; ++k) {
            const int p = (int)(i0 + k);
            if (i0 + k < used && c[k] <= 0) pr.holes[hr++] = p;
            if (i0 + k >= used && i0 + k < pr.npages && c[k] > 0) {
                pr.movers[mr] = p;
                pr.rank[p] = mr++;
            }
        }
        holes += sh.all;
        movers += sm.all;
    }
    if (tid == 0) {
        pr.sizes[0] = used;
        pr.sizes[1] = movers;
    }
}

// Compact, work: pages move by parts of some rows, the table's numbers and the counts
// follow.
__global__ __launch_bounds__(256) void compact_apply(CompactProblem pr) {
    const int tid = threadIdx.x, used = pr.sizes[0], moved = pr.sizes[1];
    const int64_t step = (int64_t)gridDim.x * 256, at = (int64_t)blockIdx.x * 256 + tid;
    for (int64_t i = at; i < (int64_t)pr.B * pr.maxp; i += step) {
        const int b = (int)(i / pr.maxp), p = pr.pages[b * pr.pages_row + (i - (int64_t)b * pr.maxp)];
        pr.out_pages[i] = is_page(p, pr.npages) && p >= used && pr.counts[p] > 0 ? pr.holes[pr.rank[p]] : p;
    }
    for (int64_t i = at; i < pr.npages; i += step)
        if (i >= used) pr.out_counts[i] = pr.counts[i] > 0 ? 0 : pr.counts[i];
        else if (pr.counts[i] > 0) pr.out_counts[i] = pr.counts[i];
    for (int64_t i = at; i < moved; i += step) pr.out_counts[pr.holes[i]] = pr.counts[pr.movers[i]];
    for (int64_t i = blockIdx.x; i < (int64_t)moved * 2; i += gridDim.x)
        copy_page(pr.shape, i & 1, pr.movers[i >> 1], pr.holes[i >> 1], 1 << pr.page_log2, tid, 256);
}

unsigned blocks_for(int64_t items) {
    const int64_t n = (items + 255) / 256;
    return (unsigned)(n < 1 ? 1 : n < 2048 ? n : 2048);
}

}  // namespace

hipError_t launch_fork(const ForkProblem &pr, hipStream_t s) {
    const int64_t items = (int64_t)pr.N * pr.maxp;
    fork_rows<<<blocks_for(items > pr.npages ? items : pr.npages), 256, 0, s>>>(pr);
    fork_counts<<<(unsigned)pr.B, 256, 0, s>>>(pr);
    return hipGetLastError();
}

// ranks, needs (B each) and the list of free pages
int64_t resize_workspace_ints(int64_t B, int64_t npages) { return 2 * B + npages; }
hipError_t launch_resize(ResizeProblem pr, int32_t *work, hipStream_t s) {
    pr.ranks = work;
    pr.needs = work + pr.B;
    pr.free_list = work + 2 * (int64_t)pr.B;
    resize_plan<<<1, kPlan, 0, s>>>(pr);
    resize_apply<<<dim3((unsigned)pr.B, 2), 256, 0, s>>>(pr);
    return hipGetLastError();
}

// sizes (4), holes and movers (half the pages each at most) and ranks of movers
int64_t compact_workspace_ints(int64_t npages) { return 4 + 3 * npages; }
hipError_t launch_compact(CompactProblem pr, int32_t *work, hipStream_t s) {
    pr.sizes = work;
    pr.holes = work + 4;
    pr.movers = pr.holes + pr.npages;
    pr.rank = pr.movers + pr.npages;
    compact_plan<<<1, kPlan, 0, s>>>(pr);
    const int64_t items = (int64_t)pr.B * pr.maxp, pages = 256 * (int64_t)pr.npages;
    compact_apply<<<blocks_for(items > pages ? items : pages), 256, 0, s>>>(pr);
    return hipGetLastError();
}

}  // namespace circatt
