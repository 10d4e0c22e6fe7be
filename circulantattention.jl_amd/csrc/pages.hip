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
// the chain from load to load.  A call is two launches, a plan by one workgroup, whose
// barriers stand between its steps, and the work of it by many; or one, where the plan's
// workgroup does a small call's work as well (kSmall; a launch is some 3 us to the host
// and 3 to the GPU).  Kernels, us: fork to 128 of 64 sequences of 4096 2.8 + 2.7, resize of
// those by a token 6.4 + 5.0; of 256 sequences of up to 2048, most by 512, 17.8 + 4.0; with
// the plan's counts in memory instead of LDS that call took 31.5 in all, now 20.3.
// Compaction of 64 sequences of up to 2048 tokens, 1024 channels, half of them gone, 7.3 +
// 28.8, 5.9 TB/s of the move.
#include "token_kernels.h"

namespace circatt {
namespace {

typedef int i4 __attribute__((ext_vector_type(4)));
typedef uint32_t u4 __attribute__((ext_vector_type(4)));

__device__ __forceinline__ int uniform(int x) { return __builtin_amdgcn_readfirstlane(x); }
__device__ __forceinline__ bool is_page(int p, int npages) { return (unsigned)p < (unsigned)npages; }
// Pages that n tokens reach, of a table of maxp.
__device__ __forceinline__ int reach(int n, int page_log2, int maxp) {
    const int p = n <= 0 ? 0 : (int)(((int64_t)n + (1 << page_log2) - 1) >> page_log2);
    return p < maxp ? p : maxp;
}

constexpr int kPlan = 1024;   // threads of a plan
constexpr int kSmall = 8192;  // numbers in tables and counts that one workgroup sees to

// ---------------------------------------------------------------------------
// Fork.  First the new rows and the old counts, then the pages of every old sequence get
// as many holders more as have taken it, less itself.
__device__ __forceinline__ void fork_rows_of(const ForkProblem &pr, int64_t at, int64_t step) {
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
}
__global__ __launch_bounds__(256) void fork_rows(ForkProblem pr) {
    const int64_t at = (int64_t)blockIdx.x * 256 + threadIdx.x, step = (int64_t)gridDim.x * 256;
    fork_rows_of(pr, at, step);
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
// A small one by one workgroup, its counts in LDS.
__global__ __launch_bounds__(kPlan) void fork_small(ForkProblem pr) {
    __shared__ int takers[kSmall], counts[kSmall];
    const int tid = threadIdx.x;
    for (int b = tid; b < pr.B; b += kPlan) takers[b] = -1;
    for (int p = tid; p < pr.npages; p += kPlan) counts[p] = pr.counts[p];
    __syncthreads();
    for (int n = tid; n < pr.N; n += kPlan) {
        const int b = pr.source[n];
        if ((unsigned)b < (unsigned)pr.B) atomicAdd(takers + b, 1);
    }
    fork_rows_of(pr, tid, kPlan);
    __syncthreads();
    for (int i = tid; i < pr.B * pr.maxp; i += kPlan) {
        const int b = i / pr.maxp, e = i - b * pr.maxp, p = pr.pages[b * pr.pages_row + e];
        if (takers[b] != 0 && e < reach(pr.lengths[b], pr.page_log2, pr.maxp) && is_page(p, pr.npages))
            atomicAdd(counts + p, takers[b]);
    }
    __syncthreads();
    for (int p = tid; p < pr.npages; p += kPlan) pr.out_counts[p] = counts[p];
}

// ---------------------------------------------------------------------------
// One workgroup's sums over its threads in order: the sum before this thread's x, and
// that of all.
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

__device__ __forceinline__ void store_counts(int32_t *counts, int64_t i0, int npages, const int (&c)[kEach]) {
    if (i0 + kEach <= npages && reinterpret_cast<uintptr_t>(counts) % 16 == 0) {
#pragma unroll
        for (int k = 0; k < kEach; k += 4) *reinterpret_cast<i4 *>(counts + i0 + k) = i4{c[k], c[k + 1], c[k + 2], c[k + 3]};
    } else {
#pragma unroll
        for (int k = 0; k < kEach; ++k)
            if (i0 + k < npages) counts[i0 + k] = c[k];
    }
}

// A sequence's change of size.
struct Change {
    int from, to, has, wants, last;  // tokens, pages; the page that its last token is in
    Change() = default;
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

// Rows [0, rows) of page `from` to page `to` of one cache, by `threads` threads.
template <typename U>
__device__ __forceinline__ void copy_rows(char *cache, const PageShape &sh, int from, int to, int rows, int tid, int threads) {
    const int units = (int)(sh.C * sh.esize / (int)sizeof(U));
    const char *s = cache + (int64_t)from * sh.page_stride * sh.esize;
    char *d = cache + (int64_t)to * sh.page_stride * sh.esize;
    const int64_t row = sh.row_stride * sh.esize;
#pragma unroll 4
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

// Resize, work: a sequence's new row.  Its pages are list[rank ..] in order, first that
// of the copy (need below zero); rank -1: it stays as it is.
__device__ __forceinline__ void resize_row(const ResizeProblem &pr, int b, const Change &c, int rank, int need, const int *list,
                                           int tid, int threads) {
    const bool copy = need < 0 && rank >= 0, stays = need != 0 && rank < 0;
    const int wants = stays ? c.has : c.wants;
    const int32_t *row = pr.pages + b * pr.pages_row;
    for (int e = tid; e < pr.maxp; e += threads) {
        int p = -1;
        if (e < wants) {
            const bool own = e >= c.has || (copy && e == c.has - 1);
            p = own ? list[rank + (copy ? 1 : 0) + e - c.has] : row[e];
        }
        pr.out_pages[(int64_t)b * pr.maxp + e] = p;
    }
    if (tid == 0) pr.out_lengths[b] = stays ? c.from : c.to;
}
// The tokens of its part page, if that is copied.
__device__ __forceinline__ void resize_copy(const ResizeProblem &pr, bool v, const Change &c, int rank, int need, const int *list,
                                            int tid, int threads) {
    if (need >= 0 || rank < 0) return;
    copy_page(pr.shape, v, c.last, list[rank], c.from & ((1 << pr.page_log2) - 1), tid, threads);
}
__global__ __launch_bounds__(256) void resize_apply(ResizeProblem pr) {
    const int b = blockIdx.x, rank = pr.ranks[b], need = pr.needs[b];
    const Change c(pr, b);
    if (blockIdx.y == 0) resize_row(pr, b, c, rank, need, pr.free_list, threadIdx.x, 256);
    resize_copy(pr, blockIdx.y != 0, c, rank, need, pr.free_list, threadIdx.x, 256);
}

// What the sequences b0 + tid give back, entry by entry, by the whole workgroup.
struct Returns {
    int before[kPlan], first[kPlan];
};
__device__ __forceinline__ void give_back(const ResizeProblem &pr, int b0, const Change &c, Returns &r, int *waves, int *counts) {
    const int tid = threadIdx.x;
    const int gives = b0 + tid < pr.B && c.wants < c.has ? c.has - c.wants : 0;
    const BlockSum s = block_sum(gives, waves);
    if (s.all == 0) return;
    r.first[tid] = c.wants;
    r.before[tid] = s.before;
    __syncthreads();
    constexpr int AT_ONCE = 4;  // loads on their way
    for (int i0 = tid; i0 < s.all; i0 += AT_ONCE * kPlan) {
        int p[AT_ONCE];
#pragma unroll
        for (int k = 0; k < AT_ONCE; ++k) {
            const int i = i0 + k * kPlan < s.all ? i0 + k * kPlan : i0;
            int lo = 0;  // the last sequence that begins at i or before it
#pragma unroll
            for (int step = kPlan / 2; step; step >>= 1) lo += r.before[lo + step] <= i ? step : 0;
            p[k] = pr.pages[(b0 + lo) * pr.pages_row + r.first[lo] + i - r.before[lo]];
        }
#pragma unroll
        for (int k = 0; k < AT_ONCE; ++k)
            if (i0 + k * kPlan < s.all && is_page(p[k], pr.npages)) atomicAdd(counts + p[k], -1);
    }
    __syncthreads();
}
__device__ __forceinline__ bool copies(const ResizeProblem &pr, const Change &c) {
    return c.to > c.from && (c.from & ((1 << pr.page_log2) - 1)) != 0 && is_page(c.last, pr.npages);
}

// Resize, plan, of up to kPlan sequences and a cache of up to kHeld pages: its counts
// in LDS, where nothing waits for memory between the steps.  The counts less the pages
// given back; what every sequence needs and where its pages begin in the list of free
// ones (ranks: -1 for a sequence that stays as it is; needs: below zero with a part page
// to copy); that list; the counts of the pages that are given.
// SMALL: and the work, by the same workgroup.
constexpr int kHeld = 32768;
template <bool SMALL>
__global__ __launch_bounds__(kPlan) void resize_held(ResizeProblem pr) {
    constexpr int WAVES = kPlan / 64;
    __shared__ int waves[WAVES], counts[SMALL ? kSmall : kHeld], own_list[SMALL ? kSmall : 1];
    __shared__ Returns returns;
    __shared__ int ranks[kPlan], needs[kPlan];
    __shared__ int given;
    const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
    int *list = SMALL ? own_list : pr.free_list;
#pragma unroll 8
    for (int p = tid; p < pr.npages; p += kPlan) counts[p] = pr.counts[p];
    Change c{};
    if (tid < pr.B) c = Change(pr, tid);
    if (tid == 0) given = 0;
    __syncthreads();
    give_back(pr, 0, c, returns, waves, counts);
    const bool copy = tid < pr.B && copies(pr, c) && counts[c.last] > 1;
    const int need = tid < pr.B ? copy + (c.wants > c.has ? c.wants - c.has : 0) : 0;
    const int rank = block_sum(need, waves).before;
    // each wavefront has a run of pages: how many are free, then their places
    const int run = (pr.npages + kPlan - 1) / kPlan * 64, p0 = wave * run, p1 = p0 + run < pr.npages ? p0 + run : pr.npages;
    int free = 0;
#pragma unroll 8
    for (int p = p0 + lane; p < p1; p += 64) free += counts[p] == 0;
    const BlockSum s = block_sum(free, waves);
    int at = uniform(s.before);
#pragma unroll 4
    for (int p = p0; p < p1; p += 64) {
        const bool is = p + lane < p1 && counts[p + lane] == 0;
        const uint64_t those = __ballot(is);
        if (is) list[at + __popcll(those & ((1ull << lane) - 1))] = p + lane;
        at += __popcll(those);
    }
    const bool served = need == 0 || rank + need <= s.all;
    if (tid < pr.B) {
        ranks[tid] = served ? rank : -1;
        needs[tid] = copy ? -need : need;
        if (!SMALL) {
            pr.ranks[tid] = ranks[tid];
            pr.needs[tid] = needs[tid];
        }
        if (need > 0 && served) atomicMax(&given, rank + need);
    }
    __syncthreads();
    // the list's first `given` pages are held once now
    at = uniform(s.before);
    for (int p = p0; p < p1 && at < given; p += 64) {
        const bool is = p + lane < p1 && counts[p + lane] == 0;
        const uint64_t those = __ballot(is);
        if (is && at + __popcll(those & ((1ull << lane) - 1)) < given) counts[p + lane] = 1;
        at += __popcll(those);
    }
    __syncthreads();
    if (copy && served) atomicAdd(counts + c.last, -1);
    __syncthreads();
    for (int p = tid; p < pr.npages; p += kPlan) pr.out_counts[p] = counts[p];
    if constexpr (SMALL) {
        for (int b = wave; b < pr.B; b += WAVES)
            resize_row(pr, b, Change(pr, b), ranks[b], needs[b], own_list, lane, 64);
        for (int i = wave; i < 2 * pr.B; i += WAVES)
            resize_copy(pr, i & 1, Change(pr, i >> 1), ranks[i >> 1], needs[i >> 1], own_list, lane, 64);
    }
}

// The same for any number of sequences and pages, with the counts in memory.
__global__ __launch_bounds__(kPlan) void resize_plan(ResizeProblem pr) {
    __shared__ int waves[kPlan / 64];
    __shared__ Returns returns;
    __shared__ int given;
    const int tid = threadIdx.x;
    for (int64_t p0 = 0; p0 < pr.npages; p0 += (int64_t)kPlan * kEach) {
        int c[kEach];
        const int64_t i0 = p0 + (int64_t)tid * kEach;
        load_counts(pr.counts, i0, pr.npages, c);
        store_counts(pr.out_counts, i0, pr.npages, c);
    }
    if (tid == 0) given = 0;
    __threadfence();
    __syncthreads();
    for (int b0 = 0; b0 < pr.B; b0 += kPlan) {
        Change c{};
        if (b0 + tid < pr.B) c = Change(pr, b0 + tid);
        give_back(pr, b0, c, returns, waves, pr.out_counts);
    }
    // the counts are read again from here on, past what this compute unit holds of them
    __threadfence();
    __syncthreads();
    int64_t asked = 0;
    for (int b0 = 0; b0 < pr.B; b0 += kPlan) {
        const int b = b0 + tid;
        int need = 0, copy = 0;
        if (b < pr.B) {
            const Change c(pr, b);
            copy = copies(pr, c) && pr.out_counts[c.last] > 1;
            need = copy + (c.wants > c.has ? c.wants - c.has : 0);
        }
        const BlockSum s = block_sum(need, waves);
        if (b < pr.B) {
            const int64_t at = asked + s.before;
            pr.ranks[b] = (int)(at < INT32_MAX / 2 ? at : INT32_MAX / 2);
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
        if (need == 0) continue;
        if ((int64_t)pr.ranks[b] + need > found) pr.ranks[b] = -1;
        else atomicMax(&given, pr.ranks[b] + need);
    }
    __threadfence();  // the list, read by others
    __syncthreads();
    for (int r = tid; r < given; r += kPlan) pr.out_counts[pr.free_list[r]] = 1;
    for (int b = tid; b < pr.B; b += kPlan)
        if (pr.needs[b] < 0 && pr.ranks[b] >= 0) atomicAdd(pr.out_counts + Change(pr, b).last, -1);
}

// ---------------------------------------------------------------------------
// Compact, work: the table's numbers and the counts follow, and pages move: those of
// numbers from `first` on, `every` apart (k's and v's in turn), by `threads` threads.
__device__ __forceinline__ void compact_tables(const CompactProblem &pr, const int *counts, const int *holes, const int *movers,
                                               const int *rank, int used, int moved, int64_t at, int64_t step) {
    for (int64_t i = at; i < (int64_t)pr.B * pr.maxp; i += step) {
        const int b = (int)(i / pr.maxp), p = pr.pages[b * pr.pages_row + (i - (int64_t)b * pr.maxp)];
        pr.out_pages[i] = is_page(p, pr.npages) && p >= used && counts[p] > 0 ? holes[rank[p]] : p;
    }
    for (int64_t i = at; i < pr.npages; i += step) {
        const int c = counts[i];
        if (i >= used) pr.out_counts[i] = c > 0 ? 0 : c;
        else if (c > 0) pr.out_counts[i] = c;
    }
    for (int64_t i = at; i < moved; i += step) pr.out_counts[holes[i]] = counts[movers[i]];
}
__device__ __forceinline__ void compact_pages(const CompactProblem &pr, const int *holes, const int *movers, int moved,
                                              int64_t first, int64_t every, int tid, int threads) {
    for (int64_t i = first; i < (int64_t)moved * 2; i += every)
        copy_page(pr.shape, i & 1, movers[i >> 1], holes[i >> 1], 1 << pr.page_log2, tid, threads);
}
__global__ __launch_bounds__(256) void compact_apply(CompactProblem pr) {
    const int used = pr.sizes[0], moved = pr.sizes[1];
    compact_tables(pr, pr.counts, pr.holes, pr.movers, pr.rank, used, moved,
                   (int64_t)blockIdx.x * 256 + threadIdx.x, (int64_t)gridDim.x * 256);
    compact_pages(pr, pr.holes, pr.movers, moved, blockIdx.x, gridDim.x, threadIdx.x, 256);
}

// Compact, plan: `used`, the number of pages held, the free numbers below it (holes) and
// the held ones from it on (movers, as many), both ascending, and each mover's rank.
__global__ __launch_bounds__(kPlan) void compact_plan(CompactProblem pr) {
    __shared__ int waves[kPlan / 64];
    const int tid = threadIdx.x;
    constexpr int kRound = kPlan * kEach;
    int c[kEach], used = 0;
    for (int64_t p0 = 0; p0 < pr.npages; p0 += kRound) {
        const int64_t i0 = p0 + (int64_t)tid * kEach;
        int n = 0;
        load_counts(pr.counts, i0, pr.npages, c);
#pragma unroll
        for (int k = 0; k < kEach; ++k) n += i0 + k < pr.npages && c[k] > 0;
        used += block_sum(n, waves).all;
    }
    int holes = 0, movers = 0;
    for (int64_t p0 = 0; p0 < pr.npages; p0 += kRound) {
        const int64_t i0 = p0 + (int64_t)tid * kEach;
        int n = 0;  // holes, and 2^16 times movers: a round has at most 2^14 of them
        if (pr.npages > kRound) load_counts(pr.counts, i0, pr.npages, c);
#pragma unroll
        for (int k = 0; k < kEach; ++k)
            if (i0 + k < pr.npages) n += i0 + k < used ? (c[k] <= 0 ? 1 : 0) : (c[k] > 0 ? 1 << 16 : 0);
        const BlockSum s = block_sum(n, waves);
        int hr = holes + (s.before & 0xffff), mr = movers + (s.before >> 16);
#pragma unroll
        for (int k = 0; k < kEach; ++k) {
            const int p = (int)(i0 + k);
            if (i0 + k >= pr.npages) continue;
            if (p < used && c[k] <= 0) pr.holes[hr++] = p;
            if (p >= used && c[k] > 0) {
                pr.movers[mr] = p;
                pr.rank[p] = mr++;
            }
        }
        holes += s.all & 0xffff;
        movers += s.all >> 16;
    }
    if (tid == 0) {
        pr.sizes[0] = used;
        pr.sizes[1] = movers;
    }
}
// A small one by one workgroup, counts and lists in LDS.
__global__ __launch_bounds__(kPlan) void compact_small(CompactProblem pr) {
    constexpr int EACH = kSmall / kPlan;
    __shared__ int waves[kPlan / 64];
    __shared__ int counts[kSmall], holes[kSmall], movers[kSmall], rank[kSmall];
    const int tid = threadIdx.x;
#pragma unroll
    for (int k = 0; k < EACH; ++k) {
        const int p = tid + k * kPlan;
        counts[p] = p < pr.npages ? pr.counts[p] : 0;
    }
    __syncthreads();
    int n = 0;
#pragma unroll
    for (int k = 0; k < EACH; ++k) n += counts[tid * EACH + k] > 0;
    const int used = block_sum(n, waves).all;
    n = 0;  // holes, and 2^16 times movers
#pragma unroll
    for (int k = 0; k < EACH; ++k) {
        const int p = tid * EACH + k;
        n += p < used ? (counts[p] <= 0 ? 1 : 0) : (counts[p] > 0 ? 1 << 16 : 0);
    }
    const BlockSum s = block_sum(n, waves);
    int hr = s.before & 0xffff, mr = s.before >> 16;
#pragma unroll
    for (int k = 0; k < EACH; ++k) {
        const int p = tid * EACH + k;
        if (p < used && counts[p] <= 0) holes[hr++] = p;
        if (p >= used && counts[p] > 0) {
            movers[mr] = p;
            rank[p] = mr++;
        }
    }
    __syncthreads();
    compact_tables(pr, counts, holes, movers, rank, used, s.all >> 16, tid, kPlan);
    compact_pages(pr, holes, movers, s.all >> 16, tid >> 6, kPlan / 64, tid & 63, 64);
}

// What one workgroup copies while the host brings the next call, where another launch would
// take the host longer.  Calls from Python one after another, us, 256 KiB copied by one
// workgroup and by a second launch: resize 16 and 18.6, compact 13.5 and 16; 512 KiB: 16 to 28 and
// 18.7, 17 to 22 and 16; 1 MiB: 27 to 51 and 18.7, 28 to 39 and 16.  (The kernels alone, as
// in a captured graph: 11 to 16 and 7, 11 to 14 and 10; 64 KiB 7 and 7, 7 to 10 and 9.)
constexpr int64_t kSmallBytes = 256 * 1024;
int64_t page_bytes(const PageShape &sh, int page_log2) { return (sh.C * sh.esize << page_log2) * 2; }

unsigned blocks_for(int64_t items) {
    const int64_t n = (items + 255) / 256;
    return (unsigned)(n < 1 ? 1 : n < 2048 ? n : 2048);
}

}  // namespace

hipError_t launch_fork(const ForkProblem &pr, hipStream_t s) {
    const int64_t items = (int64_t)pr.N * pr.maxp;
    if (items + (int64_t)pr.B * pr.maxp + pr.npages <= kSmall) {
        fork_small<<<1, kPlan, 0, s>>>(pr);
    } else {
        fork_rows<<<blocks_for(items > pr.npages ? items : pr.npages), 256, 0, s>>>(pr);
        fork_counts<<<(unsigned)pr.B, 256, 0, s>>>(pr);
    }
    return hipGetLastError();
}

// ranks, needs (B each) and the list of free pages
int64_t resize_workspace_ints(int64_t B, int64_t npages) { return 2 * B + npages; }
hipError_t launch_resize(ResizeProblem pr, int32_t *work, hipStream_t s) {
    pr.ranks = work;
    pr.needs = work + pr.B;
    pr.free_list = work + 2 * (int64_t)pr.B;
    const bool small = (int64_t)pr.B * pr.maxp + pr.npages <= kSmall && pr.B * page_bytes(pr.shape, pr.page_log2) <= kSmallBytes;
    if (small && pr.B <= kPlan) {
        resize_held<true><<<1, kPlan, 0, s>>>(pr);
        return hipGetLastError();
    }
    if (pr.B <= kPlan && pr.npages <= kHeld) resize_held<false><<<1, kPlan, 0, s>>>(pr);
    else resize_plan<<<1, kPlan, 0, s>>>(pr);
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
    const int64_t items = (int64_t)pr.B * pr.maxp, bytes = pr.npages * page_bytes(pr.shape, pr.page_log2);
    // half of the pages move at most, and a quarter where half of the sequences ended
    if (items + pr.npages <= kSmall && bytes <= 4 * kSmallBytes) {
        compact_small<<<1, kPlan, 0, s>>>(pr);
    } else {
        compact_plan<<<1, kPlan, 0, s>>>(pr);
        compact_apply<<<blocks_for(items > 256 * (int64_t)pr.npages ? items : 256 * (int64_t)pr.npages), 256, 0, s>>>(pr);
    }
    return hipGetLastError();
}

}  // namespace circatt
