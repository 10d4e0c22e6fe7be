// Problems and launchers of the token operators: causal sliding-window
// attention with sinks on (batch, length, channels) signals, the same over a
// paged cache, the cache's append, and rotary positions.
#pragma once

#include "circatt.h"
#include "circatt_common.h"

namespace circatt {

// Heads of keys and values serve G = H / Hk heads of queries each.  Strides are
// in elements; channels of one token are contiguous (head g at g * D).
// Row i of signal b (i < lengths[b]) sees key j <= i with j > i - W or j < S.
struct SlidingProblem {
    int dtype;
    int B, L, H, Hk, G, D, W, S;
    float scale;
    const void *q, *k, *v;
    int64_t q_row, q_batch, k_row, k_batch, v_row, v_batch;
    const int32_t *lengths;  // (B) or NULL: all L
    void *y;                 // (B, L, H*D)
    void *y_rest;            // what y lacks for its rounding, laid out as y, or NULL
    // log2 of a row's sum of exp2(scale log2(e) q.k), +inf for a row behind the
    // signal's length: (B, Hk, L*G), row i*G + g
    float *lse;
    // backward
    const void *dy;
    int64_t dy_row, dy_batch;
    void *dq, *dk, *dv;  // contiguous; dk and dv may be NULL (both)
    float *work;         // rowsum(dy * y), laid out as lse, then partial sums
};
// How capped scores follow from products d: C tanh(x d), in powers of two
// (token_shape.h).
struct Curve {
    float x, u, C;  // scale / cap, 2 log2(e) x, log2(e) cap
    // up to these |d| the tangent is d (few[0] + few[1] d^2 + ...) or d (more[0] + ...);
    // below 0: never
    float near, far;
    float few[3], more[5];
    int fine;       // whether an error of 2^-22 of the cap would be seen in the result
};
Curve make_curve(float cap, float scale, int dtype);

// How scores follow from products, and what else a row sees (or does not).
struct ScoreShape {
    float cap;               // 0: none
    Curve curve;
    const float *slopes;     // (H) or NULL
    const int32_t *prefix;   // (B) or NULL: tokens that all rows see
    const int32_t *places;   // each token's place in its document, or NULL
    int64_t places_row;      // from signal to signal
};
struct ShapedSlidingProblem : SlidingProblem {
    ScoreShape shape;
    // of the backward, in its workspace: slope times log2(e), and token, of every
    // packed row of a head of keys ((Hk, L*G) and (L*G); with slopes), and the end of
    // every token's document ((B, L); with places)
    float *row_slopes, *row_tokens;
    int32_t *ends;
};
int64_t sliding_bwd_workspace_floats(const SlidingProblem &pr);
// Threads of the largest launch of the forward, or of the backward: a launch holds
// less than 2^32 along an axis.
int64_t sliding_threads(const SlidingProblem &pr, bool backward);
hipError_t launch_sliding_fwd(const SlidingProblem &pr, hipStream_t s);
hipError_t launch_sliding_bwd(const SlidingProblem &pr, hipStream_t s);
// The same with shaped scores.  biased: whether slopes are there; masked: what else rows
// see (the workspace is asked for without the arrays).
enum Masked { kUnmasked, kPlaces, kPrefix };
inline int masked_by(const ScoreShape &sh) {
    return sh.places != nullptr ? kPlaces : sh.prefix != nullptr ? kPrefix : kUnmasked;
}
int64_t shaped_bwd_workspace_floats(const SlidingProblem &pr, bool biased, int masked);
int64_t shaped_sliding_threads(const SlidingProblem &pr, int masked, bool backward);
hipError_t launch_shaped_fwd(const ShapedSlidingProblem &pr, hipStream_t s);
hipError_t launch_shaped_bwd(ShapedSlidingProblem pr, hipStream_t s);

// The T rows of q are the new tokens of B sequences in order: sequence b has
// rows offsets[b] .. offsets[b+1] (offsets NULL: row b alone), the last tokens
// of the lengths[b] that its pages hold.
struct PagedProblem {
    int dtype;
    int64_t T;
    int B, H, Hk, G, D, W, S;
    float scale;
    const void *q;
    int64_t q_row;
    const void *k, *v;
    int64_t page_stride, row_stride;  // of the caches, in elements
    int npages, page, page_log2;      // page = 1 << page_log2 tokens
    const int32_t *pages;             // (B, maxp)
    int64_t pages_row;
    int maxp;
    const int32_t *lengths, *offsets;
    void *y;        // (T, H*D)
    int zero_tail;  // rows behind the last sequence: 1 zeros, 0 left alone
    float *work;
};
struct ShapedPagedProblem : PagedProblem {
    ScoreShape shape;  // without places
};
// whole: of a plan for rows that may see all that the table holds, behind a prefix
int64_t paged_workspace_floats(const PagedProblem &pr, bool whole = false);
int64_t paged_threads(const PagedProblem &pr);  // along the longest axis
hipError_t launch_paged(const PagedProblem &pr, hipStream_t s);
hipError_t launch_shaped_paged(const ShapedPagedProblem &pr, bool whole, hipStream_t s);

struct AppendProblem {
    int esize;  // bytes of an element
    int64_t T;
    int B;
    int64_t C;  // channels of a token
    const void *k, *v;
    int64_t k_row, v_row;
    void *cache_k, *cache_v;
    int64_t page_stride, row_stride;
    int npages, page_log2;
    const int32_t *pages;
    int64_t pages_row;
    int maxp;
    const int32_t *lengths, *offsets;
};
int64_t append_threads(const AppendProblem &pr);
hipError_t launch_append(const AppendProblem &pr, hipStream_t s);

// Sequences of a cache and the pages that they hold: row b of pages (pages_row apart)
// has a page for every 1 << page_log2 of sequence b's tokens, counts the holders of
// every page.
struct PageTable {
    int B, maxp, npages, page_log2;
    const int32_t *pages;
    int64_t pages_row;
    const int32_t *lengths, *counts;
    int32_t *out_pages, *out_lengths, *out_counts;  // rows of maxp
};
struct ForkProblem : PageTable {
    int N;  // sequences after the fork
    const int32_t *source;
};
hipError_t launch_fork(const ForkProblem &pr, hipStream_t s);

struct PageShape {
    int esize;
    int64_t C;  // channels of a token
    void *cache_k, *cache_v;
    int64_t page_stride, row_stride;
};
struct ResizeProblem : PageTable {
    PageShape shape;
    const int32_t *to;
    int32_t *ranks, *needs, *free_list;
};
int64_t resize_workspace_ints(int64_t B, int64_t npages);
hipError_t launch_resize(ResizeProblem pr, int32_t *work, hipStream_t s);

struct CompactProblem : PageTable {
    PageShape shape;
    int32_t *sizes, *holes, *movers, *rank;
};
int64_t compact_workspace_ints(int64_t npages);
hipError_t launch_compact(CompactProblem pr, int32_t *work, hipStream_t s);

constexpr int kMaxPairs = 128;
struct RotaryProblem {
    int dtype, inverse, interleaved, naxes;
    int n1, n2;        // the grid's two fastest sizes (positions NULL)
    int64_t P, nb;     // tokens of an image, images
    int H, D;
    int pairs[3], npairs;
    const void *x;
    int64_t x_row;     // elements from token to token
    const int32_t *positions;  // (P, naxes) for every image at pos_batch, or NULL
    int64_t pos_batch;
    void *y;
    double turns[kMaxPairs];   // turns for one step of a pair's axis
};
int64_t rotary_threads(const RotaryProblem &pr);
hipError_t launch_rotary(const RotaryProblem &pr, hipStream_t s);

}  // namespace circatt
