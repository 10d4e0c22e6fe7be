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
    void *y_rest;            // what y's rounding took, laid out as y, or NULL
    // log2 of a row's sum of exp2(scale log2(e) q.k), +inf for a row behind the
    // signal's length: (B, Hk, L*G), row i*G + g
    float *lse;
    // backward
    const void *dy;
    int64_t dy_row, dy_batch;
    void *dq, *dk, *dv;  // contiguous; dk and dv may be NULL (both)
    float *work;         // rowsum(dy * y), laid out as lse, then partial sums
};
int64_t sliding_bwd_workspace_floats(const SlidingProblem &pr);
// Threads of the largest launch of the forward, or of the backward: a launch holds
// less than 2^32 along an axis.
int64_t sliding_threads(const SlidingProblem &pr, bool backward);
hipError_t launch_sliding_fwd(const SlidingProblem &pr, hipStream_t s);
hipError_t launch_sliding_bwd(const SlidingProblem &pr, hipStream_t s);

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
int64_t paged_workspace_floats(const PagedProblem &pr);
int64_t paged_threads(const PagedProblem &pr);  // along the longest axis
hipError_t launch_paged(const PagedProblem &pr, hipStream_t s);

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
