/*
 * circatt.h -- C ABI of libcircatt, the MI355X (gfx950) circulant attention
 * library.  Drop-in compute layer for CirculantAttention.jl's hot path: the
 * reference reaches these operations through @cuda kernels, NNlib and
 * CUSPARSE.bmm!; a host binding (Julia ccall, Python ctypes) calls these
 * entry points instead.  Citations are file:line in the reference repository.
 *
 * Conventions
 *  - All array pointers are device pointers owned by the caller.  Nothing in
 *    an entry point allocates device memory; the fused backward takes a
 *    caller-provided workspace (size from circatt_fused_bwd_workspace_bytes).
 *  - Arrays use the reference's Julia column-major layout.  A signal of Julia
 *    size (N1[,N2], C, nb) holds (pixel r, channel c, batch b) at
 *    r + P*(c + C*b), P = N1*N2, r = i1 + N1*i2.  dtype CIRCATT_C32 signals
 *    are ComplexF32, interleaved (re, im).
 *  - A Circulant of size (P, P, nb) is CSR with K = ws^nsp slots per row:
 *    rowPtr (P+1, nb) and colVal (P*K, nb) Int32 1-based, nzVal (P*K, nb)
 *    Float32 (src/circulant.jl:64-106, src/array.jl:1-18).  Entry points that
 *    take nzVal use the circulant pattern implied by (nsp, n1, n2, ws).
 *  - nsp is 1 or 2; for nsp == 1, n2 is ignored.  ws must be odd
 *    (src/circulant.jl:65,87).
 *  - stream is a hipStream_t (NULL = default stream).  Launches are
 *    asynchronous; arguments are validated on the host before any launch.
 *  - Return value: CIRCATT_OK or a negative error code; circatt_last_error()
 *    returns a message for the calling thread's last failure.
 */
#ifndef CIRCATT_H
#define CIRCATT_H

#include <stdint.h>

#ifdef __cplusplus
extern "C" {
#endif

#define CIRCATT_OK 0
#define CIRCATT_ERR_INVALID (-1)     /* bad argument (the reference's @assert) */
#define CIRCATT_ERR_UNSUPPORTED (-2) /* valid but not implemented here */
#define CIRCATT_ERR_HIP (-3)         /* HIP runtime error */

/* Similarity kinds: DotSimilarity / DistanceSimilarity (src/similarity.jl:1-29). */
#define CIRCATT_DOT 0
#define CIRCATT_DISTANCE 1

/* Element types of signals: Float32, ComplexF32. */
#define CIRCATT_F32 0
#define CIRCATT_C32 1
/* Element types of the token operators only (they take CIRCATT_F32 as well). */
#define CIRCATT_F16 2
#define CIRCATT_BF16 3

/*
 * Layout flag, OR-ed into dtype of the fused entry points (circatt_fused_*):
 * q, k, v, y, dy and the gradients are channels-last, Julia size
 * (C, N1[,N2], B): (channel c, pixel r, batch b) at c + C*(r + P*b)
 * (ComplexF32: interleaved (re, im) elements in that order).  The kernels
 * read and write this layout directly, so a model that keeps its features
 * channels-last (the layout convolutions favour) needs no transposes around
 * the attention.  lse and the workspace keep their layout.  No counterpart in
 * the reference (which is planar only); other entry points reject the flag.
 */
#define CIRCATT_CHANNELS_LAST 16

/* Library version (major*10000 + minor*100 + patch). */
int circatt_version(void);

/*
 * Arithmetic of the fused kernels' matrix products.  The reference computes
 * in Float32 throughout; it has no counterpart of this switch.
 *   CIRCATT_MATH_SPLIT_F16 (default): each Float32 operand is split into
 *     16-bit parts and a product is taken as a sum of partial products on the
 *     16-bit matrix cores with Float32 accumulation.
 *     Heads of 16 or 32 real components at the windows that are compiled in
 *     (2D: 3, 5, 7, 11, and 15 at 16 components; 1D: 15 and 63): two f16 halves,
 *     hi*hi + lo*hi + hi*lo (relative error near 2^-21 per operand).  Operands
 *     are scaled by powers of two per work item (a 16x16 tile of one head, 8x16
 *     for heads of 32 real components, runs of 256 or 128 pixels of a line)
 *     before the split, so inputs of any magnitude (1e-7 and 1e4 are tested)
 *     give Float32-class results.  The scale follows the tile's largest value: a
 *     component far smaller than the others of its tile keeps an absolute error
 *     of some 2^-27 (at most 2^-23) of that value (four digits at a ratio of 1e-4, none at 1e-8).
 *     Where q.k scores are so large that the halves could overflow, a slower
 *     exact-scale walk takes over.
 *     Other heads of up to 64 real components: three bf16 thirds, which carry a
 *     Float32 value exactly at every magnitude, and the six partial products
 *     down to 2^-16 of a product (error 2^-26 of it as a rule): no scale, and
 *     every component keeps its own precision.
 *     Calls that neither form takes: Float32 matrix products.
 *   CIRCATT_MATH_F32: Float32 matrix products.
 * Like any attention backward that recomputes the probabilities from the
 * stored log-sum-exp, the fused backward loses precision once scores reach
 * ~1e3 (Float32 rounding of the score itself); the reference's own Float32
 * computation misses the gradient tolerance there as well.
 * Process-wide; takes effect for launches after the call.
 */
#define CIRCATT_MATH_SPLIT_F16 0
#define CIRCATT_MATH_F32 1
int circatt_set_math(int mode);
int circatt_get_math(void);

/* Message describing the calling thread's last error ("" if none). */
const char *circatt_last_error(void);

/*
 * Circulant sparsity pattern, replicated over nb batches.
 * Replaces cucirculant(M,N) / cucirculant(M,N1,N2) + its kernel
 * (src/circulant.jl:46-106) and the batch repeat in Circulant{T}(M, dims)
 * (src/array.jl:6-11).  rowptr: (P+1, nb), colval: (P*K, nb), Int32 1-based,
 * bit-identical to the reference, also for ws > N.
 */
int circatt_pattern(int nsp, int64_t n1, int64_t n2, int32_t ws, int64_t nb, int32_t *rowptr,
                    int32_t *colval, void *stream);

/*
 * nzval[:, b] = scale * similarity(x[..., b], y[..., b]) on the pattern.
 * Replaces circulant_similarity! and its Dot / Distance kernels
 * (src/similarity.jl:31-103, :138-142).  x is the row (query) argument, y the
 * column (key) argument; Dot: Re(sum_c x*conj(y)), Distance:
 * -sum_c |x-y|^2 / 2.  x, y: (P, C, nb) of dtype; nzval: (P*K, nb) Float32.
 * circulant_attention (src/attention.jl:19-23) uses scale = 1/sqrt(C).
 */
int circatt_similarity(int kind, int dtype, int nsp, int64_t n1, int64_t n2, int32_t ws,
                       int64_t C, int64_t nb, float scale, const void *x, const void *y,
                       float *nzval, void *stream);

/*
 * Row softmax over the K slots of each of `rows` rows (rows = P*nb); in == out
 * allowed.  Replaces circulant_softmax! / NNlib.softmax(::Circulant)
 * (src/similarity.jl:105-126).
 */
int circatt_softmax(int64_t K, int64_t rows, const float *in, float *out, void *stream);

/*
 * dS = A .* (dA .- sum(A .* dA, dims=slots)).  Replaces the softmax pullback
 * (src/rrules.jl:42-56, NNlib.∇softmax_data).  dS may alias dA.
 */
int circatt_softmax_bwd(int64_t K, int64_t rows, const float *A, const float *dA, float *dS,
                        void *stream);

/*
 * y = A ⊗ x (trans = 0) or y = Aᵀ ⊗ x (trans = 1) with A = nzval on the
 * pattern; x, y: (P, C, nb) of dtype (real A times complex x is the promotion
 * of src/batchedmul.jl:72-75).  Replaces circulant_attention!(y, A, x) /
 * circulant_transposed_attention! (src/attention.jl:53-80) and their
 * CUSPARSE.bmm! calls (src/batchedmul.jl:82-110).  Multi-head ⨷
 * (src/attention.jl:89-103) is the same call with C = channels/nheads and
 * nb = nheads*B.
 */
int circatt_apply(int trans, int dtype, int nsp, int64_t n1, int64_t n2, int32_t ws, int64_t C,
                  int64_t nb, const float *nzval, const void *x, void *y, void *stream);

/*
 * Pullback of nzval = scale * similarity(x, y):
 *   Dot:      dx = scale * dS ⊠ y,            dy = scale * dSᵀ ⊠ x
 *   Distance: dx = scale * (dS ⊠ y - rowsum(dS) .* x),
 *             dy = scale * (dSᵀ ⊠ x - colsum(dS) .* y)
 * Replaces the similarity rrules (src/rrules.jl:1-32) including their
 * sum(ΔS; dims=1/2) (src/array.jl:119-130).  dx or dy may be NULL.
 */
int circatt_similarity_bwd(int kind, int dtype, int nsp, int64_t n1, int64_t n2, int32_t ws,
                           int64_t C, int64_t nb, float scale, const float *dS, const void *x,
                           const void *y, void *dx, void *dy, void *stream);

/*
 * sum(A; dims=2) (out: (P, nb)) and sum(A; dims=1) (out: (P, nb)) of a
 * Circulant's nzval (src/array.jl:119-130, :156-177).
 */
int circatt_rowsum(int nsp, int64_t n1, int64_t n2, int32_t ws, int64_t nb, const float *nzval,
                   float *out, void *stream);
int circatt_colsum(int nsp, int64_t n1, int64_t n2, int32_t ws, int64_t nb, const float *nzval,
                   float *out, void *stream);

/*
 * Z[:, b] = alpha_b * X[:, b] + beta_b * Y[:, b] over nzval slices of nnz
 * entries, alpha_b = alpha ? alpha[b] : alpha0 (same for beta; Y may be NULL).
 * Covers X + Y, X - Y, c*X, -X (src/array.jl:66-81) and scale(c, A) with c of
 * size (1,1,nh,B) (src/array.jl:179-189); Z may alias X or Y.
 */
int circatt_axpby(int64_t nnz, int64_t nb, const float *alpha, float alpha0, const float *X,
                  const float *beta, float beta0, const float *Y, float *Z, void *stream);

/*
 * out[b] = sum_i X[i, b] * Y[i, b] over nnz entries per batch (Y == NULL:
 * sum_i X[i, b]); accumulated in double in a fixed order, so results are
 * reproducible.  Covers dot(X, Y) (src/array.jl:83-85, nb = 1 over all
 * batches), sum(A) and sum(A; dims=(1,2)) (src/array.jl:132-177) and the ∂c
 * of the scale rrule (src/rrules.jl:101-104).  workspace: at least
 * circatt_batch_dot_workspace_bytes(nnz, nb) bytes of device memory.
 */
int64_t circatt_batch_dot_workspace_bytes(int64_t nnz, int64_t nb);
int circatt_batch_dot(int64_t nnz, int64_t nb, const float *X, const float *Y, float *out,
                      void *workspace, int64_t workspace_bytes, void *stream);

/*
 * Fused forward of circulant (multi-head) attention without materialising A:
 * for head g of batch b (channels g*dh .. g*dh+dh-1, dh = C/nheads),
 *   y = softmax_rows(scale * sim(q, k)) ⊗ v,   scale = 1/sqrt(dh),
 * and lse[r, g + nheads*b] = log(sum_c exp(scale * sim(q_r, k_c))).
 * Equals circulant_attention (src/attention.jl:19-26, nheads = 1) and
 * circulant_mh_attention (src/attention.jl:38-42) for the returned y.
 * q, k, v, y: (P, C, B) of dtype; lse: (P, nheads*B) Float32.
 * Any number of channels per head (the reference's similarity loops over
 * any C, src/similarity.jl:97-99): heads of up to 64 real components run on
 * kernels that hold a pixel's components at once, wider heads on kernels
 * that sum the score products over 32-component chunks and form the outputs
 * in 64-component passes.  Windows whose 2D block columns exceed the LDS
 * budget (ws beyond 63) return CIRCATT_ERR_UNSUPPORTED.
 */
int circatt_fused_fwd(int kind, int dtype, int nsp, int64_t n1, int64_t n2, int32_t ws,
                      int64_t C, int64_t nheads, int64_t B, const void *q, const void *k,
                      const void *v, void *y, float *lse, void *stream);

/* Bytes of workspace circatt_fused_bwd needs (per-row D = <dy, y>). */
int64_t circatt_fused_bwd_workspace_bytes(int nsp, int64_t n1, int64_t n2, int64_t nheads,
                                          int64_t B);

/*
 * Fused backward matching the composition of the rrules of similarity,
 * softmax and ⊗ (src/rrules.jl:1-72) and the q, k scaling of
 * src/attention.jl:21: given dy, returns dq, dk, dv.  lse from
 * circatt_fused_fwd.  No atomics: a query-centric pass writes dq, a
 * key-centric pass writes dk and dv.
 */
int circatt_fused_bwd(int kind, int dtype, int nsp, int64_t n1, int64_t n2, int32_t ws,
                      int64_t C, int64_t nheads, int64_t B, const void *q, const void *k,
                      const void *v, const void *y, const void *dy, const float *lse, void *dq,
                      void *dk, void *dv, void *workspace, int64_t workspace_bytes,
                      void *stream);

/*
 * The two passes of circatt_fused_bwd, for callers that time or schedule them
 * separately.  circatt_fused_bwd_dq writes dq and the per-row D = <dy, y>
 * into workspace; circatt_fused_bwd_dkdv reads that D and writes dk, dv, so
 * it must follow circatt_fused_bwd_dq on the same stream with the same
 * workspace.
 */
int circatt_fused_bwd_dq(int kind, int dtype, int nsp, int64_t n1, int64_t n2, int32_t ws,
                         int64_t C, int64_t nheads, int64_t B, const void *q, const void *k,
                         const void *v, const void *y, const void *dy, const float *lse,
                         void *dq, void *workspace, int64_t workspace_bytes, void *stream);
int circatt_fused_bwd_dkdv(int kind, int dtype, int nsp, int64_t n1, int64_t n2, int32_t ws,
                           int64_t C, int64_t nheads, int64_t B, const void *q, const void *k,
                           const void *v, const void *dy, const float *lse, void *dk, void *dv,
                           const void *workspace, int64_t workspace_bytes, void *stream);

/*
 * circatt_fused_bwd without a workspace argument, for callers that cannot
 * allocate device memory (code under HIP graph capture, tight serving loops,
 * harnesses that forbid hipMalloc).  No counterpart in the reference.  The
 * per-row D = <dy, y> lives in a fixed device array inside the library, one
 * per GPU, held until the process ends: 16 MiB, i.e. at most
 * circatt_fused_bwd_noalloc_max_rows() = 4194304 rows (P * nheads * B);
 * larger problems fail with CIRCATT_ERR_INVALID.  The entry point calls no
 * allocating routine.  Every call on one GPU shares that array: calls that
 * overlap on one GPU (different streams, or different host threads) race
 * and must be serialised by the caller.  Nothing in the array needs to start
 * at zero (the dq pass writes every row's D before the dk/dv pass reads it).
 */
int64_t circatt_fused_bwd_noalloc_max_rows(void);
int circatt_fused_bwd_noalloc(int kind, int dtype, int nsp, int64_t n1, int64_t n2, int32_t ws,
                              int64_t C, int64_t nheads, int64_t B, const void *q,
                              const void *k, const void *v, const void *y, const void *dy,
                              const float *lse, void *dq, void *dk, void *dv, void *stream);

/*
 * Batch-dimension operations on a Circulant's CSR arrays (and other device
 * arrays), so that a host binding needs no array-library kernels of its own:
 *
 * circatt_fill: dst[i] = value for i < n.  The nzVal = 1 of a new pattern
 * (CUDA.ones at src/circulant.jl:68,90), a constant cotangent made dense.
 *
 * circatt_copy_blocks: for o < nouter, i < ninner, copies block_bytes bytes
 * from src + o*src_stride_outer + i*src_stride_inner to
 * dst + o*dst_stride_outer + i*dst_stride_inner (all in bytes; a stride of 0
 * replicates).  repeat over batch dims (src/array.jl:9,49-52), cat along a
 * batch dim (src/array.jl:62-64), the broadcast of a scale factor over heads
 * or batches (src/array.jl:179-186).  Destination blocks must not overlap each
 * other or the source; works on any element type (16, 8, 4 or 1-byte units,
 * the widest that divides every address, size and stride).
 *
 * circatt_sum_middle: dst[i + inner*o] = sum_s src[i + inner*(s + nsum*o)]
 * for a column-major (inner, nsum, outer) Float32 array, summed in double in
 * order of s.  sum(A; dims=d) over a batch dim d (src/array.jl:132-154), the
 * ∂c of the scale rrule over c's size-1 dims (src/rrules.jl:98-104), and the
 * pullback of repeat.
 *
 * circatt_count_unequal: *count (one device int64, overwritten) = the number
 * of i < n with a[i] != b[i], comparing 32-bit words (kind 0: Int32 rowPtr,
 * colVal) or Float32 values as floats (kind 1: -0 == 0, NaN != NaN).  == of
 * Circulants (src/array.jl:87-117) reads the count back.
 */
int circatt_fill(float *dst, int64_t n, float value, void *stream);
int circatt_copy_blocks(void *dst, const void *src, int64_t block_bytes, int64_t ninner,
                        int64_t dst_stride_inner, int64_t src_stride_inner, int64_t nouter,
                        int64_t dst_stride_outer, int64_t src_stride_outer, void *stream);
int circatt_sum_middle(const float *src, float *dst, int64_t inner, int64_t nsum, int64_t outer,
                       void *stream);
int circatt_count_unequal(int kind, int64_t n, const void *a, const void *b, int64_t *count,
                          void *stream);

/*
 * Token operators.  No counterpart in the reference: the attention of this
 * library for models of token sequences, whose window ends at the query (a
 * token sees no later one) and does not wrap.
 *
 * Signals are channels-last, Julia size (C, L, B), of CIRCATT_F32,
 * CIRCATT_F16 or CIRCATT_BF16: channel c of head g of token i of signal b at
 * g*dh + c + i*row + b*batch, strides in elements (row >= channels; rows
 * 16-byte aligned), so that the three parts of one projection's output are
 * read in place.  Outputs are contiguous.  kv_heads heads of keys and values
 * serve nheads/kv_heads heads of queries each: head h of q reads head
 * h / (nheads/kv_heads) of k and v.  dh is a multiple of 8 up to 128.  Sums,
 * softmax and statistics are Float32; probabilities and score gradients are
 * rounded to the element type where they enter a matrix product.
 *
 * circatt_sliding_fwd: token i of signal b, i < lengths[b] (lengths NULL: L),
 * sees key j <= i if j > i - window or j < sinks, and
 *   y = softmax_j(scale * <q_i, k_j>) v,
 * which is NaN where all visible scores are -inf.  Rows from lengths[b] on are
 * zero and nothing of q, k, v behind lengths[b] has an influence, whatever it
 * holds.  lse (nheads*L*B floats, for the backward) may be NULL.  y_rest (laid out
 * as y, 16-bit types only) receives what the rounding of y took, for the backward,
 * or is NULL.
 *
 * circatt_sliding_bwd: dq, dk, dv of the same (dk and dv both NULL: dq alone),
 * from y, y_rest and lse of the forward.  y_rest may be NULL; then <dy, y> is that
 * of the rounded y, which costs dq precision where few keys carry a row (up to 3
 * times the error of a form that rounds its results alone, else 1.6).  No
 * atomics; gradients of a shared head are summed over its queries' heads in a
 * fixed order.  Results overlap neither the arguments nor one another.
 */
int circatt_sliding_fwd(int dtype, int64_t L, int64_t B, int64_t nheads, int64_t kv_heads, int64_t dh,
                        int64_t window, int64_t sinks, float scale, const void *q, int64_t q_row,
                        int64_t q_batch, const void *k, int64_t k_row, int64_t k_batch, const void *v,
                        int64_t v_row, int64_t v_batch, const int32_t *lengths, void *y, void *y_rest,
                        float *lse, void *stream);
int64_t circatt_sliding_bwd_workspace_bytes(int dtype, int64_t L, int64_t B, int64_t nheads,
                                            int64_t kv_heads, int64_t dh, int64_t window, int64_t sinks);
int circatt_sliding_bwd(int dtype, int64_t L, int64_t B, int64_t nheads, int64_t kv_heads, int64_t dh,
                        int64_t window, int64_t sinks, float scale, const void *q, int64_t q_row,
                        int64_t q_batch, const void *k, int64_t k_row, int64_t k_batch, const void *v,
                        int64_t v_row, int64_t v_batch, const int32_t *lengths, const void *y,
                        const void *y_rest, const float *lse, const void *dy, int64_t dy_row,
                        int64_t dy_batch, void *dq, void *dk, void *dv, void *workspace,
                        int64_t workspace_bytes, void *stream);

/*
 * The same attention for serving, over a paged cache: a cache holds npages
 * pages of page_size tokens (a power of two), token s of page p at
 * p*page_stride + s*row_stride, and token j of sequence b lies in page
 * pages[b*pages_row + j/page_size].  lengths[b] tokens of sequence b are in
 * the cache, its new ones (the last) included.  The T rows of q are the new
 * tokens of the B sequences in order: sequence b has the rows offsets[b] ..
 * offsets[b+1] - 1 (offsets: B+1 ascending numbers from 0; NULL: one row for
 * each sequence, T = B).  pages, lengths and offsets are device arrays that
 * are read when the kernel runs, so a captured call follows their contents.
 * A page number outside [0, npages) is never followed: its tokens are hidden.
 * Tokens from max_pages * page_size on see nothing, and a row that sees nothing is
 * zero.  Offsets that do not ascend leave rows unspecified.  Rows of y behind the last sequence are
 * zero with zero_tail = 1 and left as they were with 0.  y must not overlap q or
 * the caches.  Row strides are at most 2^22 elements, a cache 63 GiB end to end.
 *
 * circatt_paged_append writes the new tokens' k and v, packed the same way,
 * into their pages; a token whose page number is outside the cache is dropped.
 * No two tokens may share a slot, and k and v hold no slot that is written.
 */
int64_t circatt_paged_workspace_bytes(int dtype, int64_t T, int64_t B, int64_t nheads, int64_t kv_heads,
                                      int64_t dh, int64_t window, int64_t sinks, int64_t page_size,
                                      int64_t max_pages);
int circatt_paged_attention(int dtype, int64_t T, int64_t B, int64_t nheads, int64_t kv_heads,
                            int64_t dh, int64_t window, int64_t sinks, float scale, const void *q,
                            int64_t q_row, const void *cache_k, const void *cache_v, int64_t npages,
                            int64_t page_size, int64_t page_stride, int64_t row_stride,
                            const int32_t *pages, int64_t pages_row, int64_t max_pages,
                            const int32_t *lengths, const int32_t *offsets, void *y, int zero_tail,
                            void *workspace, int64_t workspace_bytes, void *stream);
int circatt_paged_append(int dtype, int64_t T, int64_t B, int64_t channels, const void *k, int64_t k_row,
                         const void *v, int64_t v_row, void *cache_k, void *cache_v, int64_t npages,
                         int64_t page_size, int64_t page_stride, int64_t row_stride,
                         const int32_t *pages, int64_t pages_row, int64_t max_pages,
                         const int32_t *lengths, const int32_t *offsets, void *stream);

/*
 * The same attention with shaped scores.  With x = scale * <q_i, k_j>,
 *   s_ij = cap * tanh(x / cap) - slopes[h] * |i - j|
 * takes the place of x: cap 0 leaves x as it is, slopes (nheads Float32 numbers on the
 * device) may be NULL.  With prefix (B numbers) every token of signal b also sees the
 * first prefix[b] tokens, those before them included.  With places ((B, L) numbers,
 * places_row apart from signal to signal) a signal holds documents one after another:
 * token i's begins at i - places[i], and tokens before that are not seen; sinks are a
 * document's first tokens.  Places of a document count up from 0, others give
 * unspecified rows.  Prefix and places do not go together.  slopes need L (or max_pages *
 * page_size) of at most 2^24.  No gradient of the slopes is formed.
 *
 * biased: whether slopes will be given; masked: 0, 1 with places, 2 with a prefix.
 */
int circatt_shaped_fwd(int dtype, int64_t L, int64_t B, int64_t nheads, int64_t kv_heads, int64_t dh,
                       int64_t window, int64_t sinks, float scale, float cap, const float *slopes,
                       const int32_t *prefix, const int32_t *places, int64_t places_row, const void *q,
                       int64_t q_row, int64_t q_batch, const void *k, int64_t k_row, int64_t k_batch,
                       const void *v, int64_t v_row, int64_t v_batch, const int32_t *lengths, void *y,
                       void *y_rest, float *lse, void *stream);
int64_t circatt_shaped_bwd_workspace_bytes(int dtype, int64_t L, int64_t B, int64_t nheads,
                                           int64_t kv_heads, int64_t dh, int64_t window, int64_t sinks,
                                           int biased, int masked);
int circatt_shaped_bwd(int dtype, int64_t L, int64_t B, int64_t nheads, int64_t kv_heads, int64_t dh,
                       int64_t window, int64_t sinks, float scale, float cap, const float *slopes,
                       const int32_t *prefix, const int32_t *places, int64_t places_row, const void *q,
                       int64_t q_row, int64_t q_batch, const void *k, int64_t k_row, int64_t k_batch,
                       const void *v, int64_t v_row, int64_t v_batch, const int32_t *lengths, const void *y,
                       const void *y_rest, const float *lse, const void *dy, int64_t dy_row,
                       int64_t dy_batch, void *dq, void *dk, void *dv, void *workspace,
                       int64_t workspace_bytes, void *stream);
/* circatt_paged_attention likewise.  Its workspace is circatt_shaped_paged_workspace_bytes';
 * prefixed: whether a prefix will be given.  (circatt_paged_workspace_bytes' is enough, but
 * leaves the walk of a long prefix to few workgroups.) */
int64_t circatt_shaped_paged_workspace_bytes(int dtype, int64_t T, int64_t B, int64_t nheads,
                                             int64_t kv_heads, int64_t dh, int64_t window, int64_t sinks,
                                             int64_t page_size, int64_t max_pages, int prefixed);
int circatt_shaped_paged(int dtype, int64_t T, int64_t B, int64_t nheads, int64_t kv_heads, int64_t dh,
                         int64_t window, int64_t sinks, float scale, float cap, const float *slopes,
                         const int32_t *prefix, const void *q, int64_t q_row, const void *cache_k,
                         const void *cache_v, int64_t npages, int64_t page_size, int64_t page_stride,
                         int64_t row_stride, const int32_t *pages, int64_t pages_row, int64_t max_pages,
                         const int32_t *lengths, const int32_t *offsets, void *y, int zero_tail,
                         void *workspace, int64_t workspace_bytes, void *stream);

/*
 * The pages of a paged cache.  A sequence of n tokens holds the first n / page_size
 * (rounded up) pages of its row of the table, and counts[p] (npages numbers) says how
 * often page p is held, 0: it is free.  Tables, lengths and counts are read on the device
 * and written to new arrays (rows of max_pages, -1 behind a sequence's pages), which
 * overlap nothing that is read; numbers outside the cache are kept and not counted.
 *
 * circatt_paged_fork: new sequence n of N goes on from sequence source[n], with which it
 * shares all pages; a number outside [0, B) gives an empty one.  Old sequences that
 * nobody goes on from give their pages back.
 *
 * circatt_paged_resize: sequence b comes to to[b] tokens, no more than its row of the
 * table holds (below 0: it stays as it is).  First pages behind the new lengths are given
 * back.  Then sequences get the pages that they lack, in their order, the free pages
 * of the lowest numbers first.  A sequence that grows and whose last page is
 * partly filled and held more than once gets one for it too, and the part's tokens are
 * copied there, in both caches; of several that do so in one call each gets one.  A
 * sequence that shrinks gets none: where tokens are taken off a sequence and new ones
 * appended, it is resized to what stays of it, and then to that with the new ones.  From the first sequence on that finds too few free
 * pages, those that need any stay as they are, which their new lengths show.
 *
 * circatt_paged_compact: the held pages from number `used` on, `used` being how many are
 * held, move in order to the free numbers below it, in both caches, and table and counts
 * follow.  What the pages from `used` on hold stays there.
 *
 * The pages of a cache do not overlap one another, B and N are at most 65535, and
 * B * (max_pages + 1) is below 2^31.
 */
int circatt_paged_fork(int64_t B, int64_t npages, int64_t page_size, const int32_t *pages,
                       int64_t pages_row, int64_t max_pages, const int32_t *lengths,
                       const int32_t *counts, int64_t N, const int32_t *source, int32_t *out_pages,
                       int32_t *out_lengths, int32_t *out_counts, void *stream);
int64_t circatt_paged_resize_workspace_bytes(int64_t B, int64_t npages);
int circatt_paged_resize(int dtype, int64_t channels, void *cache_k, void *cache_v, int64_t npages,
                         int64_t page_size, int64_t page_stride, int64_t row_stride, int64_t B,
                         const int32_t *pages, int64_t pages_row, int64_t max_pages,
                         const int32_t *lengths, const int32_t *counts, const int32_t *to,
                         int32_t *out_pages, int32_t *out_lengths, int32_t *out_counts, void *workspace,
                         int64_t workspace_bytes, void *stream);
int64_t circatt_paged_compact_workspace_bytes(int64_t npages);
int circatt_paged_compact(int dtype, int64_t channels, void *cache_k, void *cache_v, int64_t npages,
                          int64_t page_size, int64_t page_stride, int64_t row_stride, int64_t B,
                          const int32_t *pages, int64_t pages_row, int64_t max_pages,
                          const int32_t *counts, int32_t *out_pages, int32_t *out_counts,
                          void *workspace, int64_t workspace_bytes, void *stream);

/*
 * Rotary positions with naxes (1 to 3) axes on P tokens of each of nb signals
 * (rows x_row elements apart): the first 2*p1 channels of a head belong to
 * axis 1, the next 2*p2 to axis 2, then 2*p3; pair i of an axis (channels i
 * and i + p of its section, or 2i and 2i + 1 when interleaved) is turned by
 * position * base^(-i/p); the channels behind stay.  positions (Int32, naxes a
 * token, P tokens; pos_batch apart from signal to signal, 0: shared), or NULL:
 * token i1 + n1*(i2 + n2*i3) has the positions (i1, i2, i3).  inverse: the
 * turn the other way, which is the gradient.  The angle is formed in Float64.
 *
 * circatt_axial_rotary_wide takes the base as a sum of two Float32 numbers, the
 * nearest one and what that leaves (48 bits): position * base^(-i/p) of a base that
 * Float32 does not hold is off by 1e-3 at position 2^20 if it is rounded first.
 */
int circatt_axial_rotary(int dtype, int inverse, int interleaved, int naxes, int64_t n1, int64_t n2,
                         int64_t n3, int64_t P, int64_t nb, int64_t nheads, int64_t dh, int32_t p1,
                         int32_t p2, int32_t p3, float base, const void *x, int64_t x_row,
                         const int32_t *positions, int64_t pos_batch, void *y, void *stream);
int circatt_axial_rotary_wide(int dtype, int inverse, int interleaved, int naxes, int64_t n1, int64_t n2,
                              int64_t n3, int64_t P, int64_t nb, int64_t nheads, int64_t dh, int32_t p1,
                              int32_t p2, int32_t p3, float base, float base_rest, const void *x,
                              int64_t x_row, const int32_t *positions, int64_t pos_batch, void *y,
                              void *stream);

/*
 * Device memory helpers for hosts without a GPU array package (the reference
 * gets these from CUDA.jl).  kind: 0 host->device, 1 device->host,
 * 2 device->device.
 */
int circatt_malloc(void **ptr, int64_t bytes);
int circatt_free(void *ptr);
int circatt_memcpy(void *dst, const void *src, int64_t bytes, int kind);
int circatt_stream_synchronize(void *stream);

#ifdef __cplusplus
}
#endif

#endif /* CIRCATT_H */
