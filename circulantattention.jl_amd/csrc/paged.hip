// Attention of new tokens over a paged cache, and the cache's append.
#include "token_tile.h"

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
// Attention.  Rows are packed as in sliding.hip: row r of a sequence and a head
// of keys is head r % G of its new token r / G.  A block is R of them:
//   R = 128, a tile of keys for four wavefronts of 32 rows each (chunks);
//   R = 32, tiles of 32 keys for each of NW wavefronts, which share the rows and
//   join their sums at the end (single tokens: bound by reading the cache).
// Blocks of sequence b are numbered from offsets[b] G / R + b on, so that a block
// finds its sequence from the offsets on the device.  Where blocks are few, each
// is split along its tiles over `splits` workgroups, whose partial sums
// paged_join adds up.
struct PagedGrid {
    int blocks;   // numbers of blocks of one head of keys
    int splits;
    int64_t rows;  // of partial sums
};

// Sequence b with its block's first row, rows and positions; b < 0: none.
struct Block {
    int b, r0, rows, first, len;
    int64_t q0;  // row of q of its first new token
};
template <int R>
__device__ __forceinline__ Block find_block(const PagedProblem &pr, int id) {
    Block x;
    if (pr.offsets == nullptr) {
        const int per = (pr.G + R - 1) / R;
        x.b = id / per;
        x.r0 = (id - x.b * per) * R;
        x.rows = pr.G;
        x.q0 = x.b;
    } else {
        // the last b whose number is not past id: ascending, so a count
        const int lane = threadIdx.x & 63;
        int count = 0;
        for (int b0 = 0; b0 < pr.B; b0 += 64) {
            const int b = b0 + lane;
            const bool in = b < pr.B && (int64_t)pr.offsets[b] * pr.G / R + b <= id;
            const int got = __popcll(__ballot(in));
            count += got;
            if (got < 64) break;
        }
        x.b = uniform(count - 1);
        if (x.b < 0) return x;
        const int o = uniform(pr.offsets[x.b]), m = uniform(pr.offsets[x.b + 1]) - o;
        x.r0 = (id - (int)((int64_t)o * pr.G / R + x.b)) * R;
        x.rows = m * pr.G;
        x.q0 = o;
        if (o < 0 || m < 0 || (int64_t)o + m > pr.T) x.rows = 0;
    }
    x.len = uniform(pr.lengths[x.b]);
    x.len = x.len > 0 ? x.len : 0;
    x.first = x.len - x.rows / pr.G;
    if (x.r0 >= x.rows) x.b = -1;
    return x;
}

// What a block's rows may read of the cache: keys [0, S) and [low, len) below
// the table's end.
template <typename T>
struct Pages {
    const T *k, *v;
    const int32_t *table;
    int64_t page_stride, row_stride;
    int npages, log2, low, S, len;
    // the cache row of key j, -1 if it is not there
    __device__ __forceinline__ int row(int j) const {
        if (j >= len || (j < low && j >= S)) return -1;
        const int pg = table[j >> log2];
        return (unsigned)pg < (unsigned)npages ? (pg << log2) | (j & ((1 << log2) - 1)) : -1;
    }
    __device__ __forceinline__ int64_t at(int row) const {
        return (row >> log2) * page_stride + (row & ((1 << log2) - 1)) * row_stride;
    }
};

__device__ const uint32_t kZeros[4] = {0, 0, 0, 0};

// KT keys and values, lane l of the calling wavefronts holding the cache row of
// the tile's key l, into LDS by THREADS threads; rows that are not there and
// units from D on are zeros.
template <typename T, int DP, int KT, int THREADS>
__device__ __forceinline__ void fetch_pages(const Pages<T> &pg, int row, int D, const CIRCATT_LDS char *kt) {
    typedef Tile<T, DP> Tl;
    const int tid = threadIdx.x & (THREADS - 1), units = D * (int)sizeof(T) / 16;
    const unsigned m0 = lds_byte(kt) + uniform(tid >> 6) * 1024;
#pragma unroll
    for (int k = 0; k < KT * Tl::PC / THREADS; ++k) {
        const int slot = tid + k * THREADS, r = slot / Tl::PC, u = (slot % Tl::PC) ^ Tl::f(r);
        const int cr = __shfl(row, r, 64);
        const bool there = cr >= 0 && u < units;
        const int64_t at = there ? pg.at(cr) + u * (16 / (int)sizeof(T)) : 0;
        dma16_global(there ? (const void *)(pg.k + at) : (const void *)kZeros, m0 + k * THREADS * 16);
        dma16_global(there ? (const void *)(pg.v + at) : (const void *)kZeros, m0 + KT * Tl::ROW + k * THREADS * 16);
    }
}

// A row's partial sums: its output channels (D), maximum and sum behind all.
struct Partial {
    float *o, *ml;
    __device__ Partial(const PagedProblem &pr, const PagedGrid &gr, int64_t row)
        : o(pr.work + row * pr.D), ml(pr.work + gr.rows * pr.D + row * 2) {}
};
template <int OT>
__device__ __forceinline__ void store_partial(const f16v (&o)[OT], Partial p, float m, float l, int D, int lane) {
    if (l != 0.f)
#pragma unroll
        for (int t = 0; t < OT; ++t)
#pragma unroll
            for (int i = 0; i < 16; i += 4) {
                const int d = 32 * t + 2 * i + 4 * (lane >> 5);
                if (d < D) *reinterpret_cast<f4v *>(p.o + d) = f4v{o[t][i], o[t][i + 1], o[t][i + 2], o[t][i + 3]};
            }
    if (lane < 32) {
        p.ml[0] = m;
        p.ml[1] = l;
    }
}

template <typename T>
__device__ __forceinline__ PagedKV<T> paged_rows_of(const PagedProblem &pr, int b, int64_t head) {
    return PagedKV<T>{static_cast<const T *>(pr.k) + head, static_cast<const T *>(pr.v) + head, pr.page_stride,
                      pr.row_stride, pr.pages + b * pr.pages_row, pr.npages, pr.page_log2};
}

// One workgroup: a block, a head of keys and a part of the block's tiles.
// ONE: R = 32 and the wavefronts share the rows.
template <typename T, int DP, bool ONE>
struct PagedShape {
    static constexpr int NW = ONE && sizeof(T) == 4 && DP > 64 ? 2 : 4;
    static constexpr int R = ONE ? 32 : 128;
    static constexpr int KT = ONE || sizeof(T) == 4 ? 32 : 64;
    static constexpr int TILE = KT * Tile<T, DP>::ROW;
    static constexpr int LDS = (ONE ? NW : 1) * 4 * TILE;
};

template <typename T, int DP, bool ONE>
__global__ __launch_bounds__((64 * PagedShape<T, DP, ONE>::NW), ((sizeof(T) == 4 && DP > 64) || ONE ? 1 : 2))
void paged_kernel(PagedProblem pr, PagedGrid gr) {
    typedef PagedShape<T, DP, ONE> Sh;
    typedef Tile<T, DP> Tl;
    constexpr int KT = Sh::KT, NB = KT / 32, R = Sh::R, NW = Sh::NW, OT = DP / 32;
    __shared__ __attribute__((aligned(1024))) char lds_mem[Sh::LDS];
    const int lane = threadIdx.x & 63, wave = uniform(threadIdx.x >> 6);
    const CIRCATT_LDS char *lds = (const CIRCATT_LDS char *)lds_mem + (ONE ? wave * 4 * Sh::TILE : 0);
    const int hk = blockIdx.y, split = blockIdx.z;
    if ((int)blockIdx.x >= gr.blocks) {
        // rows behind the last sequence
        if (hk != 0 || split != 0) return;
        const int end = pr.offsets[pr.B];
        const int64_t per = (int64_t)pr.H * pr.D / (16 / (int)sizeof(T)), from = (int64_t)(end < 0 ? 0 : end) * per;
        const int64_t step = (int64_t)(gridDim.x - gr.blocks) * blockDim.x;
        typedef uint32_t u4 __attribute__((ext_vector_type(4)));
        for (int64_t i = from + (int64_t)(blockIdx.x - gr.blocks) * blockDim.x + threadIdx.x; i < pr.T * per; i += step)
            static_cast<u4 *>(pr.y)[i] = u4{};
        return;
    }
    const Block w = find_block<R>(pr, blockIdx.x);
    if (w.b < 0) return;
    const int r0 = w.r0 + (ONE ? 0 : 32 * wave), r = r0 + (lane & 31);
    const int rr = r < w.rows ? r : w.rows - 1, tok = rr / pr.G, g = rr - tok * pr.G;
    const int64_t held = (int64_t)pr.maxp << pr.page_log2;
    // a position before the first token or behind the table: the row sees nothing
    const int pos = w.first + tok, at = pos >= held ? -1 : pos;
    const bool live = r0 < w.rows;
    // the block's positions, and this wavefront's
    const int b_last = w.r0 + R - 1 < w.rows ? w.r0 + R - 1 : w.rows - 1;
    int blo = w.first + w.r0 / pr.G, bhi = w.first + b_last / pr.G;
    if (bhi >= held) bhi = (int)held - 1;
    if (blo < 0) blo = 0;
    const int lo = uniform(at), hi = __builtin_amdgcn_readlane(at, 31);
    const bool plain = lo >= 0 && hi >= lo;  // ascending: no row without sight
    const Sight see{pr.W, pr.S};
    const TileList<KT> tiles(blo, blo > bhi ? -1 : bhi, pr.W, pr.S);
    const int64_t head = (int64_t)hk * pr.D;
    const Pages<T> pg{static_cast<const T *>(pr.k) + head, static_cast<const T *>(pr.v) + head,
                      pr.pages + w.b * pr.pages_row, pr.page_stride, pr.row_stride, pr.npages, pr.page_log2,
                      blo - pr.W + 1, pr.S, bhi + 1};
    const int parts = gr.splits * (ONE ? NW : 1), part = split * (ONE ? NW : 1) + (ONE ? wave : 0);
    const int i0 = (int)((int64_t)tiles.count * part / parts), i1 = (int)((int64_t)tiles.count * (part + 1) / parts);
    const float c = pr.scale * kLog2e;
    Rows<T, DP> x;
    const T *qr = static_cast<const T *>(pr.q) + (w.q0 + tok) * pr.q_row + (head * pr.G + (int64_t)g * pr.D);
    if (i0 < i1) {
        const unsigned row_at = Tl::row_lane(lane), col_at = Tl::col_lane(lane);
        auto key_row = [&](int i) { return lane < KT ? pg.row(tiles.key(i) + lane) : -1; };
        // the rows of the tile in work, of the next one, and of the one after
        int now = key_row(i0), next = i0 + 1 < i1 ? key_row(i0 + 1) : -1;
        fetch_pages<T, DP, KT, ONE ? 64 : 256>(pg, now, pr.D, lds);
        x.start(qr, pr.D, lane);
        loads_here();
        for (int i = i0; i < i1; ++i) {
            if (ONE) dma_wait();
            else dma_barrier();
            int after = -1;
            if (i + 1 < i1) {
                fetch_pages<T, DP, KT, ONE ? 64 : 256>(pg, next, pr.D, lds + ((i + 1 - i0) & 1) * 2 * Sh::TILE);
                if (i + 2 < i1) after = key_row(i + 2);
            }
            const int k0 = tiles.key(i);
            const uint64_t hidden = ~__ballot(now >= 0) & (KT == 64 ? ~0ull : 0xffffffffull);
            now = next;
            next = after;
            if (!live || (plain && see.none(lo, hi, k0, KT))) continue;
            const unsigned to = lds_byte(lds) + ((i - i0) & 1) * 2 * Sh::TILE;
            x.template tile<NB>(row_at + to, col_at + to + Sh::TILE, lane, at, k0, see,
                                !(plain && see.all(lo, hi, k0, KT)) || hidden != 0, hidden, c);
        }
    } else {
        x.start(qr, 0, lane);
    }
    float l = x.total(), m = x.m;
    if (ONE) {
        // join the wavefronts' sums in LDS: each one's maximum and sum, then the
        // outputs, 32 channels at a time, in the order of the wavefronts
        __syncthreads();
        float *ml = reinterpret_cast<float *>(lds_mem), *buf = ml + NW * 64;
        if (lane < 32) {
            ml[wave * 64 + lane] = m;
            ml[wave * 64 + 32 + lane] = l;
        }
        __syncthreads();
        float mm = -INFINITY, ll = 0.f;
        for (int v = 0; v < NW; ++v) mm = fmaxf(mm, ml[v * 64 + (lane & 31)]);
        for (int v = 0; v < NW; ++v) {
            const float mv = ml[v * 64 + (lane & 31)];
            ll += mv == -INFINITY ? ml[v * 64 + 32 + (lane & 31)] : ml[v * 64 + 32 + (lane & 31)] * __builtin_amdgcn_exp2f(mv - mm);
        }
        const float f = m == -INFINITY ? 1.f : __builtin_amdgcn_exp2f(m - mm);
#pragma unroll
        for (int t = 0; t < OT; ++t) {
#pragma unroll
            for (int i = 0; i < 16; ++i) buf[(wave * 16 + i) * 64 + lane] = x.o[t][i] * f;
            __syncthreads();
            if (wave == 0)
#pragma unroll
                for (int i = 0; i < 16; ++i) {
                    float sum = 0.f;
                    for (int v = 0; v < NW; ++v) sum += buf[(v * 16 + i) * 64 + lane];
                    x.o[t][i] = sum;
                }
            __syncthreads();
        }
        m = mm;
        l = ll;
        if (wave != 0) return;
    }
    if (!live) return;
    if (gr.splits > 1) {
        if (r < w.rows)
            store_partial(x.o, Partial(pr, gr, (((int64_t)blockIdx.x * pr.Hk + hk) * gr.splits + split) * R + r - w.r0), m, l,
                          pr.D, lane);
        return;
    }
    const float inv = l == 0.f ? 0.f : 1.f / l;
    T *y = static_cast<T *>(pr.y) + w.q0 * pr.H * pr.D + head * pr.G;
    uint64_t again = __ballot(r < w.rows && store_channels(x.o, y + ((int64_t)tok * pr.H + g) * pr.D, pr.D, lane, inv));
    again = (again | again >> 32) & 0xffffffffu;
    const PagedKV<T> kv = paged_rows_of<T>(pr, w.b, head);
    for (; again; again &= again - 1) {
        const int j = __builtin_ctzll(again);
        const int tj = __builtin_amdgcn_readlane(tok, j), gj = __builtin_amdgcn_readlane(g, j);
        forward_row(static_cast<const T *>(pr.q) + (w.q0 + tj) * pr.q_row + (head * pr.G + (int64_t)gj * pr.D),
                    y + ((int64_t)tj * pr.H + gj) * pr.D, (float *)nullptr, kv, __builtin_amdgcn_readlane(at, j), pr.W, pr.S,
                    pr.D, c);
    }
}

// Adds up a row's partial sums in the order of the splits: a wavefront a row.
template <typename T, int R>
__global__ __launch_bounds__(256) void paged_join(PagedProblem pr, PagedGrid gr) {
    const int64_t id = (int64_t)blockIdx.x * 4 + (threadIdx.x >> 6);
    const int lane = threadIdx.x & 63;
    const int64_t t = id / pr.H;
    if (t >= pr.T) return;
    const int h = (int)(id - t * pr.H), hk = h / pr.G, g = h - hk * pr.G;
    const NewToken w = new_token(pr.offsets, pr.lengths, pr.B, t);
    if (w.b >= pr.B) return;
    int64_t block, row;
    if (pr.offsets == nullptr) {
        block = t * ((pr.G + R - 1) / R) + g / R;
        row = g % R;
    } else {
        const int64_t o = pr.offsets[w.b], r = (t - o) * pr.G + g;
        block = o * pr.G / R + w.b + r / R;
        row = r % R;
    }
    const int64_t slot = ((block * pr.Hk + hk) * gr.splits) * R + row;
    float m = -INFINITY, l = 0.f;
    for (int s = 0; s < gr.splits; ++s) m = fmaxf(m, Partial(pr, gr, slot + s * R).ml[0]);
    Pair o{0.f, 0.f};
    for (int s = 0; s < gr.splits; ++s) {
        const Partial p(pr, gr, slot + s * R);
        const float ls = p.ml[1];
        if (ls == 0.f) continue;  // saw nothing, and wrote no outputs
        const float f = __builtin_amdgcn_exp2f(p.ml[0] - m);
        const Pair x = load_row(p.o, lane, pr.D);
        l += ls * f;
        o.a += x.a * f;
        o.b += x.b * f;
    }
    const float inv = l == 0.f ? 0.f : 1.f / l;
    o.a *= inv;
    o.b *= inv;
    T *y = static_cast<T *>(pr.y) + (t * pr.H + h) * pr.D;
    store_row(y, lane, pr.D, o);
    if (__any(!(fabsf(o.a) + fabsf(o.b) < INFINITY))) {
        const int64_t held = (int64_t)pr.maxp << pr.page_log2;
        forward_row(static_cast<const T *>(pr.q) + t * pr.q_row + (int64_t)h * pr.D, y, (float *)nullptr,
                    paged_rows_of<T>(pr, w.b, (int64_t)hk * pr.D), w.pos >= held ? -1 : w.pos, pr.W, pr.S, pr.D,
                    pr.scale * kLog2e);
    }
}

// Rows of 32 for each sequence and head of keys where there is no more than
// that on average, else of 128.
bool rows_of_32(const PagedProblem &pr) { return pr.T * pr.G <= (int64_t)pr.B * 32; }

PagedGrid paged_grid(const PagedProblem &pr) {
    const bool one = rows_of_32(pr);
    const int R = one ? 32 : 128;
    const bool wide = pr.dtype == CIRCATT_F32;
    const int KT = one || wide ? 32 : 64, NW = !one ? 1 : wide && pr.D > 64 ? 2 : 4;
    PagedGrid gr;
    gr.blocks = (int)(pr.T * pr.G / R) + pr.B;
    // two workgroups a compute unit, four tiles for each wavefront at least
    const int64_t span = (int64_t)pr.maxp * pr.page, most = (int64_t)pr.W + pr.S + R / pr.G + KT;
    const int64_t tiles = ((span < most ? span : most) + KT - 1) / KT;
    int64_t splits = 512 / ((int64_t)gr.blocks * pr.Hk), limit = tiles / (4 * NW);
    splits = splits < limit ? splits : limit;
    gr.splits = (int)(splits < 1 ? 1 : splits > 256 ? 256 : splits);
    gr.rows = gr.splits > 1 ? (int64_t)gr.blocks * pr.Hk * gr.splits * R : 0;
    return gr;
}

template <typename T, int DP>
void launch(const PagedProblem &pr, hipStream_t s) {
    const PagedGrid gr = paged_grid(pr);
    const bool tail = pr.zero_tail && pr.offsets != nullptr;
    const int R = rows_of_32(pr) ? 32 : 128;
    const dim3 grid(pr.offsets == nullptr ? pr.B * ((pr.G + R - 1) / R) : gr.blocks + (tail ? 8 : 0), pr.Hk, gr.splits);
    if (rows_of_32(pr)) paged_kernel<T, DP, true><<<grid, 64 * PagedShape<T, DP, true>::NW, 0, s>>>(pr, gr);
    else paged_kernel<T, DP, false><<<grid, 256, 0, s>>>(pr, gr);
    if (gr.splits > 1) {
        const unsigned rows = (unsigned)((pr.T * pr.H + 3) / 4);
        if (rows_of_32(pr)) paged_join<T, 32><<<rows, 256, 0, s>>>(pr, gr);
        else paged_join<T, 128><<<rows, 256, 0, s>>>(pr, gr);
    }
}
template <int DT>
void launch(const PagedProblem &pr, hipStream_t s) {
    typedef typename Elem<DT>::T T;
    if (pr.D <= 32) launch<T, 32>(pr, s);
    else if (pr.D <= 64) launch<T, 64>(pr, s);
    else if (pr.D <= 96) launch<T, 96>(pr, s);
    else launch<T, 128>(pr, s);
}

// ---------------------------------------------------------------------------
// Append.
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

int64_t paged_workspace_floats(const PagedProblem &pr) { return paged_grid(pr).rows * (pr.D + 2); }

hipError_t launch_paged(const PagedProblem &pr, hipStream_t s) {
    if (pr.dtype == CIRCATT_F32) launch<0>(pr, s);
    else if (pr.dtype == CIRCATT_F16) launch<2>(pr, s);
    else launch<3>(pr, s);
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
