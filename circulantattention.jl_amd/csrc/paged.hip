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
// of keys is head r % G of its new token r / G.  A block is R of them.
//   few_rows (R = 32): tiles of 32 keys for each of NW wavefronts, which share the
//   rows and join their sums at the end; bound by reading the cache.  The next
//   token of 64 sequences of up to 8192, window 4096, 8 heads of 128 keys, bf16:
//   182 us, 5.2 TB/s, the rate of a large copy.
//   chunk_rows (R = 128): four wavefronts of 32 rows share the tiles, as in
//   sliding_fwd, and NG such groups share the block's keys, half a round apart (in
//   step: 91 us at the size that follows); bound by the products.  Two chunks of
//   512 tokens behind up to 12000, window 4096, 32 heads of 128 over 8: 86 us, 650
//   TFLOP/s.
// Where blocks are few, each is split along its tiles over `splits` workgroups,
// whose partial sums paged_join adds up.  A mixed batch has both kinds in one launch
// (33 sequences, some of one token, some of up to 128: 59 us; in two launches 104).
enum Which { kAll, kShort, kLong };  // sequences: all, those of up to 32 rows, the others
struct PagedGrid {
    int which;
    int blocks;        // numbers of blocks of one head of keys
    int splits;
    int64_t at, rows;  // of partial sums: floats before them, rows
};

// Sequence b with its block's first row, rows and positions; b < 0: none.
struct Block {
    int b, r0, rows, first, len;
    int64_t q0;  // row of q of its first new token
};
// Blocks of sequence b are numbered from offsets[b] G / R + b on (from b without
// offsets or among short sequences, which have one), so that a block finds its
// sequence from the offsets on the device.
template <int R>
__device__ __forceinline__ Block find_block(const PagedProblem &pr, int which, int id) {
    Block x;
    if (pr.offsets == nullptr) {
        const int per = (pr.G + R - 1) / R;
        x.b = id / per;
        x.r0 = (id - x.b * per) * R;
        x.rows = pr.G;
        x.q0 = x.b;
        if (x.b >= pr.B) x.b = -1;
    } else {
        if (which == kShort) {
            x.b = id < pr.B ? id : -1;
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
        }
        if (x.b < 0) return x;
        const int o = uniform(pr.offsets[x.b]), m = uniform(pr.offsets[x.b + 1]) - o;
        x.r0 = which == kShort ? 0 : (id - (int)((int64_t)o * pr.G / R + x.b)) * R;
        x.rows = m * pr.G;
        x.q0 = o;
        if (o < 0 || m < 0 || (int64_t)o + m > pr.T) x.rows = 0;
        if (which != kAll && (x.rows <= 32) != (which == kShort)) x.rows = 0;
    }
    if (x.b < 0) return x;
    x.len = uniform(pr.lengths[x.b]);
    x.len = x.len > 0 ? x.len : 0;
    x.first = x.len - x.rows / pr.G;
    // (before its first row: offsets that do not ascend)
    if (x.r0 < 0 || x.r0 >= x.rows) x.b = -1;
    return x;
}

// One row of a block as its lane sees it, and what the block's rows see together.
// at: its position, -1 where it sees nothing (before the first token, or behind the
// table's end); blo, bhi: the block's first and last position that see something.
struct RowSight {
    int tok, g, at, blo, bhi;
    template <int R>
    __device__ static __forceinline__ RowSight of(const PagedProblem &pr, const Block &w, int r) {
        RowSight x;
        const int rr = r < w.rows ? r : w.rows - 1, last = w.r0 + R - 1 < w.rows ? w.r0 + R - 1 : w.rows - 1;
        const int64_t held = (int64_t)pr.maxp << pr.page_log2;
        x.tok = rr / pr.G;
        x.g = rr - x.tok * pr.G;
        const int pos = w.first + x.tok;
        x.at = pos >= held ? -1 : pos;
        x.blo = w.first + w.r0 / pr.G;
        x.bhi = w.first + last / pr.G;
        if (x.bhi >= held) x.bhi = (int)held - 1;
        if (x.blo < 0) x.blo = 0;
        if (x.blo > x.bhi) x.bhi = -1;  // nothing: no tiles
        return x;
    }
};

// What a block's rows may read of the cache: keys [0, S) and [low, len).
template <typename T>
struct Pages {
    const T *k, *v;
    const int32_t *table;
    uint32_t page_units, row_units;  // strides in 16 bytes
    int npages, log2, low, S, len;
    __device__ __forceinline__ Pages(const PagedProblem &pr, const Block &w, const RowSight &x, int hk)
        : k(static_cast<const T *>(pr.k) + (int64_t)hk * pr.D), v(static_cast<const T *>(pr.v) + (int64_t)hk * pr.D),
          table(pr.pages + w.b * pr.pages_row), page_units((uint32_t)(pr.page_stride * (int)sizeof(T) / 16)),
          row_units((uint32_t)(pr.row_stride * (int)sizeof(T) / 16)), npages(pr.npages), log2(pr.page_log2),
          low(x.blo - pr.W + 1), S(pr.S), len(x.bhi + 1) {}
    // key j's row in units of 16 bytes from the cache's start, kNone if not there
    // from its page's number.  The number is loaded a round before the row is
    // formed: a load that is used in its own round would make the wavefront wait for
    // the DMA that it issued since.
    static constexpr uint32_t kNone = ~0u;
    __device__ __forceinline__ int page(int j) const { return table[(j < len ? j : len - 1) >> log2]; }
    __device__ __forceinline__ uint32_t row(int j, int pg) const {
        if (j >= len || (j < low && j >= S) || (unsigned)pg >= (unsigned)npages) return kNone;
        return pg * page_units + (j & ((1 << log2) - 1)) * row_units;
    }
};

__device__ const uint32_t kZeros[4] = {0, 0, 0, 0};

// KT keys (or values) from p into LDS by THREADS threads, this one the tid-th;
// lane l of each of their wavefronts holds the row of the tile's key l.  Rows that
// are not there and units from D on are zeros.
template <typename T, int DP, int KT, int THREADS>
__device__ __forceinline__ void fetch_paged(const T *p, uint32_t row, int D, int tid, unsigned to) {
    typedef Tile<T, DP> Tl;
    const int units = D * (int)sizeof(T) / 16;
    const unsigned m0 = to + uniform(tid >> 6) * 1024;
#pragma unroll
    for (int k = 0; k < KT * Tl::PC / THREADS; ++k) {
        const int slot = tid + k * THREADS, r = slot / Tl::PC, u = (slot % Tl::PC) ^ Tl::f(r);
        const uint32_t cr = __shfl(row, r, 64);
        const char *at = reinterpret_cast<const char *>(p) + u * 16 + ((uint64_t)cr << 4);
        dma16_global(cr != Pages<T>::kNone && u < units ? (const void *)at : (const void *)kZeros, m0 + k * THREADS * 16);
    }
}

// A row's partial sums: its output channels (D), maximum and sum behind all.
struct Partial {
    float *o, *ml;
    __device__ Partial(const PagedProblem &pr, const PagedGrid &gr, int64_t row)
        : o(pr.work + gr.at + row * pr.D), ml(pr.work + gr.at + gr.rows * pr.D + row * 2) {}
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

// Rows of y behind the last sequence: zeros, by the workgroups behind the blocks.
template <typename T>
__device__ __forceinline__ void zero_rows(const PagedProblem &pr, int blocks) {
    if (blockIdx.y != 0 || blockIdx.z != 0) return;
    typedef uint32_t u4 __attribute__((ext_vector_type(4)));
    const int end = pr.offsets[pr.B];
    const int64_t per = (int64_t)pr.H * pr.D / (16 / (int)sizeof(T)), from = (int64_t)(end < 0 ? 0 : end) * per;
    const int64_t step = (int64_t)(gridDim.x - blocks) * blockDim.x;
    for (int64_t i = from + (int64_t)(blockIdx.x - blocks) * blockDim.x + threadIdx.x; i < pr.T * per; i += step)
        static_cast<u4 *>(pr.y)[i] = u4{};
}

// Whether one of the values that a block's tiles hold but hide from one of its rows,
// before its window or behind it, is not finite.
template <typename T>
__device__ __forceinline__ bool hidden_values(const PagedProblem &pr, const PagedKV<T> &kv, const RowSight &rs) {
    const int low = rs.blo - pr.W + 1;
    return bad_values(kv, low > 0 ? low : 0, rs.bhi - pr.W + 1, pr.D) || bad_values(kv, rs.blo + 1, rs.bhi + 1, pr.D);
}

// A row whose weights sum to zero is zero where it sees nothing; where all that it sees
// has the score -inf, its softmax is NaN.
__device__ __forceinline__ float without_weights(bool sees) { return sees ? NAN : 0.f; }

// A wavefront's 32 rows (lane: row r of the block's sequence): their outputs, or
// their partial sums.  Outputs that are not finite are formed again from the keys that
// the row sees alone, if a value that is not finite lies where they do not see it.
template <typename T, int DP, int R>
__device__ __forceinline__ void finish_rows(const PagedProblem &pr, const PagedGrid &gr, int id, const Block &w,
                                            const RowSight &rs, int r, int lane, const f16v (&o)[DP / 32], float m, float l) {
    const int hk = blockIdx.y;
    const int64_t head = (int64_t)hk * pr.D;
    if (gr.splits > 1) {
        if (r < w.rows)
            store_partial(o, Partial(pr, gr, (((int64_t)id * pr.Hk + hk) * gr.splits + blockIdx.z) * R + r - w.r0), m,
                          l, pr.D, lane);
        return;
    }
    const float inv = l == 0.f ? 0.f : 1.f / l;
    T *y = static_cast<T *>(pr.y) + w.q0 * pr.H * pr.D + head * pr.G;
    const bool bad = r < w.rows && store_channels(o, y + ((int64_t)rs.tok * pr.H + rs.g) * pr.D, pr.D, lane, inv);
    // NaN weights: the row is NaN, whatever it sees
    uint32_t again = rows_of(__ballot(bad && l > 0.f)), empty = rows_of(__ballot(r < w.rows && l == 0.f));
    const PagedKV<T> kv = paged_rows_of<T>(pr, w.b, head);
    if ((again | empty) != 0) __threadfence_block();  // other lanes' stores
    if (again != 0 && !hidden_values(pr, kv, rs)) again = 0;
    int asked = -1;
    bool sees = false;
    for (; empty; empty &= empty - 1) {
        const int j = __builtin_ctz(empty), at = __builtin_amdgcn_readlane(rs.at, j);
        if (at != asked) sees = sees_any(kv, at, pr.W, pr.S);  // heads of one token lie together
        asked = at;
        const float v = without_weights(sees);
        store_row(y + ((int64_t)__builtin_amdgcn_readlane(rs.tok, j) * pr.H + __builtin_amdgcn_readlane(rs.g, j)) * pr.D, lane,
                  pr.D, Pair{v, v});
    }
    for (; again; again &= again - 1) {
        const int j = __builtin_ctz(again);
        const int tj = __builtin_amdgcn_readlane(rs.tok, j), gj = __builtin_amdgcn_readlane(rs.g, j);
        forward_row(static_cast<const T *>(pr.q) + (w.q0 + tj) * pr.q_row + (head * pr.G + (int64_t)gj * pr.D),
                    y + ((int64_t)tj * pr.H + gj) * pr.D, (T *)nullptr, kv, __builtin_amdgcn_readlane(rs.at, j), pr.W, pr.S,
                    pr.D, pr.scale * kLog2e);
    }
}

template <typename T, int DP>
struct FewShape {
    static constexpr int NW = sizeof(T) == 4 && DP > 64 ? 2 : 4, TILE = 32 * Tile<T, DP>::ROW, LDS = NW * 4 * TILE;
};

// Block number id, by the first NW wavefronts of a workgroup.
template <typename T, int DP>
__device__ __forceinline__ void few_rows(const PagedProblem &pr, const PagedGrid &gr, int id, char *lds_mem) {
    typedef FewShape<T, DP> Sh;
    typedef Tile<T, DP> Tl;
    constexpr int NW = Sh::NW, OT = DP / 32;
    if (threadIdx.x >= 64 * NW) return;
    const Block w = find_block<32>(pr, gr.which, id);
    if (w.b < 0) return;
    const int lane = threadIdx.x & 63, wave = uniform(threadIdx.x >> 6), hk = blockIdx.y;
    const unsigned lds = lds_byte((const CIRCATT_LDS char *)lds_mem) + wave * 4 * Sh::TILE;
    const int r = w.r0 + (lane & 31);
    const RowSight rs = RowSight::of<32>(pr, w, r);
    const Sight see{pr.W, pr.S};
    const TileList<32> tiles(rs.blo, rs.bhi, pr.W, pr.S);
    const Pages<T> pg(pr, w, rs, hk);
    const int parts = gr.splits * NW, part = blockIdx.z * NW + wave;
    const int i0 = (int)((int64_t)tiles.count * part / parts), i1 = (int)((int64_t)tiles.count * (part + 1) / parts);
    Rows<T, DP> x;
    const T *qr = static_cast<const T *>(pr.q) + (w.q0 + rs.tok) * pr.q_row + ((int64_t)(hk * pr.G + rs.g) * pr.D);
    if (i0 < i1) {
        const unsigned row_at = Tl::row_lane(lane) + lds, col_at = Tl::col_lane(lane) + lds + Sh::TILE;
        const int lo = uniform(rs.at), hi = __builtin_amdgcn_readlane(rs.at, 31);
        const bool plain = lo >= 0 && hi >= lo;  // ascending: no row without sight
        auto fetch = [&](uint32_t row, int i) {
            const unsigned to = lds + ((i - i0) & 1) * 2 * Sh::TILE;
            fetch_paged<T, DP, 32, 64>(pg.k, row, pr.D, lane, to);
            fetch_paged<T, DP, 32, 64>(pg.v, row, pr.D, lane, to + Sh::TILE);
        };
        auto key = [&](int i) { return tiles.key(i < i1 ? i : i1 - 1) + (lane & 31); };
        // the rows of the tile in work, and the page numbers of the next one
        uint32_t now = pg.row(key(i0), pg.page(key(i0)));
        fetch(now, i0);
        x.start(qr, pr.D, lane);
        int raw = pg.page(key(i0 + 1));
        loads_here();
        for (int i = i0; i < i1; ++i) {
            dma_wait();
            const uint32_t next = pg.row(key(i + 1), raw);
            if (i + 1 < i1) fetch(next, i + 1);
            raw = pg.page(key(i + 2));
            const int k0 = tiles.key(i);
            const uint32_t there = (uint32_t)__ballot(now != Pages<T>::kNone);
            now = next;
            const unsigned to = ((i - i0) & 1) * 2 * Sh::TILE;
            f16v s[1];
            V8<T> p[2];
            x.scores(row_at + to, s);
            if (there != ~0u || !(plain && see.all(lo, hi, k0, 32))) {
                asm volatile("");
                hide_keys(s[0], see.bits(rs.at, k0) & there, lane);
            }
            x.raise(x.largest(s) * (pr.scale * kLog2e));
            x.weigh(s, p, pr.scale * kLog2e);
            x.template add<1>(col_at + to, p);
        }
    } else {
        x.start(qr, 0, lane);
    }
    // join the wavefronts' sums in LDS: each one's maximum and sum, then the outputs,
    // 32 channels at a time, in the order of the wavefronts
    float m = x.m, l = x.total();
    static_assert(NW * (64 + 16 * 64) * 4 <= Sh::LDS, "");
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
        const float mv = ml[v * 64 + (lane & 31)], lv = ml[v * 64 + 32 + (lane & 31)];
        ll += mv == -INFINITY ? lv : lv * __builtin_amdgcn_exp2f(mv - mm);
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
    if (wave == 0) finish_rows<T, DP, 32>(pr, gr, id, w, rs, r, lane, x.o, mm, ll);
}

template <typename T, int DP>
struct ChunkShape {
    static constexpr int NB = sizeof(T) == 2 ? 2 : 1, KT = 32 * NB, TILE = KT * Tile<T, DP>::ROW;
    // Float32 operands of wide heads take more than half the registers
    static constexpr int NG = sizeof(T) == 2 || DP <= 64 ? 2 : 1;
    static constexpr int LDS = NG * 4 * TILE;
};

template <typename T, int DP>
__device__ __forceinline__ void chunk_rows(const PagedProblem &pr, const PagedGrid &gr, int id, char *lds_mem) {
    typedef ChunkShape<T, DP> Sh;
    typedef Tile<T, DP> Tl;
    constexpr int KT = Sh::KT, NB = Sh::NB, NG = Sh::NG, OT = DP / 32;
    const Block w = find_block<128>(pr, gr.which, id);
    if (w.b < 0) return;
    const int lane = threadIdx.x & 63, wave = uniform(threadIdx.x >> 6) & 3, group = uniform(threadIdx.x >> 8);
    const int tid = threadIdx.x & 255, hk = blockIdx.y;
    const unsigned lds = lds_byte((const CIRCATT_LDS char *)lds_mem) + group * 4 * Sh::TILE;
    const int r0 = w.r0 + 32 * wave, r = r0 + (lane & 31);
    const RowSight rs = RowSight::of<128>(pr, w, r);
    const bool live = r0 < w.rows;
    const Sight see{pr.W, pr.S};
    const TileList<KT> tiles(rs.blo, rs.bhi, pr.W, pr.S);
    const Pages<T> pg(pr, w, rs, hk);
    const int parts = gr.splits * NG;
    auto bound = [&](int part) { return (int)((int64_t)tiles.count * part / parts); };
    const int part = blockIdx.z * NG + group, i0 = bound(part), i1 = bound(part + 1);
    int rounds = 0;  // of the longest group: they share their barriers
    for (int g = 0; g < NG; ++g) {
        const int n = bound(blockIdx.z * NG + g + 1) - bound(blockIdx.z * NG + g);
        rounds = n > rounds ? n : rounds;
    }
    const float c = pr.scale * kLog2e;
    Rows<T, DP> x;
    const T *qr = static_cast<const T *>(pr.q) + (w.q0 + rs.tok) * pr.q_row + ((int64_t)(hk * pr.G + rs.g) * pr.D);
    x.start(qr, i0 < i1 ? pr.D : 0, lane);
    if (rounds > 0) {
        const unsigned row_at = Tl::row_lane(lane) + lds, col_at = Tl::col_lane(lane) + lds + Sh::TILE;
        const int lo = uniform(rs.at), hi = __builtin_amdgcn_readlane(rs.at, 31);
        const bool plain = lo >= 0 && hi >= lo;
        auto key = [&](int i) { return tiles.key(i < i1 ? i : i1 > 0 ? i1 - 1 : 0) + (lane & (KT - 1)); };
        auto fetch = [&](uint32_t row, int i) {
            if (i >= i1) return;
            const unsigned to = lds + ((i - i0) & 1) * 2 * Sh::TILE;
            fetch_paged<T, DP, KT, 256>(pg.k, row, pr.D, tid, to);
            fetch_paged<T, DP, KT, 256>(pg.v, row, pr.D, tid, to + Sh::TILE);
        };
        uint32_t now = pg.row(key(i0), pg.page(key(i0)));
        fetch(now, i0);
        int raw = pg.page(key(i0 + 1));
        loads_here();
        // The two groups are half a round apart: one's score products run beside the
        // other's exponentials and value products.
        if (group == 1) __builtin_amdgcn_s_barrier();
        for (int i = i0; i < i0 + rounds; ++i) {
            dma_barrier();
            const uint32_t next = pg.row(key(i + 1), raw);
            fetch(next, i + 1);
            raw = pg.page(key(i + 2));
            const uint64_t there = __ballot(now != Pages<T>::kNone);
            now = next;
            const bool mine = live && i < i1;
            const int k0 = tiles.key(i);
            const unsigned to = ((i - i0) & 1) * 2 * Sh::TILE;
            constexpr uint64_t kFull = KT == 64 ? ~0ull : 0xffffffffull;
            f16v s[NB];
            V8<T> p[2 * NB];
            if (mine) x.scores(row_at + to, s);
            if (NG == 2) __builtin_amdgcn_s_barrier();
            if (!mine) continue;
            if ((there & kFull) != kFull || !(plain && see.all(lo, hi, k0, KT))) {
                asm volatile("");
#pragma unroll
                for (int m = 0; m < NB; ++m)
                    hide_keys(s[m], see.bits(rs.at, k0 + 32 * m) & (uint32_t)(there >> (32 * m)), lane);
            }
            x.raise(x.largest(s) * c);
            x.weigh(s, p, c);
            x.template add<NB>(col_at + to, p);
        }
        if (NG == 2 && group == 0) __builtin_amdgcn_s_barrier();
    }
    float m = x.m, l = x.total();
    if (NG == 2) {
        // the second group's sums through LDS
        static_assert(NG == 1 || 4 * (16 * OT + 2) * 64 * 4 <= Sh::LDS, "");
        CIRCATT_LDS float *buf = (CIRCATT_LDS float *)lds_mem + wave * (16 * OT + 2) * 64;
        __syncthreads();
        if (group == 1) {
#pragma unroll
            for (int t = 0; t < OT; ++t)
#pragma unroll
                for (int i = 0; i < 16; ++i) buf[(16 * t + i) * 64 + lane] = x.o[t][i];
            buf[16 * OT * 64 + lane] = m;
            buf[(16 * OT + 1) * 64 + lane] = l;
        }
        __syncthreads();
        if (group == 1) return;
        const float m1 = buf[16 * OT * 64 + lane], l1 = buf[(16 * OT + 1) * 64 + lane], mm = fmaxf(m, m1);
        const float f0 = m == -INFINITY ? 1.f : __builtin_amdgcn_exp2f(m - mm);
        const float f1 = m1 == -INFINITY ? 1.f : __builtin_amdgcn_exp2f(m1 - mm);
        l = l * f0 + l1 * f1;
        m = mm;
#pragma unroll
        for (int t = 0; t < OT; ++t)
#pragma unroll
            for (int i = 0; i < 16; ++i) x.o[t][i] = x.o[t][i] * f0 + buf[(16 * t + i) * 64 + lane] * f1;
    }
    if (live) finish_rows<T, DP, 128>(pr, gr, id, w, rs, r, lane, x.o, m, l);
}

// A call's blocks: those of 128 rows (which take longest) first, those of 32 behind
// them, and workgroups for the rows behind the last sequence.
template <typename T, int DP>
__global__ __launch_bounds__((64 * FewShape<T, DP>::NW), 1) void paged_few(PagedProblem pr, PagedGrid gr) {
    __shared__ __attribute__((aligned(1024))) char lds_mem[FewShape<T, DP>::LDS];
    if ((int)blockIdx.x >= gr.blocks) return zero_rows<T>(pr, gr.blocks);
    few_rows<T, DP>(pr, gr, blockIdx.x, lds_mem);
}
template <typename T, int DP>
__global__ __launch_bounds__((256 * ChunkShape<T, DP>::NG), 1) void paged_chunk(PagedProblem pr, PagedGrid chunk, PagedGrid few) {
    constexpr int LDS = FewShape<T, DP>::LDS > ChunkShape<T, DP>::LDS ? FewShape<T, DP>::LDS : ChunkShape<T, DP>::LDS;
    __shared__ __attribute__((aligned(1024))) char lds_mem[LDS];
    const int id = blockIdx.x, split = blockIdx.z;
    if (id < chunk.blocks) {
        if (split < chunk.splits) chunk_rows<T, DP>(pr, chunk, id, lds_mem);
    } else if (id < chunk.blocks + few.blocks) {
        if (split < few.splits) few_rows<T, DP>(pr, few, id - chunk.blocks, lds_mem);
    } else {
        zero_rows<T>(pr, chunk.blocks + few.blocks);
    }
}

// Adds up the partial sums of a block's rows in the order of the splits: half a
// wavefront a row, four channels a lane.
template <typename T, int R>
__global__ __launch_bounds__(256, 8) void paged_join(PagedProblem pr, PagedGrid gr) {
    const Block w = find_block<R>(pr, gr.which, blockIdx.x);
    if (w.b < 0) return;
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, hk = blockIdx.y, d = 4 * (lane & 31);
    const int64_t slot = ((int64_t)blockIdx.x * pr.Hk + hk) * gr.splits * R, head = (int64_t)hk * pr.D;
    const int rows = w.rows - w.r0 < R ? w.rows - w.r0 : R;
    int hidden = -1;  // hidden_values of the block, once asked for
    for (int i0 = 2 * wave; i0 < rows; i0 += 8) {
        const int i = i0 + (lane >> 5), ii = i < rows ? i : rows - 1;
        float m = -INFINITY, l = 0.f;
        for (int s = 0; s < gr.splits; ++s) m = fmaxf(m, Partial(pr, gr, slot + s * R + ii).ml[0]);
        f4v o = f4v{};
        for (int s = 0; s < gr.splits; ++s) {
            const Partial p(pr, gr, slot + s * R + ii);
            const float ls = p.ml[1];
            if (ls == 0.f) continue;  // saw nothing, and wrote no outputs
            const float f = __builtin_amdgcn_exp2f(p.ml[0] - m);
            l += ls * f;
            if (d < pr.D) o += *reinterpret_cast<const f4v *>(p.o + d) * f;
        }
        const float inv = l == 0.f ? 0.f : 1.f / l;
        const int tok = (w.r0 + ii) / pr.G, g = w.r0 + ii - tok * pr.G;
        T *y = static_cast<T *>(pr.y) + (w.q0 + tok) * pr.H * pr.D + head * pr.G + (int64_t)g * pr.D;
        V4<T> v;
        bool bad = false;
#pragma unroll
        for (int e = 0; e < 4; ++e) {
            v[e] = (T)(o[e] * inv);
            bad |= !(fabsf(o[e] * inv) < INFINITY);
        }
        if (i < rows && d < pr.D) *reinterpret_cast<V4<T> *>(y + d) = v;
        const bool in = i < rows && d < pr.D;
        const uint64_t empty = __ballot(l == 0.f && in);
        uint64_t again = __ballot(bad && l > 0.f && in);
        const PagedKV<T> kv = paged_rows_of<T>(pr, w.b, head);
        if ((again | empty) != 0) __threadfence_block();  // other lanes' stores
        if (again != 0) {
            if (hidden < 0) hidden = hidden_values(pr, kv, RowSight::of<R>(pr, w, w.r0));
            if (!hidden) again = 0;
        }
        for (int h = 0; h < 2; ++h) {
            const bool form = (uint32_t)(again >> (32 * h)) != 0, none = (uint32_t)(empty >> (32 * h)) != 0;
            if (!form && !none) continue;
            const int rj = w.r0 + i0 + h, tj = rj / pr.G, gj = rj - tj * pr.G;
            const int64_t held = (int64_t)pr.maxp << pr.page_log2;
            const int pos = w.first + tj, at = pos >= held ? -1 : pos;
            T *yj = static_cast<T *>(pr.y) + (w.q0 + tj) * pr.H * pr.D + head * pr.G + (int64_t)gj * pr.D;
            if (form) {
                forward_row(static_cast<const T *>(pr.q) + (w.q0 + tj) * pr.q_row + (head * pr.G + (int64_t)gj * pr.D), yj,
                            (T *)nullptr, kv, at, pr.W, pr.S, pr.D, pr.scale * kLog2e);
            } else {
                const float v = without_weights(sees_any(kv, at, pr.W, pr.S));
                store_row(yj, lane, pr.D, Pair{v, v});
            }
        }
    }
}

// The kernels of a call: blocks of 32 rows where a sequence has one token, or no more
// rows than that on average; else blocks of 128, and blocks of 32 for the sequences of a
// batch that have no more.
struct PagedPlan {
    bool few, chunk;
    PagedGrid few_grid, chunk_grid;
    int64_t floats;
};

// Splits: the estimate counts rounds of the chip's 256 compute units at a
// workgroup's rounds of tiles, three tiles' time for its start and end, and eight
// for another kernel that adds up.  blocks: about as many as will have rows.
int count_splits(double blocks, double tiles) {
    int best = 1;
    double least = 1e300;
    for (int p = 1; p <= 64 && p <= tiles; ++p) {
        const double rounds = (double)(int64_t)((blocks * p + 255) / 256);
        const double cost = rounds * (tiles / p + 3) + (p > 1 ? 8 : 0);
        if (cost < least) least = cost, best = p;
    }
    return best;
}

PagedPlan paged_plan(const PagedProblem &pr) {
    PagedPlan pl;
    const int64_t rows = pr.T * pr.G;
    pl.chunk = pr.T != pr.B && rows > (int64_t)pr.B * 32;
    pl.few = !pl.chunk || pr.B > 1;
    const bool wide = pr.dtype == CIRCATT_F32;
    const int64_t held = (int64_t)pr.maxp * pr.page, window = (int64_t)pr.W + pr.S;
    auto grid = [&](int R, int KT, int waves, int which) {
        PagedGrid gr;
        gr.which = which;
        gr.blocks = which == kShort ? pr.B : (int)(rows / R) + pr.B;
        const int64_t seen = window + R / pr.G < held ? window + R / pr.G : held;
        const double blocks = which == kLong ? (double)rows / R + 1 : gr.blocks;
        gr.splits = count_splits(blocks * pr.Hk, (double)((seen + KT - 1) / KT) / waves);
        gr.rows = gr.splits > 1 ? (int64_t)gr.blocks * pr.Hk * gr.splits * R : 0;
        return gr;
    };
    pl.few_grid = grid(32, 32, wide && pr.D > 64 ? 2 : 4, pl.chunk ? kShort : kAll);
    pl.chunk_grid = grid(128, wide ? 32 : 64, wide && pr.D > 64 ? 1 : 2, pl.few ? kLong : kAll);
    pl.few_grid.at = 0;
    pl.chunk_grid.at = pl.few ? (pl.few_grid.rows * (pr.D + 2) + 3) & ~(int64_t)3 : 0;
    pl.floats = pl.chunk ? pl.chunk_grid.at + pl.chunk_grid.rows * (pr.D + 2) : pl.few_grid.rows * (pr.D + 2);
    return pl;
}

template <typename T, int DP>
void launch(const PagedProblem &pr, hipStream_t s) {
    const PagedPlan pl = paged_plan(pr);
    const int tail = pr.zero_tail && pr.offsets != nullptr ? 8 : 0;
    if (pl.chunk) {
        PagedGrid few = pl.few_grid;
        if (!pl.few) few.blocks = 0, few.splits = 1;
        const PagedGrid &chunk = pl.chunk_grid;
        const int splits = chunk.splits > few.splits ? chunk.splits : few.splits;
        paged_chunk<T, DP><<<dim3(chunk.blocks + few.blocks + tail, pr.Hk, splits), 256 * ChunkShape<T, DP>::NG, 0, s>>>(
            pr, chunk, few);
        if (chunk.splits > 1) paged_join<T, 128><<<dim3(chunk.blocks, pr.Hk), 256, 0, s>>>(pr, chunk);
        if (few.splits > 1) paged_join<T, 32><<<dim3(few.blocks, pr.Hk), 256, 0, s>>>(pr, few);
    } else {
        const PagedGrid &gr = pl.few_grid;
        // without offsets the numbers of blocks end at the last sequence's
        const unsigned blocks = pr.offsets == nullptr ? pr.B * ((pr.G + 31) / 32) : gr.blocks;
        paged_few<T, DP><<<dim3(blocks + tail, pr.Hk, gr.splits), 64 * FewShape<T, DP>::NW, 0, s>>>(pr, gr);
        if (gr.splits > 1) paged_join<T, 32><<<dim3(blocks, pr.Hk), 256, 0, s>>>(pr, gr);
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

int64_t paged_workspace_floats(const PagedProblem &pr) { return paged_plan(pr).floats; }

int64_t paged_threads(const PagedProblem &pr) {
    const PagedPlan pl = paged_plan(pr);
    // and the workgroups for the rows behind the last sequence
    return 512 * ((int64_t)(pl.chunk ? pl.chunk_grid.blocks : 0) + pl.few_grid.blocks + 8);
}

hipError_t launch_paged(const PagedProblem &pr, hipStream_t s) {
    if (pr.dtype == CIRCATT_F32) launch<0>(pr, s);
    else if (pr.dtype == CIRCATT_F16) launch<2>(pr, s);
    else launch<3>(pr, s);
    return hipGetLastError();
}

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
