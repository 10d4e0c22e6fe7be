// Tiles of keys and values in LDS, and the matrix-core forward of 32 rows of
// queries over one of them.
//
// Score tile, transposed: S' = K Q' (32 keys x 32 query rows, K the first
// operand).  In the 32x32 result lane l holds column l % 32, one query row, and
// the keys 8 (i / 4) + 4 (l / 32) + i % 4 in registers i = 0 .. 15: the softmax
// runs over registers, with one exchange between the two halves of the
// wavefront, and the probabilities are already the second operand of
// O' = V' P' (lane l: column l % 32, eight consecutive places along k), when
// the places of k are read in the same order of keys.  V' is the first operand
// of that product: lane l needs one channel of eight keys, which the
// transposing LDS read gives out of rows of channels (4 keys x 16 channels for
// 16 lanes).  Nothing crosses lanes between the two products.  Float32 operands
// take the same registers: place j of every lane is one 32x32x2 product.
//
// Rows lie in LDS as PC 16-byte units, the unit c of row r at c ^ f(r): 16 rows of
// one unit (the 16-byte reads) and four rows of four units (the transposing reads
// of 32 lanes) each fill the 64 banks once.  The tiles arrive by
// 16-byte LDS-DMA, whose lanes write consecutive units, so the permutation is
// applied to the addresses that they read.
#pragma once

#include "buffer_dma.h"
#include "token_rows.h"

namespace circatt {
namespace tok {

typedef float f16v __attribute__((ext_vector_type(16)));
typedef short s4v __attribute__((ext_vector_type(4)));
template <typename T>
using V4 = T __attribute__((ext_vector_type(4)));
#define CIRCATT_LDS __attribute__((address_space(3)))

__device__ __forceinline__ f16v mma(V8<__bf16> a, V8<__bf16> b, f16v c) {
    return __builtin_amdgcn_mfma_f32_32x32x16_bf16(a, b, c, 0, 0, 0);
}
__device__ __forceinline__ f16v mma(V8<_Float16> a, V8<_Float16> b, f16v c) {
    return __builtin_amdgcn_mfma_f32_32x32x16_f16(a, b, c, 0, 0, 0);
}
__device__ __forceinline__ f16v mma(V8<float> a, V8<float> b, f16v c) {
#pragma unroll
    for (int j = 0; j < 8; ++j) c = __builtin_amdgcn_mfma_f32_32x32x2f32(a[j], b[j], c, 0, 0, 0);
    return c;
}

// DP: channels of a head, padded to a multiple of 32 (zeros).
template <typename T, int DP>
struct Tile {
    static constexpr int UNITS = DP * (int)sizeof(T) / 16;  // read
    static constexpr int PC = UNITS <= 4 ? 4 : UNITS <= 8 ? 8 : UNITS <= 16 ? 16 : 32;
    static constexpr int ROW = PC * 16;  // bytes
    __device__ static __forceinline__ constexpr int f(int r) {
        return PC >= 16 ? ((r & 3) << 2) | ((r >> 2) & 3)
                        : PC == 8 ? ((r & 2) << 1) | ((r >> 2) & 3) : (r >> 2) & 3;
    }
    // LDS bytes are 32-bit numbers here: a lane's place in a tile, and every read
    // of it is that number with a few bits flipped (the unit's number) and a
    // constant added (rows): one register holds all of a lane's addresses.
    //
    // A lane's place for row(): row lane % 32, channels 8 (lane / 32) ..
    __device__ static __forceinline__ unsigned row_lane(int lane) {
        const int r = lane & 31, u = (lane >> 5) * (sizeof(T) == 2 ? 1 : 2);
        return r * ROW + ((u ^ f(r)) << 4);
    }
    // channels 16 k + 8 (lane / 32) .. + 7 of row m + lane % 32, m a multiple of 32
    __device__ static __forceinline__ V8<T> row(unsigned at, int m, int k) {
        if constexpr (sizeof(T) == 2) {
            return *(const CIRCATT_LDS V8<T> *)((at ^ (k << 5)) + m * ROW);
        } else {
            const f4v a = *(const CIRCATT_LDS f4v *)((at ^ (k << 6)) + m * ROW);
            const f4v b = *(const CIRCATT_LDS f4v *)((at ^ (k << 6 | 16)) + m * ROW);
            return V8<T>{a[0], a[1], a[2], a[3], b[0], b[1], b[2], b[3]};
        }
    }
    // A lane's place for col(); 16-bit: rows 4 (lane / 32) + lane % 16 / 4, four
    // channels of 16 (lane / 16 % 2) on; Float32: channel lane % 32.
    __device__ static __forceinline__ unsigned col_lane(int lane) {
        if constexpr (sizeof(T) == 2) {
            const int i = lane & 15, r = 4 * (lane >> 5) + (i >> 2), u = 2 * ((lane >> 4) & 1) + ((i & 3) >> 1);
            return r * ROW + ((u ^ f(r)) << 4) + ((i & 1) << 3);
        } else {
            const int r = 4 * (lane >> 5), d = lane & 31;
            return r * ROW + (((d >> 2) ^ f(r)) << 4) + ((d & 3) << 2);
        }
    }
    // channel 32 t + lane % 32 of the rows m + 8 (j / 4) + 4 (lane / 32) + j % 4,
    // j = 0 .. 7; m a multiple of 16.  f(x + y) = f(x) ^ f(y) for the disjoint bits
    // x = 4 (lane / 32) (and lane % 16 / 4), y = 8 (j / 4) (and j % 4).
    __device__ static __forceinline__ V8<T> col(unsigned at, int m, int t) {
        if constexpr (sizeof(T) == 2) {
            union {
                s4v s[2];
                V8<T> v;
            } u;
#pragma unroll
            for (int k = 0; k < 2; ++k)
                u.s[k] = __builtin_amdgcn_ds_read_tr16_b64_v4i16(
                    (CIRCATT_LDS s4v *)((at ^ (t << 6) ^ (f(8 * k) << 4)) + (m + 8 * k) * ROW));
            return u.v;
        } else {
            V8<T> v;
#pragma unroll
            for (int j = 0; j < 8; ++j) {
                const int r = 8 * (j >> 2) + (j & 3);
                v[j] = *(const CIRCATT_LDS float *)((at ^ (t << 7) ^ (f(r) << 4)) + (m + r) * ROW);
            }
            return v;
        }
    }
};

// waits for this wavefront's DMA and LDS reads, then for the workgroup
__device__ __forceinline__ void dma_barrier() {
    asm volatile("s_waitcnt vmcnt(0) lgkmcnt(0)\n\ts_barrier" ::: "memory");
}
__device__ __forceinline__ void dma_wait() { asm volatile("s_waitcnt vmcnt(0) lgkmcnt(0)" ::: "memory"); }
// All loads of this wavefront are here, said so that the compiler knows it too: a
// load that is first used inside a loop makes it wait there in every round, and for
// the DMA of the next tile with it.
__device__ __forceinline__ void loads_here() { __builtin_amdgcn_s_waitcnt(0x0f70); }
// 16 bytes from every lane's own address to LDS byte m0 + 16 lane
__device__ __forceinline__ void dma16_global(const void *p, unsigned m0) {
    asm volatile("s_nop 0\n\tglobal_load_lds_dwordx4 %0, off" : : "v"(p), "{m0}"(m0) : "memory");
}
__device__ __forceinline__ unsigned lds_byte(const CIRCATT_LDS char *p) { return (unsigned)(uintptr_t)p; }
__device__ __forceinline__ int uniform(int x) { return __builtin_amdgcn_readfirstlane(x); }

// the other half's value of the same query row
__device__ __forceinline__ float other_half(float x) {
    const auto r = __builtin_amdgcn_permlane32_swap(__builtin_bit_cast(unsigned, x), __builtin_bit_cast(unsigned, x),
                                                    false, false);
    return __builtin_bit_cast(float, (threadIdx.x & 32) ? r[0] : r[1]);
}

// N products whose first operands are read from LDS, read(i) AHEAD products before
// use(i, operand): a read takes several products' time to arrive, and the
// compiler's own order asks for most of them one product ahead.
template <typename T, int N, int AHEAD, typename Read, typename Use>
__device__ __forceinline__ void products(Read read, Use use) {
    if constexpr (sizeof(T) == 2) {
        V8<T> a[AHEAD];
#pragma unroll
        for (int i = 0; i < AHEAD && i < N; ++i) a[i] = read(i);
#pragma unroll
        for (int i = 0; i < N; ++i) {
            __builtin_amdgcn_sched_barrier(0x0006);  // arithmetic may pass
            use(i, a[i % AHEAD]);
            if (i + AHEAD < N) a[i % AHEAD] = read(i + AHEAD);
        }
        __builtin_amdgcn_sched_barrier(0x0006);
    } else {
#pragma unroll
        for (int i = 0; i < N; ++i) use(i, read(i));
    }
}

// Bits x of [lo, hi) among 0 .. 31.
__device__ __forceinline__ uint32_t bits_between(int lo, int hi) {
    const uint32_t below = hi <= 0 ? 0u : hi >= 32 ? ~0u : (1u << hi) - 1u;
    return lo <= 0 ? below : lo >= 32 ? 0u : below & (~0u << lo);
}
// The place of a 32x32 result's register i in a word of 32 places that is shifted
// down by 4 for the lanes of the second half.
__device__ __forceinline__ constexpr uint32_t place_bit(int i) { return 1u << (8 * (i >> 2) + (i & 3)); }

// What a query row sees: keys j with j <= at and j > at - W or j < S.
struct Sight {
    int W, S;
    __device__ __forceinline__ bool operator()(int at, int j) const {
        const int back = at - j;
        return back >= 0 && (back < W || j < S);
    }
    // of the keys k0 .. k0 + 31, a bit each
    __device__ __forceinline__ uint32_t bits(int at, int k0) const {
        const int end = at + 1 - k0, sinks = S - k0;
        return bits_between(end - W, end) | bits_between(0, end < sinks ? end : sinks);
    }
    // keys [k0, k0 + n): seen by none, or by all, of the rows at [lo, hi]
    __device__ __forceinline__ bool none(int lo, int hi, int k0, int n) const {
        return k0 > hi || (k0 + n - 1 <= lo - W && k0 >= S);
    }
    __device__ __forceinline__ bool all(int lo, int hi, int k0, int n) const {
        return k0 + n - 1 <= lo && (k0 > hi - W || k0 + n <= S);
    }
};

// The tiles of KT keys that rows at [lo, hi] see, in order: tiles of sinks, then
// of the window.
template <int KT>
struct TileList {
    int sinks, first, count;
    __device__ TileList(int lo, int hi, int W, int S) {
        const int w = lo - W + 1 > 0 ? (lo - W + 1) / KT : 0, s = (S + KT - 1) / KT;
        first = w;
        sinks = s < w ? s : w;
        count = hi < 0 ? 0 : sinks + hi / KT + 1 - w;
    }
    __device__ __forceinline__ int key(int i) const { return (i < sinks ? i : first + i - sinks) * KT; }
};

// A workgroup's tiles of KT keys in LDS, three places for K and two for V.  Round
// i forms the scores of tile i + 1 from its K tile while it adds the values of tile
// i; then V tile i + 1 and K tile i + 3 set out for the places that round i - 1
// left.
template <typename T, int DP>
struct Ring {
    typedef Tile<T, DP> Tl;
    // Float32 rows are twice as long: half the keys fill the same LDS
    static constexpr int NB = sizeof(T) == 2 ? 2 : 1, KT = 32 * NB;
    static constexpr int TILE = KT * Tl::ROW, BYTES = 5 * TILE, V = 3 * TILE;
    static constexpr int EACH = KT * Tl::PC / 256;  // a thread's DMA for one tile
    static_assert(EACH >= 1, "");
    // the workgroup's DMA but for the last tile's, or all of it, is done, and every
    // wavefront is past the round before
    __device__ static __forceinline__ void wait(bool but_one) {
        if (but_one) asm volatile("s_waitcnt vmcnt(%0) lgkmcnt(0)\n\ts_barrier" ::"i"(EACH) : "memory");
        else dma_barrier();
    }
};

// One tensor's n rows on the way into a ring: byte offsets of this thread's units
// of a tile, which are the same for every tile, and the buffer.  A tensor whose
// rows span less than 2 GiB is one buffer, and a tile an offset in it; else every
// tile is a buffer of its own.
template <typename T, int DP>
struct Feed {
    typedef Tile<T, DP> Tl;
    static constexpr int KT = Ring<T, DP>::KT, EACH = Ring<T, DP>::EACH;
    const T *p;
    int64_t row;
    int n, rb, last;  // bytes from row to row, and of a row's channels
    bool one;
    dma::i4v all;
    int off[EACH];
    __device__ __forceinline__ Feed(const T *p, int64_t row, int n, int D) : p(p), row(row), n(n) {
        rb = (int)(row * (int)sizeof(T));
        last = D * (int)sizeof(T);
        const int64_t bytes = (int64_t)(n - 1) * rb + last;
        one = bytes + KT * (int64_t)rb < dma::kMaxBytes;
        all = dma::dma_rsrc(reinterpret_cast<const float *>(p), one ? (int)bytes : 0);
#pragma unroll
        for (int k = 0; k < EACH; ++k) {
            const int slot = threadIdx.x + k * 256, r = slot / Tl::PC, u = (slot % Tl::PC) ^ Tl::f(r);
            off[k] = u * 16 < last ? r * rb + u * 16 : dma::kOut;
        }
    }
    // rows [k0, k0 + KT), k0 < n, to LDS byte `to`; rows from n on are zeros
    __device__ __forceinline__ void fetch(int k0, unsigned to) const {
        const unsigned m0 = to + uniform(threadIdx.x >> 6) * 1024;
        if (__builtin_expect(one, 1)) {
#pragma unroll
            for (int k = 0; k < EACH; ++k) dma::dma16(all, m0 + k * 4096, off[k], k0 * rb);
        } else {
            const int64_t bytes = (int64_t)(n - 1 - k0) * rb + last;
            const dma::i4v rs = dma::dma_rsrc(reinterpret_cast<const float *>(p + k0 * row),
                                              (int)(bytes < dma::kMaxBytes ? bytes : dma::kMaxBytes));
#pragma unroll
            for (int k = 0; k < EACH; ++k) dma::dma16(rs, m0 + k * 4096, off[k], 0);
        }
    }
};

// Hides the keys of a 32x32 block of scores whose bits are not set.  (Callers keep
// the branch to it, as few tiles need it, by an empty asm before.)
__device__ __forceinline__ void hide_keys(f16v &s, uint32_t seen, int lane) {
    const uint32_t half = seen >> (4 * (lane >> 5));
#pragma unroll
    for (int i = 0; i < 16; ++i)
        if (!(half & place_bit(i))) s[i] = -INFINITY;
}

// c + a + b by one instruction.
__device__ __forceinline__ float add_pair(__bf16 a, __bf16 b, float c) {
    typedef __bf16 Pair __attribute__((ext_vector_type(2)));
    return __builtin_amdgcn_fdot2_f32_bf16(Pair{a, b}, Pair{1.f, 1.f}, c, false);
}
__device__ __forceinline__ float add_pair(_Float16 a, _Float16 b, float c) {
    typedef _Float16 Pair __attribute__((ext_vector_type(2)));
    return __builtin_amdgcn_fdot2(Pair{a, b}, Pair{1.f, 1.f}, c, false);
}

// Running softmax and output of 32 rows (lane l and l + 32: row l % 32).
// Scores count in units of log2(e) scale; the row's maximum is raised only when
// a score passes it by more than 2^6 in the exponent, so that most tiles leave
// the output as it is: probabilities stay below 2^6, which Float32 sums and
// either 16-bit type hold with their full relative precision.
template <typename T, int DP>
struct Rows {
    static constexpr int STEPS = DP / 16, OT = DP / 32;
    static constexpr float RAISE = 6.f;
    V8<T> q[STEPS];
    f16v o[OT];
    float m, l;  // l: this lane's keys alone
    float rounded;

    __device__ __forceinline__ void start(const T *qrow, int D, int lane) {
#pragma unroll
        for (int s = 0; s < STEPS; ++s) q[s] = load8(qrow, 16 * s + 8 * (lane >> 5), D);
#pragma unroll
        for (int t = 0; t < OT; ++t) o[t] = f16v{};
        m = -INFINITY;
        l = rounded = 0.f;
    }

    // A round of NB blocks of 32 keys, in steps.
    template <int NB>
    __device__ __forceinline__ void scores(unsigned kt, f16v (&s)[NB]) const {
#pragma unroll
        for (int n = 0; n < NB; ++n) s[n] = f16v{};
#pragma unroll
        for (int k = 0; k < STEPS; ++k)
#pragma unroll
            for (int n = 0; n < NB; ++n) s[n] = mma(Tile<T, DP>::row(kt, 32 * n, k), q[k], s[n]);
    }
    // the row's largest score, over both halves
    template <int NB>
    __device__ __forceinline__ static float largest(const f16v (&s)[NB]) {
        float mx = s[0][0];
#pragma unroll
        for (int n = 0; n < NB; ++n)
#pragma unroll
            for (int i = 0; i < 16; ++i) mx = fmaxf(mx, s[n][i]);
        return fmaxf(mx, other_half(mx));
    }
    __device__ __forceinline__ void raise(float mx) {
        if (__any(mx > m + RAISE || (m == -INFINITY && mx > -INFINITY))) {
            const float mn = fmaxf(m, mx), r = m == -INFINITY ? 0.f : __builtin_amdgcn_exp2f(m - mn);
            l *= r;
            rounded *= r;
#pragma unroll
            for (int t = 0; t < OT; ++t)
#pragma unroll
                for (int i = 0; i < 16; ++i) o[t][i] *= r;
            m = mn;
        }
    }
    // KEPT: `rounded` sums the weights as they are rounded.  Where few keys carry a row,
    // most of that error cancels from an output divided by this sum.
    template <int NB, bool KEPT = false>
    __device__ __forceinline__ void weigh(const f16v (&s)[NB], V8<T> (&p)[2 * NB], float c) {
        const float mu = m == -INFINITY ? 0.f : m;
        float sum = 0.f;
#pragma unroll
        for (int n = 0; n < NB; ++n)
#pragma unroll
            for (int i = 0; i < 16; ++i) {
                const float e = __builtin_amdgcn_exp2f(fmaf(s[n][i], c, -mu));
                sum += e;
                p[2 * n + (i >> 3)][i & 7] = (T)e;
            }
        l += sum;
        if constexpr (KEPT) {
#pragma unroll
            for (int i = 0; i < 8; i += 2)
#pragma unroll
                for (int n = 0; n < 2 * NB; ++n) rounded = add_pair(p[n][i], p[n][i + 1], rounded);
        }
    }
    // The same of exponents: scores from which the reference is taken off.
    template <int NB>
    __device__ __forceinline__ void weigh(const f16v (&s)[NB], V8<T> (&p)[2 * NB]) {
        float sum = 0.f;
#pragma unroll
        for (int n = 0; n < NB; ++n)
#pragma unroll
            for (int i = 0; i < 16; ++i) {
                const float e = __builtin_amdgcn_exp2f(s[n][i]);
                sum += e;
                p[2 * n + (i >> 3)][i & 7] = (T)e;
            }
        l += sum;
    }
    // (of those: `most` is the row's largest, and they are lowered too)
    template <int NB>
    __device__ __forceinline__ void raise(f16v (&s)[NB], float most) {
        if (__any(most > RAISE || (m == -INFINITY && most > -INFINITY))) {
            const float mu = reference(), mn = fmaxf(m, most + mu), r = m == -INFINITY ? 0.f : __builtin_amdgcn_exp2f(m - mn);
            l *= r;
#pragma unroll
            for (int t = 0; t < OT; ++t)
#pragma unroll
                for (int i = 0; i < 16; ++i) o[t][i] *= r;
            m = mn;
            lower(s, reference() - mu);
        }
    }
    // what exponents are lowered by; nothing until a row has seen something
    __device__ __forceinline__ float reference() const { return m == -INFINITY ? 0.f : m; }
    template <int NB>
    __device__ __forceinline__ static void lower(f16v (&s)[NB], float by) {
#pragma unroll
        for (int n = 0; n < NB; ++n)
#pragma unroll
            for (int i = 0; i < 16; ++i) s[n][i] -= by;
    }
    template <int NB>
    __device__ __forceinline__ void add(unsigned vt, const V8<T> (&p)[2 * NB]) {
#pragma unroll
        for (int n = 0; n < 2 * NB; ++n)
#pragma unroll
            for (int t = 0; t < OT; ++t) o[t] = mma(Tile<T, DP>::col(vt, 16 * n, t), p[n], o[t]);
    }

    // sums over both halves' keys
    __device__ __forceinline__ float total() const { return l + __shfl_xor(l, 32, 64); }
    __device__ __forceinline__ float total_rounded() const { return rounded + __shfl_xor(rounded, 32, 64); }
};

// The rows of a wavefront (bits: lanes, a row's two halves) as bits 0 .. 31.
__device__ __forceinline__ uint32_t rows_of(uint64_t bits) { return (uint32_t)(bits | bits >> 32); }

// A kernel's first argument read anew, for what follows a loop: its fields hold no
// scalar registers through the loop.
template <typename P>
__device__ __forceinline__ P argument_again() {
    typedef const __attribute__((address_space(4))) uint32_t *Words;
    Words p = (Words)__builtin_amdgcn_kernarg_segment_ptr();
    asm volatile("" : "+s"(p));
    struct {
        uint32_t w[sizeof(P) / 4];
    } c;
#pragma unroll
    for (int i = 0; i < (int)sizeof(P) / 4; ++i) c.w[i] = p[i];
    return __builtin_bit_cast(P, c);
}

// Rows that a workgroup forms again, by all of its WAVES wavefronts in turn, as they
// tend to lie together: `from`, which of four wavefronts with 32 rows each this one
// is (or -1), with its rows of two kinds, a bit each; `wave`, this one's turn.
// repair(row of the 128, first kind, second kind) is called by whole wavefronts.
// The list is LDS that nothing is read from any more, or with SYNC once all are here.
template <int WAVES, bool SYNC, typename Repair>
__device__ __forceinline__ void share_repairs(CIRCATT_LDS uint32_t *list, int from, int wave, uint32_t one, uint32_t two,
                                              Repair repair) {
    if ((one | two) != 0) __threadfence_block();  // other wavefronts read the rows
    if (SYNC) __syncthreads();
    if (from >= 0 && lane_again() == 0) {
        list[from] = one;
        list[4 + from] = two;
    }
    __syncthreads();
    int turn = 0;
#pragma unroll 1  // repair is long
    for (int w = 0; w < 4; ++w) {
        const uint32_t o = uniform(list[w]), t = uniform(list[4 + w]);
        for (uint32_t left = o | t; left; left &= left - 1, turn = turn + 1 == WAVES ? 0 : turn + 1) {
            const int i = __builtin_ctz(left);
            if (turn == wave) repair(32 * w + i, o >> i & 1, t >> i & 1);
        }
    }
}

// Writes a row's channels (one lane and its other half), times f, NaN for those below
// `least`; whether one of them is not finite (as Float32: one that the row's type cannot
// hold is itself).
template <typename T, int OT>
__device__ __forceinline__ bool store_channels(const f16v (&o)[OT], T *y, int D, int lane, float f, float least = 0.f) {
    bool bad = false;
#pragma unroll
    for (int t = 0; t < OT; ++t)
#pragma unroll
        for (int i = 0; i < 16; i += 4) {
            const int d = 32 * t + 2 * i + 4 * (lane >> 5);
            V4<T> v;
#pragma unroll
            for (int j = 0; j < 4; ++j) {
                const float x = fabsf(o[t][i + j]) < least ? NAN : o[t][i + j] * f;
                bad |= !(fabsf(x) < INFINITY) && d < D;
                v[j] = (T)x;
            }
            if (d < D) *reinterpret_cast<V4<T> *>(y + d) = v;
        }
    return bad;
}
// What the rounding of such a row took (0 where it is not finite); e: a factor that is
// more exact than f, that the rests take their row to, or f.
template <typename T, int OT>
__device__ __forceinline__ void store_rests(const f16v (&o)[OT], T *rest, int D, int lane, float f, float e) {
#pragma unroll
    for (int t = 0; t < OT; ++t)
#pragma unroll
        for (int i = 0; i < 16; i += 4) {
            const int d = 32 * t + 2 * i + 4 * (lane >> 5);
            V4<T> v;
#pragma unroll
            for (int j = 0; j < 4; ++j) v[j] = rounding_rest<T>(o[t][i + j] * f, o[t][i + j] * e);
            if (d < D) *reinterpret_cast<V4<T> *>(rest + d) = v;
        }
}
template <typename T>
__device__ __forceinline__ void zero_channels(T *y, int D, int lane) {
    for (int d = 4 * (lane >> 5); d < D; d += 8) *reinterpret_cast<V4<T> *>(y + d) = V4<T>{};
}

}  // namespace tok
}  // namespace circatt
