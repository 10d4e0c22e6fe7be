// Rotary positions with several axes: pair (a, b) of a head is turned by
// position * base^(-i/p) of its axis, (a cos - b sin, a sin + b cos); the
// gradient is the turn the other way.
//
// A workgroup forms the cosines and sines of its tokens once, in LDS, and
// every head of a token reads them: the angle is formed in turns in 64 bits
// (positions up to 2^31 keep it to 2^-24 of a turn) and reduced to half a
// turn, which the hardware's sine and cosine, whose argument is in turns, take
// to 1.2e-7.  Then it streams its tokens once through 16-byte units: bound by
// memory.  4 x 256 x 256 pixels of 64 Float32 channels 26 us, 5.1 TB/s; 80 x 45 x
// 16 video tokens of 16 heads of 128, bf16, whose sections end within units, 112
// us with the call, 4.2 TB/s (by single channels 310).
#include "token_kernels.h"

namespace circatt {
namespace {

template <typename T, int V>
struct alignas(sizeof(T) * V == 16 ? 16 : sizeof(T)) Vec {
    T e[V];
};

// The (nt, npairs) cosines and sines of tokens t0 .. t0 + nt of image img.
__device__ __forceinline__ void form_angles(const RotaryProblem &pr, float2 *table, int64_t img, int64_t t0, int nt,
                                            FastDiv d1, FastDiv d2, FastDiv dpairs) {
    for (int e = threadIdx.x; e < nt * pr.npairs; e += 256) {
        const int t = fdiv(e, dpairs), i = e - t * pr.npairs;
        const int axis = i < pr.pairs[0] ? 0 : i < pr.pairs[0] + pr.pairs[1] ? 1 : 2;
        int at;
        if (pr.positions != nullptr) {
            at = pr.positions[img * pr.pos_batch + (t0 + t) * pr.naxes + axis];
        } else {
            const int p = (int)(t0 + t), r = fdiv(p, d1), s = fdiv(r, d2);
            at = axis == 0 ? p - r * pr.n1 : axis == 1 ? r - s * pr.n2 : s;
        }
        const double turns = (double)at * pr.turns[i];
        const float f = (float)(turns - __builtin_rint(turns)), sn = __builtin_amdgcn_sinf(f);
        table[e] = make_float2(__builtin_amdgcn_cosf(f), pr.inverse ? -sn : sn);
    }
}

// The section of channel c of a head: its first channel and pair, and its pairs
// (0: the channel stays).  Sections of 2 p channels follow axis by axis.
struct Section {
    int at, pair, p;
    __device__ __forceinline__ Section(const RotaryProblem &pr, int c) : at(0), pair(0), p(0) {
        for (int a = 0; a < pr.naxes; ++a) {
            p = pr.pairs[a];
            if (c < at + 2 * p) return;
            at += 2 * p;
            pair += p;
        }
        p = 0;
    }
};

// Heads of 16-byte units whose sections may end within one: TB tokens
// go to LDS, and every channel reads its partner and its angle there, at places
// that a thread, which has the same unit of a head for every token and head,
// knows from the start.
template <typename T>
__global__ __launch_bounds__(256) void rotary_any_kernel(RotaryProblem pr, int TB, FastDiv d1, FastDiv d2, FastDiv dheads,
                                                         FastDiv dpairs) {
    constexpr int V = 16 / sizeof(T);
    typedef uint32_t u4 __attribute__((ext_vector_type(4)));
    extern __shared__ char mem[];
    const int row = pr.H * pr.D, uph = pr.D / V, upt = pr.H * uph;
    T *xs = reinterpret_cast<T *>(mem);                            // (TB, row)
    float2 *table = reinterpret_cast<float2 *>(xs + TB * row);     // (TB, npairs)
    const int64_t blocks = (pr.P + TB - 1) / TB;
    const int64_t img = blockIdx.x / blocks, t0 = (blockIdx.x - img * blocks) * TB;
    const int nt = pr.P - t0 < TB ? (int)(pr.P - t0) : TB;
    const T *x = static_cast<const T *>(pr.x) + (img * pr.P + t0) * pr.x_row;
    T *y = static_cast<T *>(pr.y) + (img * pr.P + t0) * (int64_t)row;
    // whole heads: the threads behind the last one are idle
    const int step = 256 / uph, h0 = threadIdx.x / uph, u = threadIdx.x - h0 * uph;
    if (h0 < step)
        for (int n = h0; n < nt * pr.H; n += step) {
            const int t = fdiv(n, dheads);
            reinterpret_cast<u4 *>(xs)[n * uph + u] =
                reinterpret_cast<const u4 *>(x + t * pr.x_row)[(n - t * pr.H) * uph + u];
        }
    form_angles(pr, table, img, t0, nt, d1, d2, dpairs);
    __syncthreads();
    if (h0 >= step) return;
    int partner[V], pair[V];
    bool second[V];
    for (int e = 0; e < V; ++e) {
        const int c = u * V + e;
        const Section sec(pr, c);
        const int k = c - sec.at;
        second[e] = sec.p > 0 && (pr.interleaved ? k & 1 : k >= sec.p);
        partner[e] = sec.p == 0 ? 0 : pr.interleaved ? (k & 1 ? -1 : 1) : k < sec.p ? sec.p : -sec.p;
        pair[e] = sec.p == 0 ? -1 : sec.pair + (pr.interleaved ? k / 2 : k < sec.p ? k : k - sec.p);
    }
    for (int n = h0; n < nt * pr.H; n += step) {
        const int t = fdiv(n, dheads);
        const T *xr = xs + n * pr.D + u * V;
        const float2 *cs = table + t * pr.npairs;
        union {
            u4 u;
            T e[V];
        } v;
        v.u = *reinterpret_cast<const u4 *>(xr);
#pragma unroll
        for (int e = 0; e < V; ++e) {
            if (pair[e] < 0) continue;
            const float2 w = cs[pair[e]];
            const float m = (float)xr[e + partner[e]] * w.y;
            v.e[e] = (T)fmaf((float)v.e[e], w.x, second[e] ? m : -m);
        }
        reinterpret_cast<u4 *>(y)[n * uph + u] = v.u;
    }
}

// TB tokens a workgroup; V channels a unit (V divides D, every section and
// every row); a thread turns the unit that holds a pair's first member, and the
// unit of its second where the two lie apart.
template <typename T, int V, bool INTERLEAVED>
__global__ __launch_bounds__(256) void rotary_kernel(RotaryProblem pr, int TB, FastDiv d1, FastDiv d2, FastDiv dtoken,
                                                     FastDiv dunits, FastDiv dpairs) {
    extern __shared__ float2 table[];  // (TB, npairs): cos, sin
    const int64_t blocks = (pr.P + TB - 1) / TB;
    const int64_t img = blockIdx.x / blocks, t0 = (blockIdx.x - img * blocks) * TB;
    const int nt = pr.P - t0 < TB ? (int)(pr.P - t0) : TB;
    form_angles(pr, table, img, t0, nt, d1, d2, dpairs);
    __syncthreads();
    const T *x = static_cast<const T *>(pr.x) + (img * pr.P + t0) * pr.x_row;
    T *y = static_cast<T *>(pr.y) + (img * pr.P + t0) * ((int64_t)pr.H * pr.D);
    const int upt = pr.H * pr.D / V, uph = pr.D / V;
    typedef Vec<T, V> U;
    for (int n = threadIdx.x; n < nt * upt; n += 256) {
        const int t = fdiv(n, dtoken), u = n - t * upt;
        const float2 *cs = table + t * pr.npairs;
        const int c = (u - fdiv(u, dunits) * uph) * V;  // channel in the head
        const U *xp = reinterpret_cast<const U *>(x + t * pr.x_row) + u;
        U *yp = reinterpret_cast<U *>(y) + n;
        const Section sec(pr, c);
        const int p = sec.p;
        if (p == 0) {
            *yp = *xp;
        } else if (INTERLEAVED) {
            U v = *xp;
            const int i = sec.pair + (c - sec.at) / 2;
            for (int e = 0; e < V / 2; ++e) {
                const float2 w = cs[i + e];
                const float a = (float)v.e[2 * e], b = (float)v.e[2 * e + 1];
                v.e[2 * e] = (T)fmaf(a, w.x, -(b * w.y));
                v.e[2 * e + 1] = (T)fmaf(b, w.x, a * w.y);
            }
            *yp = v;
        } else if (c < sec.at + p) {
            const int i = sec.pair + c - sec.at, far = p / V;
            U va = *xp, vb = xp[far];
            for (int e = 0; e < V; ++e) {
                const float2 w = cs[i + e];
                const float a = (float)va.e[e], b = (float)vb.e[e];
                va.e[e] = (T)fmaf(a, w.x, -(b * w.y));
                vb.e[e] = (T)fmaf(b, w.x, a * w.y);
            }
            *yp = va;
            yp[far] = vb;
        }
    }
}

// Units of 16 bytes where they divide the head, its sections, the token stride
// and both addresses; by way of LDS where they divide all but the sections; else
// single pairs (interleaved) or channels.
enum Route { kUnits, kAny, kPairs, kSingle };
struct Plan {
    Route route;
    int TB;  // tokens a workgroup: about 1024 units, four a thread, and at most 32 KiB of angles
    int64_t blocks;
};
Plan plan_of(const RotaryProblem &pr) {
    const int per = pr.interleaved ? 2 : 1, W = pr.dtype == CIRCATT_F32 ? 4 : 8, row = pr.H * pr.D;
    int sections = pr.D;
    for (int a = 0; a < pr.naxes; ++a) sections |= pr.pairs[a] * per;
    const uint64_t addr = reinterpret_cast<uint64_t>(pr.x) | reinterpret_cast<uint64_t>(pr.y);
    auto tokens = [&](int units) {
        const int most = 4096 / pr.npairs, some = (1024 + units - 1) / units;
        return some < most ? some : most;
    };
    Plan pl{pr.interleaved ? kPairs : kSingle, 0, 0};
    if (pr.D % W == 0 && pr.x_row % W == 0 && addr % 16 == 0) {
        pl.TB = tokens(row / W);
        if (sections % W == 0) pl.route = kUnits;
        else if (pr.D / W <= 256 && (int64_t)pl.TB * (row * (16 / W) + pr.npairs * 8) <= 64 * 1024) pl.route = kAny;
    }
    if (pl.route == kPairs || pl.route == kSingle) pl.TB = tokens(row / (pl.route == kPairs ? 2 : 1));
    pl.blocks = pr.nb * ((pr.P + pl.TB - 1) / pl.TB);
    return pl;
}

template <typename T, int V>
void launch(const RotaryProblem &pr, const Plan &pl, hipStream_t s) {
    const size_t lds = (size_t)pl.TB * pr.npairs * 8;
    const FastDiv d1 = make_fastdiv(pr.n1), d2 = make_fastdiv(pr.n2), dt = make_fastdiv(pr.H * pr.D / V),
                  du = make_fastdiv(pr.D / V), dp = make_fastdiv(pr.npairs);
    if (pr.interleaved)
        rotary_kernel<T, V, true><<<(unsigned)pl.blocks, 256, lds, s>>>(pr, pl.TB, d1, d2, dt, du, dp);
    else
        rotary_kernel<T, V, false><<<(unsigned)pl.blocks, 256, lds, s>>>(pr, pl.TB, d1, d2, dt, du, dp);
}

template <typename T>
void route(const RotaryProblem &pr, hipStream_t s) {
    const Plan pl = plan_of(pr);
    if (pl.route == kUnits) {
        launch<T, 16 / sizeof(T)>(pr, pl, s);
    } else if (pl.route == kAny) {
        const size_t lds = (size_t)pl.TB * (pr.H * pr.D * sizeof(T) + pr.npairs * 8);
        rotary_any_kernel<T><<<(unsigned)pl.blocks, 256, lds, s>>>(pr, pl.TB, make_fastdiv(pr.n1), make_fastdiv(pr.n2),
                                                                   make_fastdiv(pr.H), make_fastdiv(pr.npairs));
    } else if (pl.route == kPairs) {
        launch<T, 2>(pr, pl, s);
    } else {
        launch<T, 1>(pr, pl, s);
    }
}

}  // namespace

int64_t rotary_threads(const RotaryProblem &pr) { return 256 * plan_of(pr).blocks; }

hipError_t launch_rotary(const RotaryProblem &pr, hipStream_t s) {
    if (pr.dtype == CIRCATT_F32) route<float>(pr, s);
    else if (pr.dtype == CIRCATT_F16) route<_Float16>(pr, s);
    else route<__bf16>(pr, s);
    return hipGetLastError();
}

}  // namespace circatt
