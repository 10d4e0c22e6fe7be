// Rotary positions with several axes: pair (a, b) of a head is turned by
// position * base^(-i/p) of its axis, (a cos - b sin, a sin + b cos); the
// gradient is the turn the other way.
//
// A workgroup forms the cosines and sines of its tokens once, in LDS, and
// every head of a token reads them: the angle is formed in turns in 64 bits
// (positions up to 2^31 keep it to 2^-24 of a turn) and reduced to half a
// turn, which the hardware's sine and cosine, whose argument is in turns, take
// to 1.2e-7.  Then it streams its tokens once through 16-byte units.
#include "token_kernels.h"

namespace circatt {
namespace {

template <typename T, int V>
struct alignas(sizeof(T) * V == 16 ? 16 : sizeof(T)) Vec {
    T e[V];
};

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
        // the section of the channel: sections of 2 p channels, axis by axis
        int at = 0, pair = 0, p = 0;
        for (int a = 0; a < pr.naxes; ++a) {
            p = pr.pairs[a];
            if (c < at + 2 * p) break;
            at += 2 * p;
            pair += p;
            p = 0;
        }
        if (p == 0) {
            *yp = *xp;
        } else if (INTERLEAVED) {
            U v = *xp;
            const int i = pair + (c - at) / 2;
            for (int e = 0; e < V / 2; ++e) {
                const float2 w = cs[i + e];
                const float a = (float)v.e[2 * e], b = (float)v.e[2 * e + 1];
                v.e[2 * e] = (T)fmaf(a, w.x, -(b * w.y));
                v.e[2 * e + 1] = (T)fmaf(a, w.y, b * w.x);
            }
            *yp = v;
        } else if (c < at + p) {
            const int i = pair + c - at, far = p / V;
            U va = *xp, vb = xp[far];
            for (int e = 0; e < V; ++e) {
                const float2 w = cs[i + e];
                const float a = (float)va.e[e], b = (float)vb.e[e];
                va.e[e] = (T)fmaf(a, w.x, -(b * w.y));
                vb.e[e] = (T)fmaf(a, w.y, b * w.x);
            }
            *yp = va;
            yp[far] = vb;
        }
    }
}

template <typename T, int V>
void launch(const RotaryProblem &pr, hipStream_t s) {
    // about 1024 units, four a thread, and at most 32 KiB of angles
    const int upt = pr.H * pr.D / V, most = 4096 / pr.npairs;
    int TB = (1024 + upt - 1) / upt;
    TB = TB < most ? TB : most;
    const unsigned blocks = (unsigned)(pr.nb * ((pr.P + TB - 1) / TB));
    const size_t lds = (size_t)TB * pr.npairs * 8;
    const FastDiv d1 = make_fastdiv(pr.n1), d2 = make_fastdiv(pr.n2), dt = make_fastdiv(upt), du = make_fastdiv(pr.D / V),
                  dp = make_fastdiv(pr.npairs);
    if (pr.interleaved)
        rotary_kernel<T, V, true><<<blocks, 256, lds, s>>>(pr, TB, d1, d2, dt, du, dp);
    else
        rotary_kernel<T, V, false><<<blocks, 256, lds, s>>>(pr, TB, d1, d2, dt, du, dp);
}

// Units of 16 bytes, or of one pair (interleaved) or one channel, by what
// divides the head, its sections, the token stride and both addresses.
template <typename T>
void route(const RotaryProblem &pr, hipStream_t s) {
    const int per = pr.interleaved ? 2 : 1;
    int sections = pr.D;
    for (int a = 0; a < pr.naxes; ++a) sections |= pr.pairs[a] * per;
    auto fits = [&](int v) {
        const uint64_t addr = reinterpret_cast<uint64_t>(pr.x) | reinterpret_cast<uint64_t>(pr.y);
        return sections % v == 0 && pr.x_row % v == 0 && addr % (v * sizeof(T)) == 0;
    };
    constexpr int W = 16 / sizeof(T);
    if (fits(W)) launch<T, W>(pr, s);
    else if (pr.interleaved) launch<T, 2>(pr, s);
    else launch<T, 1>(pr, s);
}

}  // namespace

hipError_t launch_rotary(const RotaryProblem &pr, hipStream_t s) {
    if (pr.dtype == CIRCATT_F32) route<float>(pr, s);
    else if (pr.dtype == CIRCATT_F16) route<_Float16>(pr, s);
    else route<__bf16>(pr, s);
    return hipGetLastError();
}

}  // namespace circatt
