// Token attention whose scores are biased by distance, or masked by documents or a
// prefix (sliding_impl.h); those that are capped as well are capped.hip's.
#include <cmath>

#include "sliding_impl.h"

namespace circatt {

hipError_t launch_capped_fwd(const ShapedSlidingProblem &pr, hipStream_t s);
hipError_t launch_capped_bwd(const ShapedSlidingProblem &pr, hipStream_t s);

namespace {

// What the keys' pass reads of every packed row and token: slopes times log2(e) and
// tokens as Float32 (exact up to 2^24 of them), and where a token's document ends: at
// the first later token whose own begins behind it.  (Starts ascend; whatever the
// places hold, an end lies behind its token and not behind the signal, and those behind
// its length are not looked at.)
__global__ __launch_bounds__(256) void shape_rows(ShapedSlidingProblem pr) {
    const int64_t i = (int64_t)blockIdx.x * 256 + threadIdx.x;
    const int64_t rows = (int64_t)pr.L * pr.G;
    if (pr.shape.slopes != nullptr) {
        if (i < rows) pr.row_tokens[i] = (float)(int)(i / pr.G);
        if (i < rows * pr.Hk) pr.row_slopes[i] = pr.shape.slopes[(int)(i / rows) * pr.G + (int)(i % pr.G)] * kLog2e;
    }
    if (pr.shape.places != nullptr && i < (int64_t)pr.B * pr.L) {
        const int b = (int)(i / pr.L), j = (int)(i - (int64_t)b * pr.L);
        const int32_t *places = pr.shape.places + b * pr.shape.places_row;
        const int n = signal_length(pr, b);
        int lo = j + 1, hi = n > j ? n : j + 1;  // the first t of (j, n) that begins behind j
        while (lo < hi) {
            const int t = (lo + hi) >> 1;
            if (document_start(places, t) > j) hi = t;
            else lo = t + 1;
        }
        pr.ends[i] = lo;
    }
}

struct ShapedRegions {
    int64_t slopes, tokens, ends, floats;
    ShapedRegions(const SlidingProblem &pr, const WalkSplit &sp, bool biased, bool documents) {
        auto up = [](int64_t n) { return (n + 3) & ~(int64_t)3; };
        const int64_t rows = (int64_t)pr.L * pr.G;
        slopes = up(bwd_floats(pr, sp));
        tokens = slopes + (biased ? up(rows * pr.Hk) : 0);
        ends = tokens + (biased ? up(rows) : 0);
        floats = ends + (documents ? up((int64_t)pr.B * pr.L) : 0);
    }
};

}  // namespace

// The series are the odd polynomials of degree 5 and 9 whose largest relative errors on
// [0, 0.3] and [0, 0.7] are least, 1.2e-6 and 3.0e-7 (found by linear programming over
// 4000 places): 3.4e-7 and 1.8e-7 of the cap.  x is worked into their coefficients; where
// Float32 does not hold one of those (scale / cap below some 1e-4 or above 1e4) they are
// not taken.  An error of 9e-5 of a score, 3.4e-7 of a cap of 256, is what 16-bit weights do
// not show; under larger caps the series end at scores that have it.
Curve make_curve(float cap, float scale, int dtype) {
    Curve c{};
    c.near = c.far = -1.f;
    if (!(cap > 0.f)) return c;
    constexpr double kFew[3] = {0.999998839, -0.333100214, 0.126339431};
    constexpr double kMore[5] = {0.999999697, -0.333302129, 0.132811127, -0.0508362388, 0.0137737143};
    const double x = (double)scale / cap;
    c.x = (float)x;
    c.u = (float)(2 * 1.4426950408889634 * x);
    c.C = (float)(1.4426950408889634 * cap);
    c.fine = dtype == CIRCATT_F32 || cap > 256.f;
    bool held = 0.49 / (x * x) <= 3e38;
    double power = x;
    for (int i = 0; i < 5; ++i, power *= x * x) {
        held &= std::fabs(kMore[i] * power) >= 1.2e-38 && std::fabs(power) <= 3e38;
        c.more[i] = (float)(kMore[i] * power);
        if (i < 3) c.few[i] = (float)(kFew[i] * power);
    }
    const double within = cap > 256.f ? 256.0 / cap : 1.0;
    if (held) c.near = (float)(0.3 * within / x), c.far = (float)(0.7 * within / x);
    return c;
}

int64_t shaped_bwd_workspace_floats(const SlidingProblem &pr, bool biased, int masked) {
    return ShapedRegions(pr, walk_split(pr, masked), biased, masked == kPlaces).floats;
}
int64_t shaped_sliding_threads(const SlidingProblem &pr, int masked, bool backward) {
    const int64_t n = threads_of(pr, walk_split(pr, masked), backward), rows = (int64_t)pr.L * pr.H + 256;
    return n > rows ? n : rows;
}
hipError_t launch_shaped_fwd(const ShapedSlidingProblem &pr, hipStream_t s) {
    return pr.shape.cap > 0.f ? launch_capped_fwd(pr, s) : forward_of<Shaped<false>>(pr, s);
}
hipError_t launch_shaped_bwd(ShapedSlidingProblem pr, hipStream_t s) {
    const bool biased = pr.shape.slopes != nullptr;
    const WalkSplit sp = walk_split(pr, masked_by(pr.shape));
    const ShapedRegions at(pr, sp, biased, pr.shape.places != nullptr);
    pr.row_slopes = pr.work + at.slopes;
    pr.row_tokens = pr.work + at.tokens;
    pr.ends = reinterpret_cast<int32_t *>(pr.work + at.ends);
    if (pr.dk != nullptr && (biased || pr.shape.places != nullptr)) {
        const int64_t rows = (int64_t)pr.L * pr.H, tokens = (int64_t)pr.B * pr.L, n = rows > tokens ? rows : tokens;
        shape_rows<<<(unsigned)((n + 255) / 256), 256, 0, s>>>(pr);
    }
    return pr.shape.cap > 0.f ? launch_capped_bwd(pr, s) : backward_of<Shaped<false>>(pr, sp, s);
}

}  // namespace circatt
