// Attention over a paged cache with shaped scores (paged_impl.h).
#include "paged_impl.h"

namespace circatt {

hipError_t launch_shaped_paged(const ShapedPagedProblem &pr, bool whole, hipStream_t s) {
    const PagedPlan pl = paged_plan(pr, whole);
    return pr.shape.cap > 0.f ? launch_of<Shaped<true>>(pr, pl, s) : launch_of<Shaped<false>>(pr, pl, s);
}

}  // namespace circatt
