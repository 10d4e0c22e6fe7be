// Attention over a paged cache with shaped scores (paged_impl.h).
#include "paged_impl.h"

namespace circatt {

hipError_t launch_shaped_paged(const ShapedPagedProblem &pr, hipStream_t s) {
    return pr.shape.cap > 0.f ? launch_of<Shaped<true>>(pr, s) : launch_of<Shaped<false>>(pr, s);
}

}  // namespace circatt
