// Token attention with capped scores (sliding_impl.h), called from shaped.hip.
#include "sliding_impl.h"

namespace circatt {

hipError_t launch_capped_fwd(const ShapedSlidingProblem &pr, hipStream_t s) { return forward_of<Shaped<true>>(pr, s); }
hipError_t launch_capped_bwd(const ShapedSlidingProblem &pr, hipStream_t s) {
    return backward_of<Shaped<true>>(pr, walk_split(pr, pr.shape.places != nullptr || pr.shape.prefix != nullptr), s);
}

}  // namespace circatt
