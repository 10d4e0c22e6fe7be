// Token attention with capped scores (sliding_impl.h), called from shaped.hip.
#include "sliding_impl.h"

namespace circatt {

hipError_t launch_capped_fwd(const ShapedSlidingProblem &pr, hipStream_t s) { return forward_of<Shaped<true>>(pr, s); }
hipError_t launch_capped_bwd(const ShapedSlidingProblem &pr, hipStream_t s) {
    return backward_of<Shaped<true>>(pr, walk_split(pr, masked_by(pr.shape)), s);
}

}  // namespace circatt
