// Token attention with plain scores (sliding_impl.h).
#include "sliding_impl.h"

namespace circatt {

int64_t sliding_bwd_workspace_floats(const SlidingProblem &pr) { return bwd_floats(pr, walk_split(pr)); }
int64_t sliding_threads(const SlidingProblem &pr, bool backward) { return threads_of(pr, walk_split(pr), backward); }
hipError_t launch_sliding_fwd(const SlidingProblem &pr, hipStream_t s) { return forward_of<Plain>(pr, s); }
hipError_t launch_sliding_bwd(const SlidingProblem &pr, hipStream_t s) {
    return backward_of<Plain>(pr, walk_split(pr), s);
}

}  // namespace circatt
