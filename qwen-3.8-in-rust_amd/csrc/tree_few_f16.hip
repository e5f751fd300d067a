// tree_few_f16.hip — attention of trees of few rows over pages of type F16 (paged_few.h).
#include "paged_few.h"

namespace aq {

int launch_tree_few_f16(const AttnPagedArgs &a, int D, int R, hipStream_t stream) {
    if (a.q.type == AQ_TYPE_F32) return few_pick<AQ_TYPE_F16, true, true>(a, D, R, stream);
    return few_pick<AQ_TYPE_F16, false, true>(a, D, R, stream);
}

} // namespace aq
