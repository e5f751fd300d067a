// tree_few_f32.hip — attention of trees of few rows over pages of type F32 (paged_few.h).
#include "paged_few.h"

namespace aq {

int launch_tree_few_f32(const AttnPagedArgs &a, int D, int R, hipStream_t stream) {
    return few_pick<AQ_TYPE_F32, true, true>(a, D, R, stream);
}

} // namespace aq
