// paged_few_f16.hip — attention of few rows over pages of type F16 (paged_few.h).
#include "paged_few.h"

namespace aq {

int launch_paged_few_f16(const AttnPagedArgs &a, int D, int R, hipStream_t stream) {
    if (a.q.type == AQ_TYPE_F32) return few_pick<AQ_TYPE_F16, true, false>(a, D, R, stream);
    return few_pick<AQ_TYPE_F16, false, false>(a, D, R, stream);
}

} // namespace aq
