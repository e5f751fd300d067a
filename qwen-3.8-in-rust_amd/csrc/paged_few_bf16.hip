// paged_few_bf16.hip — attention of few rows over pages of type BF16 (paged_few.h).
#include "paged_few.h"

namespace aq {

int launch_paged_few_bf16(const AttnPagedArgs &a, int D, int R, hipStream_t stream) {
    if (a.q.type == AQ_TYPE_F32) return few_pick<AQ_TYPE_BF16, true>(a, D, R, stream);
    return few_pick<AQ_TYPE_BF16, false>(a, D, R, stream);
}

} // namespace aq
