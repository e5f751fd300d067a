// paged_chunk.hip — attention of many 16-bit rows over pages of their type (paged_chunk.h).
#include "paged_chunk.h"

namespace aq {

int launch_paged_chunk(const AttnPagedArgs &a, int D, hipStream_t stream) { return chunk_pick<false>(a, D, stream); }

} // namespace aq
