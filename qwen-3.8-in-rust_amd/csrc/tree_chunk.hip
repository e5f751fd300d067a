// tree_chunk.hip — attention of trees of many 16-bit rows over pages of their type (paged_chunk.h).
#include "paged_chunk.h"

namespace aq {

int launch_tree_chunk(const AttnPagedArgs &a, int D, hipStream_t stream) { return chunk_pick<true>(a, D, stream); }

} // namespace aq
