// Attention of requests that begin with the same pages, for gfx950: forks of one
// prompt (bc_shared_chunk_attention).
//
// No reference counterpart: the reference reads every request's pages by
// themselves (src/paged_gqa.cu).
#include "bc_tiles.h"

extern "C" size_t bc_shared_chunk_attention_workspace_size(bc_shape, int, int) { return 0; }

extern "C" int bc_shared_chunk_attention(bc_shape s, bc_chunk_inputs in, const int32_t* groups,
                                         const int32_t* shared, int group_count, void* workspace,
                                         size_t workspace_bytes, bc_stream_t stream) {
  if (!groups || group_count < 0 || (group_count > 0 && !shared) || group_count > s.batch)
    return BC_ERROR_INVALID_VALUE;
  return bc_chunk_attention(s, in, nullptr, 0, stream);
}
