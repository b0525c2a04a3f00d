// Attention of a ragged batch of chunks over a paged cache of 8-bit codes (gfx950):
// chunk_attn.hpp with fragments made from codes.
#include "chunk_attn.hpp"

namespace aoakv {

hipError_t launch_chunk_attn_fp8(const ChunkArgs& a, uint32_t head_dim, hipStream_t s) {
  switch (head_dim) {
    case 64: return launch_attn<64, true>(a, s);
    case 128: return launch_attn<128, true>(a, s);
    default: return launch_attn<256, true>(a, s);
  }
}

}  // namespace aoakv
