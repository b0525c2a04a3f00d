// Attention of a ragged batch of chunks over a paged cache of 8-bit codes (gfx950):
// chunk_attn.hpp with fragments made from codes.
//
//   o = softmax(mod(q k^T / sqrt(D)) + mask) v,  k = code * 2^exp,  v likewise (fp8.hpp)
//
// Tiles of K and V are codes in LDS too: half the bytes on every way but the last, where
// one instruction makes two fp16 values of two codes and the power of two of their block,
// exactly.  K's lanes read 16 codes of a row, two fragments; V's go through the transposing
// read of 8-bit elements.  The four waves of a workgroup turn the same codes each for
// itself, 128 instructions per wave and tile at head dim 128 beside 32 matrix instructions:
// a prompt of 8192 tokens of 32 heads takes 616 to 632 us (890 TFLOP/s), 572 to 590 over
// fp16; with slopes 674 (fp16 619); 4096 tokens with a cap 228 (204), in pages of 12 232
// (181), 16 heads of 256 239 (220); 8192 tokens of 32 heads of 64 366 (345).
// 5 drafted tokens of 8 sequences over up to 16384, 8 kv heads (165 MB), take 53 us: of a
// workgroup's four waves one has rows, and its chain per tile bounds.  Tiles dealt to the
// four waves took as long (a buffer per wave: it waits out its own loads), four buffers
// filled three tiles ahead 55, and the prompt then 655.
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
