// Pieces of the MFMA kernels that walk 64-key tiles (prefill.hip, chunk.hip): the
// 32x32x16 product and its lane layouts, the tiles' swizzles and the global ->
// LDS copy.
#pragma once

#include "device.hpp"

namespace aoakv {

typedef _Float16 half8 __attribute__((ext_vector_type(8)));
typedef _Float16 half4 __attribute__((ext_vector_type(4)));
typedef float floatx16 __attribute__((ext_vector_type(16)));
typedef short short4v __attribute__((ext_vector_type(4)));
typedef __attribute__((address_space(3))) short4v lds_short4;
typedef __attribute__((address_space(3))) char lds_char;

constexpr int kPfTileKeys = 64;
constexpr float kLog2e = 1.4426950408889634f;

__device__ inline floatx16 mfma32(const half8& a, const half8& b, const floatx16& c) {
  return __builtin_amdgcn_mfma_f32_32x32x16_f16(a, b, c, 0, 0, 0);
}

// This lane's value and lane l^32's, combined: v_permlane32_swap exchanges
// the two halves of the wave in registers, where __shfl_xor would go through
// the LDS unit (ds_bpermute) and queue behind the tile reads.
__device__ inline float pair_max(float x) {
  const auto r = __builtin_amdgcn_permlane32_swap(__float_as_uint(x), __float_as_uint(x), false, false);
  return fmaxf(__uint_as_float(r[0]), __uint_as_float(r[1]));
}
__device__ inline float pair_sum(float x) {
  const auto r = __builtin_amdgcn_permlane32_swap(__float_as_uint(x), __float_as_uint(x), false, false);
  return __uint_as_float(r[0]) + __uint_as_float(r[1]);
}

// row of accumulator register i for lane group g
__device__ inline int crow(int i, int g) { return 8 * (i / 4) + 4 * g + (i % 4); }

// Chunk swizzles (16-byte chunk j of key row r sits at chunk j ^ swz(r));
// a row of D dims has CH = D / 8 chunks.  K is read as one chunk of 32
// consecutive rows per instruction: XOR with r % CH spreads them over all
// chunk positions.  V is read with the transpose read: a 16-lane group takes
// 2 adjacent chunks of 4 consecutive rows (the other group of the half-wave
// the next 2 chunks), so XOR with (CH / 4) * (r % 4) gives those chunks
// distinct positions (D = 128: 16 chunks, conflict-free as measured).
template <int CH>
__device__ inline int k_swz(int r) { return r & (CH - 1); }
template <int CH>
__device__ inline int v_swz(int r) { return (CH / 4) * (r & 3); }

// One 16-byte global -> LDS copy per lane (the lane lands at byte 16 * lane
// of `lds`).  A plain function: the builtin's operands inside the kernel
// template would be value-dependent, and the host pass then drops the
// kernel's launch stub.
__device__ inline void load_lds16(const f16* g, char* lds) {
  __builtin_amdgcn_global_load_lds(g, lds, 16, 0, 0);
}

// byte offset of 16-byte chunk j of key row r in a K tile of D-dim rows
template <int D>
__device__ inline int tile_off(int r, int j) { return r * (2 * D) + 16 * (j ^ k_swz<D / 8>(r)); }

// Tile geometry of a D-dim head (namespace-scope constants: the kernel's
// lambdas use them without capturing anything).
template <int D>
struct PfShape {
  static constexpr int kRowBytes = D * 2;                        // one key row
  static constexpr int kTileBytes = kPfTileKeys * kRowBytes;     // 16 KB at D = 128
  static constexpr int kCh = kRowBytes / 16;                     // 16-byte chunks per row
  static constexpr int kRPI = 1024 / kRowBytes;                  // rows per load instruction
  static constexpr int kKS = D / 16;                             // k-steps of the score MFMAs
  static constexpr int kDB = D / 32;                             // dim blocks of O
};

// Running max before a query's first visible key: below every score, and
// finite, so a tile (or a whole chunk) with no visible key leaves
// probabilities of 2^-inf = 0 and no inf - inf.
constexpr float kPfNoMax = -1e30f;

}  // namespace aoakv
