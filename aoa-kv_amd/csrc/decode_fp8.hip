// Decode attention over a paged cache of 8-bit codes (gfx950): one query token per
// sequence over every page, or over the pages that a selection lists.
//
//   o = softmax(q k^T / sqrt(D)) v,  k = code * 2^exp,  v likewise (fp8.hpp),
// products of fp16 operands, sums and softmax in fp32.
//
// A workgroup takes a chunk of the page list for all query heads of a kv head, so a
// code is read once.  Its waves take batches of kUnits x 16 tokens in turn, straight
// from memory to registers:
//   S = K Q^T   16 tokens x 16 columns (the group's heads; the rest are zeros): lane l
//               holds token l % 16 and reads 16 codes at dims 64 j + 16 (l / 16);
//   O = V^T P   D x 16: a lane's scores are those of tokens 4 (l / 16) .. + 3 for head l
//               % 16, which is the second product's operand as it stands; of V the lane
//               reads D / 16 neighbouring dims of these four tokens, so that fragment t
//               (dims D / 16 m + t of lane m) is a shuffle within its own registers.
// Neither operand passes through LDS.  Chunks are joined through the workspace by the
// last one to arrive.
//
// Bounds.  16 sequences of up to 16000 tokens, 8 kv heads of 4 query heads (314 MB): HBM,
// 68 us, 4.6 TB/s; what is missing to a large copy's 5.15 is the start and the join, which
// nothing overlaps with one workgroup per CU.  One sequence: latency.  1000 tokens of 8 kv
// heads take 8.2 us: 2.3 a launch, 0.65 lengths and page ids, 1.4 the batches, 0.8 storing
// the parts, 3.1 the joins.
#include "fp8.hpp"
#include "kernels.hpp"
#include "mfma_tile.hpp"
#include "topk.hpp"

namespace aoakv {
namespace {

typedef float floatx4 __attribute__((ext_vector_type(4)));

constexpr uint32_t kDeThreads = 512, kDeWaves = kDeThreads / kWave;
constexpr uint32_t kDeList = 512;  // pages whose ids are staged at a time
// Probabilities of the second product are held 2^7 times as large, and the running
// maximum moves where one would pass 2^8 (chunk_attn.hpp)
constexpr float kDeLift = 7.f;

// x of lanes l, l ^ 16, l ^ 32, l ^ 48 combined
template <class F>
__device__ inline float quarters(float x, F&& f) {
  const auto a = __builtin_amdgcn_permlane16_swap(__float_as_uint(x), __float_as_uint(x), false, false);
  x = f(__uint_as_float(a[0]), __uint_as_float(a[1]));
  const auto b = __builtin_amdgcn_permlane32_swap(__float_as_uint(x), __float_as_uint(x), false, false);
  return f(__uint_as_float(b[0]), __uint_as_float(b[1]));
}
__device__ inline float max2(float x, float y) { return fmaxf(x, y); }
__device__ inline float add2(float x, float y) { return x + y; }

// Chunk `chunk` of `per` pages of sequence b, whose table begins at `beg` and has `held`
// pages, the last of `last` tokens.
struct Place {
  uint32_t b, chunk, per, beg;
  int32_t held;
  uint32_t last;
};
__device__ inline Place place_of(const DecodeFp8Args& a, uint32_t b, uint32_t chunk, uint32_t per) {
  const uint32_t beg = (uint32_t)a.kv_indptr[b];
  return Place{b, chunk, per, beg, a.kv_indptr[b + 1u] - (int32_t)beg,
               (uint32_t)a.kv_last_page_len[b]};
}
// The item-th of a call over every page.  A sequence without a page has one.
//
// Up to a.split / 2 sequences: the pages of all are cut into chunks of as few pages (at
// least kGenChunkPages) as leaves a.split chunks per kv head, which are all at work at once.
// (Chunks of a fixed share of each sequence were some more than the GPU holds at once: 16
// sequences 78 us where this way took 65.)
// More sequences: chunks of an equal share of all pages, and the rest of each sequence as
// one more, so up to a.split + batch: some begin when the first end, and most of the GPU
// waits for these.  8000 tokens a sequence, us and TB/s, of 8 kv heads: 15 sequences 58,
// 4.2; 16 60, 4.4; 17 92, 3.0; 24 123, 3.2; 32 (a chunk each) 102, 5.1; 33 156, 3.5; 64 205,
// 5.1.  Of 32 kv heads: 4 sequences 54, 4.9; 5 86, 3.8; 8 103, 5.1; 9 155, 3.8.
__device__ inline Place find_chunk(const DecodeFp8Args& a, uint32_t item) {
  const uint32_t lane = __lane_id();
  auto of = [](uint32_t x, uint32_t j) {
    return (uint32_t)__builtin_amdgcn_readlane((int)x, (int)j);
  };
  if (a.batch <= (uint32_t)kWave) {  // a lane per sequence
    const uint32_t i = lane < a.batch ? lane : a.batch - 1u;
    const uint32_t beg = (uint32_t)a.kv_indptr[i];
    const int32_t held = a.kv_indptr[i + 1u] - (int32_t)beg;
    const uint32_t last = (uint32_t)a.kv_last_page_len[i];
    uint32_t P = held > 0 ? (uint32_t)held : 0u;
    if (P > a.max_pages) P = a.max_pages;
    if (lane >= a.batch) P = 0u;
    const uint32_t total = of(wave_incl_scan(P), kWave - 1u);
    // chunks of `per` pages; the smallest per that leaves few enough lies between total /
    // split and total / (split - batch), where there are not too many sequences for one
    uint32_t n = 0u;
    auto chunks = [&](uint32_t per) {
      n = lane < a.batch ? (P + per - 1u) / per : 0u;
      if (lane < a.batch && n == 0u) n = 1u;
      return of(wave_incl_scan(n), kWave - 1u);
    };
    uint32_t lo = total / a.split + 1u, hi = lo;
    if (a.split >= 2u * a.batch) {
      hi = total / (a.split - a.batch) + 1u;
      --lo;
    }
    if (lo < kGenChunkPages) lo = kGenChunkPages;
    while (lo < hi) {  // (uniform)
      const uint32_t mid = (lo + hi) / 2u;
      if (chunks(mid) <= a.split) hi = mid;
      else lo = mid + 1u;
    }
    chunks(lo);
    const uint32_t upto = wave_incl_scan(n);
    const uint64_t past = __builtin_amdgcn_ballot_w64(item < upto);
    if (past == 0u) return Place{0u, ~0u, lo, 0u, 0, 0u};
    const uint32_t j = (uint32_t)__builtin_ctzll(past);
    return Place{j, item - (of(upto, j) - of(n, j)), lo, of(beg, j), (int32_t)of((uint32_t)held, j),
                 of(last, j)};
  }
  // more: sequence b's items begin at floor(pages before it / per) + b, room for its chunks
  // (and one where it has no page) whatever the lengths; 64 sequences are tried at a time
  const uint32_t first = (uint32_t)a.kv_indptr[0];
  const uint32_t total = (uint32_t)a.kv_indptr[a.batch] - first;
  uint32_t per = total / a.split + 1u, lo = 0u, n = a.batch;
  if (per < kGenChunkPages) per = kGenChunkPages;
  for (;;) {
    const uint32_t stride = (n + kWave - 1u) / kWave;
    const bool in = lane * stride < n;
    const uint32_t i = lo + (in ? lane * stride : 0u);
    const uint32_t off = ((uint32_t)a.kv_indptr[i] - first) / per + i;
    const uint64_t le = __builtin_amdgcn_ballot_w64(in && off <= item);
    if (le == 0u) return Place{0u, ~0u, per, 0u, 0, 0u};  // malformed page table
    const uint32_t j = 63u - (uint32_t)__builtin_clzll(le);
    lo += j * stride;
    if (stride == 1u)
      return place_of(a, (uint32_t)__builtin_amdgcn_readfirstlane((int)lo), item - of(off, j), per);
    const uint32_t left = n - j * stride;
    n = left < stride ? left : stride;
  }
}

constexpr uint32_t kJoin = 8u;  // parts whose loads go out together

// two floats of a part (agent-coherent, as st_agent and ld_agent)
__device__ inline void st_pair(float* p, const float2& x) {
  __hip_atomic_store(reinterpret_cast<uint64_t*>(p), __builtin_bit_cast(uint64_t, x),
                     __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
}
__device__ inline float2 ld_pair(const float* p) {
  return __builtin_bit_cast(
      float2, __hip_atomic_load(reinterpret_cast<uint64_t*>(const_cast<float*>(p)),
                                __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT));
}

// Codes of a lane: 16 of K per load, D / 16 of V.
template <int D>
struct DeShape {
  static constexpr int kUnits = D == 256 ? 1 : 2;  // of 16 tokens per batch
  static constexpr int kKL = D / 64;               // 16-byte loads of K per unit
  static constexpr int kVW = D / 64;               // 32-bit words of V per token
  static constexpr int kFr = D / 16;               // fragments of V
  static constexpr int kHeads = 8;                 // of a group, at most
};

// What is staged of a page: its id, and K's exponent, V's, and its tokens in a word.
__device__ inline float k_scale(uint32_t w) { return exp_scale((int)(int8_t)w); }
__device__ inline float v_scale(uint32_t w) { return exp_scale((int)(int8_t)(w >> 8)); }
__device__ inline uint32_t tokens(uint32_t w) { return w >> 16; }

// RUN: tokens that lie in one page, from a multiple of RUN on: 16 (pages of 16 or 32), 4
// (of a multiple of 4) or 1.
template <int D, int RUN>
__global__ __launch_bounds__(kDeThreads, 2) void decode_fp8_kernel(DecodeFp8Args a) {
  using Sh = DeShape<D>;
  constexpr bool S16 = RUN == 16;
  constexpr int kVP = RUN == 1 ? 4 : 1;  // pages of a lane's four tokens
  constexpr int kU = Sh::kUnits;
  constexpr uint32_t kBatch = 16u * kU;
  constexpr uint32_t kStride = (uint32_t)D + 4u;  // partial: o[D], m, l, pad
  __shared__ uint32_t s_page[kDeList], s_word[kDeList];
  __shared__ __attribute__((aligned(16))) float s_o[kDeWaves][Sh::kHeads][D];
  __shared__ float s_ml[kDeWaves][Sh::kHeads][2];
  __shared__ uint32_t s_last;
  const uint32_t lane = __lane_id(), col = lane % 16u, quarter = lane / 16u;
  const uint32_t wave = __builtin_amdgcn_readfirstlane(threadIdx.x / kWave);
  const uint32_t S = a.S, G = a.Hq / a.Hkv;
  const bool quest = a.sel != nullptr && (a.flags & kFlagQuestKernel) != 0u;

  uint32_t hkv;
  Place at;
  if (a.sel == nullptr) {
    hkv = blockIdx.x;
    at = find_chunk(a, blockIdx.y + gridDim.y * blockIdx.z);
  } else {
    hkv = blockIdx.y;
    at = place_of(a, blockIdx.z, blockIdx.x, a.split);
  }
  // (of a selection the ids are fetched beside the page table)
  const int32_t* const row =
      a.sel != nullptr ? a.sel + ((size_t)at.b * a.Hkv + hkv) * a.sel_stride : nullptr;
  uint32_t early = 0u;
  if (row != nullptr && threadIdx.x < at.per && at.chunk * at.per + threadIdx.x < a.sel_stride)
    early = (uint32_t)row[at.chunk * at.per + threadIdx.x];
  if (at.chunk == ~0u) return;  // (uniform)
  const uint32_t b = at.b, per = at.per, pbeg = at.beg;
  const int32_t held = at.held;
  uint32_t P = held > 0 ? (uint32_t)held : 0u;
  const uint32_t last = at.last;  // tokens of the table's last page
  if (last == 0u || last > S) P = 0u;  // malformed page table
  uint32_t L = P != 0u ? (P - 1u) * S + last : 0u;
  if (P > a.max_pages) {
    if (at.chunk == 0u && threadIdx.x == 0u) flag_error(a.error, kErrTruncated);
    P = a.max_pages;
    L = P * S;
  }
  const size_t bh0 = (size_t)b * a.Hq + hkv * G;
  if (P == 0u) {  // nothing to attend
    if (at.chunk == 0u)
      for (uint32_t i = threadIdx.x; i < G * D; i += kDeThreads) a.o[bh0 * D + i] = (f16)0.f;
    return;
  }
  uint32_t npages = P;
  if (a.sel != nullptr) {
    const uint32_t budget = a.token_budgets ? (uint32_t)a.token_budgets[b] : a.token_budget;
    npages = num_selected_pages(L, budget, S, P, quest ? kFlagQuestKernel : 0u);
    const uint32_t most = a.sel_stride + (quest ? 1u : 0u);
    if (npages > most) npages = most;
  }
  if (npages > a.max_chunks * kGenChunkPages) {  // the workspace's chunks
    npages = a.max_chunks * kGenChunkPages;
    if (at.chunk == 0u && threadIdx.x == 0u) flag_error(a.error, kErrTruncated);
  }
  if ((uint64_t)at.chunk * per >= npages) return;  // uniform
  const uint32_t nsel = quest ? npages - 1u : npages;
  const int32_t* list = row != nullptr ? row : a.kv_indices + pbeg;
  const uint32_t last_page = (uint32_t)a.kv_indices[pbeg + (uint32_t)held - 1u];

  // q of head `col` of the group, the dims of K's loads
  half8 q[2 * Sh::kKL];
#pragma unroll
  for (int j = 0; j < 2 * Sh::kKL; ++j) {
    q[j] = half8{};
    if (col < G)
      q[j] = *reinterpret_cast<const half8*>(a.q + (bh0 + col) * D + 64 * (j / 2) + 16 * quarter +
                                             8 * (j % 2));
  }
  floatx4 o[Sh::kFr];
#pragma unroll
  for (int t = 0; t < Sh::kFr; ++t) o[t] = floatx4{};
  float m = kPfNoMax, l = 0.f;

  const uint32_t i0 = at.chunk * per, i1 = i0 + per < npages ? i0 + per : npages;
  const size_t head = (size_t)hkv * a.g.head;
  for (uint32_t ib = i0; ib < i1; ib += kDeList) {
    const uint32_t np = i1 - ib < kDeList ? i1 - ib : kDeList;
    if (ib != i0) __syncthreads();  // the ids before were read
    for (uint32_t i = threadIdx.x; i < np; i += kDeThreads) {
      const bool fetched = row != nullptr && ib == i0 && i == threadIdx.x && i < per;
      s_page[i] = ib + i >= nsel ? last_page : fetched ? early : (uint32_t)list[ib + i];
    }
    __syncthreads();
    const uint32_t T = np * S, nb = (T + kBatch - 1u) / kBatch;  // token slots, batches
    // slot t of the list (past the end: one of the last): entry and slot in its page
    auto entry = [&](uint32_t t, uint32_t& slot) {
      const uint32_t e = a.page_rcp != 0u ? (uint32_t)(((uint64_t)t * a.page_rcp) >> 32) : t;
      slot = t - e * S;
      return e;
    };
    auto unit = [&](uint32_t t) { return t < T ? t : T - 16u; };   // (S16)
    auto token = [&](uint32_t t) { return t < T ? t : T - 1u; };
    // batches in registers: one computed, one on its way
    u32x4 kr[2][kU][Sh::kKL];
    uint32_t vr[2][kU][4][Sh::kVW];
    auto load = [&](uint32_t i, int s) {
#pragma unroll
      for (int u = 0; u < kU; ++u) {
        const uint32_t t0 = i * kBatch + 16u * u;
        auto load_k = [&](uint32_t page, uint32_t slot) {
          const uint8_t* p = a.kv + (size_t)page * a.g.page + head + slot * a.g.tok + 16u * quarter;
#pragma unroll
          for (int j = 0; j < Sh::kKL; ++j)
            kr[s][u][j] = __builtin_nontemporal_load(reinterpret_cast<const u32x4*>(p + 64 * j));
        };
        auto load_v = [&](int r, uint32_t page, uint32_t slot) {
          typedef uint32_t words __attribute__((ext_vector_type(Sh::kVW)));
          const uint8_t* p = a.kv + (size_t)page * a.g.page + a.g.kv + head + slot * a.g.tok +
                             (D / 16) * col;
          const words x = __builtin_nontemporal_load(reinterpret_cast<const words*>(p));
#pragma unroll
          for (int w = 0; w < Sh::kVW; ++w) vr[s][u][r][w] = x[w];
        };
        uint32_t slot;
        if constexpr (S16) {
          const uint32_t e = entry(unit(t0), slot);
          const uint32_t page = (uint32_t)__builtin_amdgcn_readfirstlane((int)s_page[e]);
          load_k(page, slot + col);
#pragma unroll
          for (int r = 0; r < 4; ++r) load_v(r, page, slot + 4u * quarter + r);
        } else {
          uint32_t e = entry(token(t0 + col), slot), page = s_page[e];
          load_k(page, slot);
#pragma unroll
          for (int r = 0; r < 4; ++r) {
            if (r < kVP) {
              // (T is a multiple of 4 where RUN is)
              const uint32_t t = t0 + 4u * quarter + r;
              e = entry(t < T ? t : T - RUN, slot);
              page = s_page[e];
            }
            load_v(r, page, slot + (kVP == 1 ? r : 0u));
          }
        }
      }
    };
    auto attend = [&](uint32_t i, int b2) {
      // the words of K's token, and of the four tokens of the lane's scores and V
      uint32_t kw[kU], vw[kU][kVP];
      bool there[kU][4], whole = true;
#pragma unroll
      for (int u = 0; u < kU; ++u) {
        const uint32_t t0 = i * kBatch + 16u * u;
        uint32_t slot;
        if constexpr (S16) {
          const uint32_t e = entry(unit(t0), slot);
          kw[u] = vw[u][0] = (uint32_t)__builtin_amdgcn_readfirstlane((int)s_word[e]);
          const uint32_t n = t0 < T ? tokens(kw[u]) : 0u;
          whole &= slot + 16u <= n;
#pragma unroll
          for (int r = 0; r < 4; ++r) there[u][r] = slot + 4u * quarter + r < n;
        } else {
          kw[u] = s_word[entry(token(t0 + col), slot)];
#pragma unroll
          for (int r = 0; r < 4; ++r) {
            const uint32_t t = t0 + 4u * quarter + r;
            if (r < kVP) vw[u][r % kVP] = s_word[entry(t < T ? t : T - RUN, slot)];
            there[u][r] = t < T && slot + (kVP == 1 ? r : 0u) < tokens(vw[u][r % kVP]);
            whole &= there[u][r];
          }
        }
      }
      floatx4 s[kU];
#pragma unroll
      for (int u = 0; u < kU; ++u) {
        const float f = k_scale(kw[u]);
        s[u] = floatx4{};
#pragma unroll
        for (int j = 0; j < Sh::kKL; ++j) {
          const u32x4 x = kr[b2][u][j];
          s[u] = __builtin_amdgcn_mfma_f32_16x16x32_f16(
              __builtin_bit_cast(half8, decode8(uint2{x[0], x[1]}, f)), q[2 * j], s[u], 0, 0, 0);
          s[u] = __builtin_amdgcn_mfma_f32_16x16x32_f16(
              __builtin_bit_cast(half8, decode8(uint2{x[2], x[3]}, f)), q[2 * j + 1], s[u], 0, 0,
              0);
        }
      }
      if (__builtin_amdgcn_ballot_w64(!whole) != 0u) {
#pragma unroll
        for (int u = 0; u < kU; ++u)
#pragma unroll
          for (int r = 0; r < 4; ++r)
            if (!there[u][r]) {
              s[u][r] = -INFINITY;
#pragma unroll
              for (int w = 0; w < Sh::kVW; ++w) vr[b2][u][r][w] = 0u;  // (0 * NaN is NaN)
            }
      }
      float top = s[0][0];
#pragma unroll
      for (int u = 0; u < kU; ++u)
#pragma unroll
        for (int r = 0; r < 4; ++r) top = fmaxf(top, s[u][r]);
      top = quarters(top, max2);
      const bool up = (top - m) * a.scale > 8.f;
      const float next = up ? top : m;
      const float neg = __builtin_fmaf(-next, a.scale, kDeLift);
      if (__builtin_amdgcn_ballot_w64(up) != 0u) {
        // (between the offsets as exponentials have them: rounded apart from them, scores of
        // 2^18 scaled units weighed what was summed before 2^-5 wrong)
        const float keep = __builtin_amdgcn_exp2f(neg - __builtin_fmaf(-m, a.scale, kDeLift));
        l *= keep;
#pragma unroll
        for (int t = 0; t < Sh::kFr; ++t) o[t] *= keep;
      }
      m = next;
#pragma unroll
      for (int u = 0; u < kU; ++u) {
        half4 p;
#pragma unroll
        for (int r = 0; r < 4; ++r) {
          const float x = __builtin_amdgcn_exp2f(__builtin_fmaf(s[u][r], a.scale, neg));
          l += x;
          p[r] = (f16)x;  // (half a step, 2^-11; the sum has it unrounded)
        }
        // rows of 4 codes to values, then fragments: a dim of four tokens
#pragma unroll
        for (int w = 0; w < Sh::kVW; ++w) {
          half2v x[4][2];
#pragma unroll
          for (int r = 0; r < 4; ++r)
            decode4(vr[b2][u][r][w], v_scale(vw[u][r % kVP]), x[r]);
#pragma unroll
          for (int e = 0; e < 4; ++e) {
            const half4 f = {x[0][e / 2][e % 2], x[1][e / 2][e % 2], x[2][e / 2][e % 2],
                             x[3][e / 2][e % 2]};
            o[4 * w + e] = __builtin_amdgcn_mfma_f32_16x16x16f16(f, p, o[4 * w + e], 0, 0, 0);
          }
        }
      }
    };
    uint32_t i = wave;
    if (i < nb) load(i, 0);
    // (beside the first loads; they are needed no earlier)
    for (uint32_t j = threadIdx.x; j < np; j += kDeThreads) {
      const uint32_t page = s_page[j];
      const int8_t* e = a.kv_exp + (size_t)page * 2u * a.Hkv + hkv;
      s_word[j] = (uint32_t)(uint8_t)e[0] | (uint32_t)(uint8_t)e[a.Hkv] << 8 |
                  (page == last_page ? last : S) << 16;
    }
    __syncthreads();
    for (; i < nb; i += 2u * kDeWaves) {
      if (i + kDeWaves < nb) load(i + kDeWaves, 1);
      attend(i, 0);
      if (i + kDeWaves >= nb) break;
      if (i + 2u * kDeWaves < nb) load(i + 2u * kDeWaves, 0);
      attend(i + kDeWaves, 1);
    }
  }
  const uint32_t nch = (npages + per - 1u) / per;

  // ---- the workgroup's waves: o of lane (quarter, col) are dims D / 16 (4 quarter + r) + t
  l = quarters(l, add2);
  if (col < G) {
#pragma unroll
    for (int r = 0; r < 4; ++r)
#pragma unroll
      for (int t = 0; t < Sh::kFr; t += 4)
        *reinterpret_cast<float4*>(&s_o[wave][col][(D / 16) * (4 * quarter + r) + t]) =
            float4{o[t][r], o[t + 1][r], o[t + 2][r], o[t + 3][r]};
    if (quarter == 0u) {
      s_ml[wave][col][0] = -__builtin_fmaf(-m, a.scale, kDeLift);  // (the offset itself)
      s_ml[wave][col][1] = l;
    }
  }
  __syncthreads();
  float* const parts = a.partial + bh0 * a.max_chunks * kStride;  // [G][max_chunks][kStride]
  auto part = [&](uint32_t g, uint32_t c) { return parts + ((size_t)g * a.max_chunks + c) * kStride; };
  for (uint32_t x = 2u * threadIdx.x; x < G * D; x += 2u * kDeThreads) {  // (two dims a thread)
    const uint32_t g = x / D, d = x % D;
    float M = s_ml[0][g][0];
#pragma unroll
    for (uint32_t w = 1; w < kDeWaves; ++w) M = fmaxf(M, s_ml[w][g][0]);
    float2 acc = {0.f, 0.f};
    float sum = 0.f;
#pragma unroll
    for (uint32_t w = 0; w < kDeWaves; ++w) {
      const float f = __builtin_amdgcn_exp2f(s_ml[w][g][0] - M);
      acc.x += f * s_o[w][g][d];
      acc.y += f * s_o[w][g][d + 1u];
      sum += f * s_ml[w][g][1];
    }
    if (nch == 1u) {
      *reinterpret_cast<half2v*>(a.o + (bh0 + g) * D + d) = half2v{r16(acc.x / sum), r16(acc.y / sum)};
    } else {
      st_pair(part(g, at.chunk) + d, acc);
      if (d == 0u) st_pair(part(g, at.chunk) + D, float2{M, sum});
    }
  }
  if (nch == 1u) return;

  // ---- the chunks: joined by the last of each kJoin to arrive, and these by the last of all
  // (one workgroup for all chunks of a kv head took 50 of 60 us at 32768 tokens of 4 kv
  // heads with 8 query heads each)
  uint32_t* const counters = &a.counters[bh0 * kCounterStride];  // of all, then of each set
  uint32_t each = G <= 2u ? 2u * kJoin : kJoin;
  if (nch > each * (kCounterStride - 1u)) each = (nch + kCounterStride - 2u) / (kCounterStride - 1u);
  const uint32_t sets = (nch + each - 1u) / each, set = at.chunk / each;
  // joins n parts from chunk c0 on, `step` chunks apart: to the output, or to the first's place
  auto join = [&](uint32_t c0, uint32_t n, uint32_t step, bool out) {
    constexpr uint32_t kMost = 8 * D / (2 * kDeThreads) > 0 ? 8 * D / (2 * kDeThreads) : 1;
    float2 acc[kMost], ml[kMost];
#pragma unroll
    for (uint32_t y = 0; y < kMost; ++y) {
      const uint32_t x = 2u * (threadIdx.x + y * kDeThreads), g = x / D, d = x % D;
      if (x >= G * D) break;
      float2 s = {0.f, 0.f};
      float M = kPfNoMax, sum = 0.f;
      for (uint32_t i0 = 0; i0 < n; i0 += kJoin) {
        float2 pm[kJoin], po[kJoin];
#pragma unroll
        for (uint32_t u = 0; u < kJoin; ++u) {
          const float* p = part(g, c0 + (i0 + u < n ? i0 + u : n - 1u) * step);
          pm[u] = ld_pair(p + D);
          po[u] = ld_pair(p + d);
        }
        float next = M;
#pragma unroll
        for (uint32_t u = 0; u < kJoin; ++u) next = fmaxf(next, pm[u].x);
        const float keep = __builtin_amdgcn_exp2f(M - next);
        sum *= keep;
        s.x *= keep;
        s.y *= keep;
#pragma unroll
        for (uint32_t u = 0; u < kJoin; ++u) {
          const float f = i0 + u < n ? __builtin_amdgcn_exp2f(pm[u].x - next) : 0.f;
          sum += f * pm[u].y;
          s.x += f * po[u].x;
          s.y += f * po[u].y;
        }
        M = next;
      }
      acc[y] = s;
      ml[y] = float2{M, sum};
    }
    __syncthreads();  // every thread has read the parts
#pragma unroll
    for (uint32_t y = 0; y < kMost; ++y) {
      const uint32_t x = 2u * (threadIdx.x + y * kDeThreads), g = x / D, d = x % D;
      if (x >= G * D) break;
      if (out) {
        *reinterpret_cast<half2v*>(a.o + (bh0 + g) * D + d) =
            half2v{r16(acc[y].x / ml[y].y), r16(acc[y].y / ml[y].y)};
      } else {
        st_pair(part(g, c0) + d, acc[y]);
        if (d == 0u) st_pair(part(g, c0) + D, ml[y]);
      }
    }
  };
  // a workspace is left zeroed (after the arrival, which would wait for these stores)
  auto clear = [&](uint32_t c0, uint32_t n, uint32_t step) {
    for (uint32_t i = wave; i < G * n; i += kDeWaves)
      for (uint32_t j = 2u * lane; j < kStride; j += 2u * kWave)
        st_pair(part(i / n, c0 + i % n * step) + j, float2{0.f, 0.f});
  };
  const uint32_t c0 = set * each, in_set = nch - c0 < each ? nch - c0 : each;
  if (in_set > 1u && !arrive_last(&counters[1u + set], in_set, &s_last)) return;
  if (sets == 1u) {
    join(c0, in_set, 1u, true);
    clear(c0, in_set, 1u);
    return;
  }
  if (in_set > 1u) join(c0, in_set, 1u, false);
  const bool last_set = arrive_last(&counters[0], sets, &s_last);
  if (in_set > 1u) clear(c0 + 1u, in_set - 1u, 1u);
  if (!last_set) return;
  join(0u, sets, each, true);
  clear(0u, sets, each);
}

// One workgroup of 8 waves per CU, each with a batch on its way beside the one it computes
// (16 KB).  Graphs of calls on three caches in turn, us, two workgroups of 4 waves / one of
// 8 / two of 8 without a batch ahead: 2048 selected of 32768 tokens, 32 heads 10.2 / 9.3 /
// 9.3; every page of 16384 29 / 28 / 29; 32768 tokens of 4 kv heads of 8 query heads 25 / 18
// / 22; head dim 256 23 / 19 / 43; 16 sequences of 2000 to 16000 64 / 68 / 65.  Twice the
// workgroups: 28 -> 33 and 18 -> 28.  At head dim 64 a CU holds two; 512 / 256 of them, 16000
// tokens of 8 kv heads: 1 sequence 13.8 / 13.5, 4 22 / 20, 16 58 / 56, 17 68 / 89, 16 ragged
// ones 40 / 43; 2000 tokens of 32 heads 10.5 / 9.6.
constexpr uint32_t kDeWorkgroups = 256;
// Pages per chunk of a selection at least (of every page 8): with a call's two joins 16 are
// 8.5 us at 2048 tokens of 8 kv heads, 8 9.9; of 1000 tokens on every page 8.5, and 8.1.
// Chunks are of one length for all sequences, so just past a fill of the GPU the rest waits
// for a few: 4096 selected tokens of 8 kv heads, 16 sequences 35 us (3.8 TB/s), 17 55 (2.6),
// 32 61 (4.4), 33 93 (3.0).
constexpr uint32_t kDeListed = 16u;

}  // namespace

hipError_t launch_decode_fp8(const DecodeFp8Args& args, uint32_t head_dim, hipStream_t s) {
  DecodeFp8Args a = args;
  auto rcp = [](uint32_t d) { return d > 1u ? (uint32_t)((1ull << 32) / d) + 1u : 0u; };
  a.page_rcp = rcp(a.S);
  a.split = kDeWorkgroups / a.Hkv > 1u ? kDeWorkgroups / a.Hkv : 1u;
  if (a.sel != nullptr) {  // pages per chunk
    const uint64_t pages = (uint64_t)a.max_chunks * kGenChunkPages * a.Hkv * a.batch;
    a.split = (uint32_t)((pages + kDeWorkgroups - 1u) / kDeWorkgroups);
    if (a.split < kDeListed) a.split = kDeListed;
  }
  dim3 grid((a.max_chunks * kGenChunkPages + a.split - 1u) / a.split, a.Hkv, a.batch);
  if (a.sel == nullptr) {
    // (up to 64 sequences the items are counted, so no more than all chunks; else a sequence's
    // begin behind room for those before it)
    const uint64_t most = (uint64_t)a.max_chunks * a.batch;
    uint32_t items = a.split + a.batch;
    if (a.batch <= (uint32_t)kWave) {
      if (a.split >= 2u * a.batch) items = a.split;
      if (items > most) items = (uint32_t)most;
    }
    constexpr uint32_t kRows = 32768u;
    grid = dim3(a.Hkv, items < kRows ? items : kRows, (items + kRows - 1u) / kRows);
  }
  const dim3 block(kDeThreads);
#define AOAKV_DE(D_)                                                                              \
  if (a.S % 16u == 0u) hipLaunchKernelGGL((decode_fp8_kernel<D_, 16>), grid, block, 0, s, a);     \
  else if (a.S % 4u == 0u) hipLaunchKernelGGL((decode_fp8_kernel<D_, 4>), grid, block, 0, s, a);  \
  else hipLaunchKernelGGL((decode_fp8_kernel<D_, 1>), grid, block, 0, s, a)
  switch (head_dim) {
    case 64: AOAKV_DE(64); break;
    case 128: AOAKV_DE(128); break;
    default: AOAKV_DE(256); break;
  }
#undef AOAKV_DE
  return hipGetLastError();
}

}  // namespace aoakv
