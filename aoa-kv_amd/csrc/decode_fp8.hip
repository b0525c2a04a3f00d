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
#include <type_traits>

#include "fp8.hpp"
#include "kernels.hpp"
#include "mfma_tile.hpp"

namespace aoakv {
namespace {

typedef float floatx4 __attribute__((ext_vector_type(4)));

constexpr uint32_t kDeThreads = 256, kDeWaves = kDeThreads / kWave;
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

// n / d, rounded up, for 1 <= n, rcp = floor(2^32 / d) + 1 (0: d = 1); from n * d = 2^32
// on it may be more
__device__ inline uint32_t div_up(uint32_t n, uint32_t rcp) {
  return rcp == 0u ? n : (uint32_t)(((uint64_t)(n - 1u) * rcp) >> 32) + 1u;
}

// Chunk `chunk` of `per` pages of sequence b.
struct Place {
  uint32_t b, chunk, per;
};
// The item-th of a call over every page: the pages of all sequences are cut into
// a.split chunks per kv head, at least kGenChunkPages pages each; sequence b's items
// begin at floor(pages before it / per) + b, room for its chunks, and for one where it
// has no page.
__device__ inline Place find_chunk(const DecodeFp8Args& a, uint32_t item) {
  const uint32_t first = (uint32_t)a.kv_indptr[0];
  const uint32_t total = (uint32_t)a.kv_indptr[a.batch] - first;
  uint32_t per = total != 0u ? div_up(total, a.split_rcp) : 1u;
  if (per < kGenChunkPages) per = kGenChunkPages;
  if (a.batch == 1u) return Place{0u, item, per};
  const uint32_t lane = __lane_id();
  uint32_t lo = 0u, n = a.batch;
  for (;;) {  // 64 sequences are tried at a time
    const uint32_t stride = (n + kWave - 1u) / kWave;
    const bool in = lane * stride < n;
    const uint32_t i = lo + (in ? lane * stride : 0u);
    const uint32_t off = ((uint32_t)a.kv_indptr[i] - first) / per + i;
    const uint64_t le = __builtin_amdgcn_ballot_w64(in && off <= item);
    if (le == 0u) return Place{0u, ~0u, per};  // malformed page table
    const uint32_t j = 63u - (uint32_t)__builtin_clzll(le);
    lo += j * stride;
    if (stride == 1u)
      return Place{(uint32_t)__builtin_amdgcn_readfirstlane((int)lo),
                   item - (uint32_t)__builtin_amdgcn_readlane((int)off, (int)j), per};
    const uint32_t left = n - j * stride;
    n = left < stride ? left : stride;
  }
}

// Codes of a lane: 16 of K per load, D / 16 of V.
template <int D>
struct DeShape {
  static constexpr int kUnits = D == 256 ? 2 : 4;  // of 16 tokens per batch
  static constexpr int kKL = D / 64;               // 16-byte loads of K per unit
  static constexpr int kVW = D / 64;               // 32-bit words of V per token
  static constexpr int kFr = D / 16;               // fragments of V
  static constexpr int kHeads = 8;                 // of a group, at most
};

// What is staged of a page: its id, and K's exponent, V's, and its tokens in a word.
__device__ inline float k_scale(uint32_t w) { return exp_scale((int)(int8_t)w); }
__device__ inline float v_scale(uint32_t w) { return exp_scale((int)(int8_t)(w >> 8)); }
__device__ inline uint32_t tokens(uint32_t w) { return w >> 16; }

// S16: pages are of 16 or 32 tokens, so that 16 tokens lie in one.
template <int D, bool S16>
__global__ __launch_bounds__(kDeThreads, 2) void decode_fp8_kernel(DecodeFp8Args a) {
  using Sh = DeShape<D>;
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
    at = Place{blockIdx.z, blockIdx.x, kGenChunkPages};
  }
  const uint32_t b = at.b, per = at.per;
  const uint32_t pbeg = (uint32_t)a.kv_indptr[b];
  const int32_t held = a.kv_indptr[b + 1u] - (int32_t)pbeg;
  uint32_t P = held > 0 ? (uint32_t)held : 0u;
  const uint32_t last = (uint32_t)a.kv_last_page_len[b];  // tokens of the table's last page
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
    const uint32_t row = a.sel_stride + (quest ? 1u : 0u);
    if (npages > row) npages = row;
  }
  if (npages > a.max_chunks * kGenChunkPages) {  // the workspace's chunks
    npages = a.max_chunks * kGenChunkPages;
    if (at.chunk == 0u && threadIdx.x == 0u) flag_error(a.error, kErrTruncated);
  }
  if ((uint64_t)at.chunk * per >= npages) return;  // uniform
  const uint32_t nsel = quest ? npages - 1u : npages;
  const int32_t* list = a.sel != nullptr ? a.sel + ((size_t)b * a.Hkv + hkv) * a.sel_stride
                                         : a.kv_indices + pbeg;
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
    __syncthreads();  // the ids before were read
    for (uint32_t i = threadIdx.x; i < np; i += kDeThreads) {
      const uint32_t page = ib + i < nsel ? (uint32_t)list[ib + i] : last_page;
      const int8_t* e = a.kv_exp + (size_t)page * 2u * a.Hkv + hkv;
      s_page[i] = page;
      s_word[i] = (uint32_t)(uint8_t)e[0] | (uint32_t)(uint8_t)e[a.Hkv] << 8 |
                  (page == last_page ? last : S) << 16;
    }
    __syncthreads();
    const uint32_t T = np * S, nb = (T + kBatch - 1u) / kBatch;  // token slots, batches
    // slot t of the list: entry and slot in its page (a slot past the end: the last)
    auto entry = [&](uint32_t t) {
      return a.page_rcp != 0u ? (uint32_t)(((uint64_t)t * a.page_rcp) >> 32) : t;
    };
    for (uint32_t i = wave; i < nb; i += kDeWaves) {
      u32x4 kr[kU][Sh::kKL];
      uint32_t vr[kU][4][Sh::kVW], kw[kU], vw[kU][S16 ? 1 : 4];
      bool whole = true;  // every slot of the batch holds a token
      const uint32_t t0 = i * kBatch;
#pragma unroll
      for (int u = 0; u < kU; ++u) {
        auto load_k = [&](uint32_t page, uint32_t slot) {
          const uint8_t* p = a.kv + (size_t)page * a.g.page + head + slot * a.g.tok + 16u * quarter;
#pragma unroll
          for (int j = 0; j < Sh::kKL; ++j)
            kr[u][j] = *reinterpret_cast<const u32x4*>(p + 64 * j);
        };
        auto load_v = [&](int r, uint32_t page, uint32_t slot) {
          const uint8_t* p = a.kv + (size_t)page * a.g.page + a.g.kv + head + slot * a.g.tok +
                             (D / 16) * col;
#pragma unroll
          for (int w = 0; w < Sh::kVW; ++w) vr[u][r][w] = reinterpret_cast<const uint32_t*>(p)[w];
        };
        if constexpr (S16) {
          const uint32_t t = t0 + 16u * u < T ? t0 + 16u * u : T - 16u;
          const uint32_t e = entry(t), slot = t - e * S;
          const uint32_t page = (uint32_t)__builtin_amdgcn_readfirstlane((int)s_page[e]);
          kw[u] = (uint32_t)__builtin_amdgcn_readfirstlane((int)s_word[e]);
          if (t0 + 16u * u >= T) kw[u] &= 0xFFFFu;  // (no token)
          whole &= slot + 16u <= tokens(kw[u]);
          load_k(page, slot + col);
#pragma unroll
          for (int r = 0; r < 4; ++r) load_v(r, page, slot + 4u * quarter + r);
        } else {
          auto place = [&](uint32_t t, uint32_t& e, uint32_t& slot, uint32_t& word) {
            const uint32_t c = t < T ? t : T - 1u;
            e = entry(c);
            slot = c - e * S;
            word = s_word[e];
            if (t >= T || slot >= tokens(word)) word &= 0xFFFFu;  // (no token)
          };
          uint32_t e, slot;
          place(t0 + 16u * u + col, e, slot, kw[u]);
          load_k(s_page[e], slot);
#pragma unroll
          for (int r = 0; r < 4; ++r) {
            place(t0 + 16u * u + 4u * quarter + r, e, slot, vw[u][r]);
            whole &= tokens(vw[u][r]) != 0u;
            load_v(r, s_page[e], slot);
          }
        }
      }
      whole = __builtin_amdgcn_ballot_w64(!whole) == 0u;
      // whether slot 4 quarter + r of unit u holds a token
      auto there = [&](int u, int r) {
        if constexpr (S16) {
          const uint32_t t = t0 + 16u * u < T ? t0 + 16u * u : T - 16u;
          return t - entry(t) * S + 4u * quarter + r < tokens(kw[u]);
        } else {
          return tokens(vw[u][r]) != 0u;
        }
      };

      floatx4 s[kU];
#pragma unroll
      for (int u = 0; u < kU; ++u) {
        const float f = k_scale(kw[u]);
        s[u] = floatx4{};
#pragma unroll
        for (int j = 0; j < Sh::kKL; ++j) {
          const u32x4 x = kr[u][j];
          s[u] = __builtin_amdgcn_mfma_f32_16x16x32_f16(
              __builtin_bit_cast(half8, decode8(uint2{x[0], x[1]}, f)), q[2 * j], s[u], 0, 0, 0);
          s[u] = __builtin_amdgcn_mfma_f32_16x16x32_f16(
              __builtin_bit_cast(half8, decode8(uint2{x[2], x[3]}, f)), q[2 * j + 1], s[u], 0, 0,
              0);
        }
      }
      if (!whole) {
#pragma unroll
        for (int u = 0; u < kU; ++u)
#pragma unroll
          for (int r = 0; r < 4; ++r)
            if (!there(u, r)) {
              s[u][r] = -INFINITY;
#pragma unroll
              for (int w = 0; w < Sh::kVW; ++w) vr[u][r][w] = 0u;  // (0 * NaN is NaN)
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
        const float keep = __builtin_amdgcn_exp2f((m - next) * a.scale);
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
            decode4(vr[u][r][w], v_scale(S16 ? kw[u] : vw[u][S16 ? 0 : r]), x[r]);
#pragma unroll
          for (int e = 0; e < 4; ++e) {
            const half4 f = {x[0][e / 2][e % 2], x[1][e / 2][e % 2], x[2][e / 2][e % 2],
                             x[3][e / 2][e % 2]};
            o[4 * w + e] = __builtin_amdgcn_mfma_f32_16x16x16f16(f, p, o[4 * w + e], 0, 0, 0);
          }
        }
      }
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
      s_ml[wave][col][0] = m * a.scale;
      s_ml[wave][col][1] = l;
    }
  }
  __syncthreads();
  for (uint32_t x = threadIdx.x; x < G * D; x += kDeThreads) {
    const uint32_t g = x / D, d = x % D;
    float M = s_ml[0][g][0];
#pragma unroll
    for (uint32_t w = 1; w < kDeWaves; ++w) M = fmaxf(M, s_ml[w][g][0]);
    float acc = 0.f, sum = 0.f;
#pragma unroll
    for (uint32_t w = 0; w < kDeWaves; ++w) {
      const float f = __builtin_amdgcn_exp2f(s_ml[w][g][0] - M);
      acc += f * s_o[w][g][d];
      sum += f * s_ml[w][g][1];
    }
    if (nch == 1u) {
      a.o[(bh0 + g) * D + d] = r16(acc / sum);
    } else {
      float* part = a.partial + ((bh0 + g) * a.max_chunks + at.chunk) * kStride;
      st_agent(part + d, acc);
      if (d == 0u) {
        st_agent(part + D, M);
        st_agent(part + D + 1u, sum);
      }
    }
  }
  if (nch == 1u) return;
  if (!arrive_last(&a.counters[bh0 * kCounterStride], nch, &s_last)) return;
  // the last chunk to arrive joins them: the loads of 8 or 16 chunks together, in order
  auto join = [&](auto group) {
    constexpr uint32_t kC = decltype(group)::value;
    for (uint32_t x = threadIdx.x; x < G * D; x += kDeThreads) {
      const uint32_t g = x / D, d = x % D;
      const float* base = a.partial + (bh0 + g) * a.max_chunks * kStride;
      float M = kPfNoMax, sum = 0.f, acc = 0.f;
      for (uint32_t c0 = 0; c0 < nch; c0 += kC) {
        float mc[kC], lc[kC], oc[kC];
#pragma unroll
        for (uint32_t u = 0; u < kC; ++u) {
          const float* part = base + (size_t)(c0 + u < nch ? c0 + u : nch - 1u) * kStride;
          mc[u] = ld_agent(part + D);
          lc[u] = ld_agent(part + D + 1u);
          oc[u] = ld_agent(part + d);
        }
        float next = M;
#pragma unroll
        for (uint32_t u = 0; u < kC; ++u) next = fmaxf(next, mc[u]);
        const float keep = __builtin_amdgcn_exp2f(M - next);
        sum *= keep;
        acc *= keep;
#pragma unroll
        for (uint32_t u = 0; u < kC; ++u) {
          const float f = c0 + u < nch ? __builtin_amdgcn_exp2f(mc[u] - next) : 0.f;
          sum += f * lc[u];
          acc += f * oc[u];
        }
        M = next;
      }
      a.o[(bh0 + g) * D + d] = r16(acc / sum);
    }
  };
  if (nch <= 8u) join(std::integral_constant<uint32_t, 8u>{});
  else join(std::integral_constant<uint32_t, 16u>{});
  __syncthreads();  // every thread has read the partials
  for (uint32_t g = 0; g < G; ++g) {  // (a workspace is left zeroed)
    uint32_t* w = reinterpret_cast<uint32_t*>(a.partial + (bh0 + g) * a.max_chunks * kStride);
    for (uint32_t i = threadIdx.x; i < nch * kStride; i += kDeThreads) st_agent_u32(w + i, 0u);
  }
}

constexpr uint32_t kDeWorkgroups = 512;  // 2 per CU

}  // namespace

hipError_t launch_decode_fp8(const DecodeFp8Args& args, uint32_t head_dim, hipStream_t s) {
  DecodeFp8Args a = args;
  auto rcp = [](uint32_t d) { return d > 1u ? (uint32_t)((1ull << 32) / d) + 1u : 0u; };
  a.page_rcp = rcp(a.S);
  a.split = kDeWorkgroups / a.Hkv > 1u ? kDeWorkgroups / a.Hkv : 1u;
  a.split_rcp = rcp(a.split);
  dim3 grid(a.max_chunks, a.Hkv, a.batch);
  if (a.sel == nullptr) {
    const uint64_t most = (uint64_t)a.max_chunks * a.batch;
    const uint32_t items =
        a.batch > 1u ? a.split + a.batch : a.split < most ? a.split : (uint32_t)most;
    constexpr uint32_t kRows = 32768u;
    grid = dim3(a.Hkv, items < kRows ? items : kRows, (items + kRows - 1u) / kRows);
  }
  const dim3 block(kDeThreads);
  const bool whole = a.S % 16u == 0u;
#define AOAKV_DE(D_)                                                                        \
  if (whole) hipLaunchKernelGGL((decode_fp8_kernel<D_, true>), grid, block, 0, s, a);       \
  else hipLaunchKernelGGL((decode_fp8_kernel<D_, false>), grid, block, 0, s, a)
  switch (head_dim) {
    case 64: AOAKV_DE(64); break;
    case 128: AOAKV_DE(128); break;
    default: AOAKV_DE(256); break;
  }
#undef AOAKV_DE
  return hipGetLastError();
}

}  // namespace aoakv
