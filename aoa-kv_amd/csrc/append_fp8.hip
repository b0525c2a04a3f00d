// New tokens of a ragged batch into a paged cache of 8-bit codes, with the position
// rotation on the way, and tokens of such a cache back as fp16 rows (gfx950).
//
// Row r of sequence b (rows q_indptr[b] .. q_indptr[b + 1] - 1 of k, v and q, the last
// n_b of its L_b cached tokens) is at position pos = L_b - n_b + r - q_indptr[b]:
//   (x_i, x_(i + D/2)) turns by pos * f_i,  f_i = theta^(-2 i / D) / scale,
//   a block (page, K or V, kv head) has the exponent e = max(the exponent of its older
//   tokens, block_exp(its new tokens' largest)), codes = e4m3(x / 2^e)
// (fp8.hpp).  The page statistics, where asked for, are those of append.hip, bit for
// bit, of the fp16 rows.
//
// Angles.  A position times a frequency in fp32 is off by 2^-24 of itself, 1e-3 at
// position 16000, more than the fp16 result's rounding.  Here f_i / 2 pi is a
// 64-bit fraction of a turn made on the host, its product with the position drops the
// whole turns by overflow, and sine and cosine take what is left.
//
// Work.  A workgroup takes one page of one sequence and the heads that its lanes hold:
// D / 8 lanes per head, 8 dims a lane.  Lengths are known on the device alone, so the
// grid has a slot for every page that n_b new tokens may touch: sequence b's begin at
// q_indptr[b] / S + 2 b, room for n_b / S + 2 pages, whatever the lengths.
#include <type_traits>

#include "fp8.hpp"
#include "kernels.hpp"

namespace aoakv {
namespace {

constexpr uint32_t kApThreads = 256;

// A page's new tokens: slots e0 .. e0 + n - 1 of page `page` hold rows row .. row + n - 1.
struct PageTokens {
  uint32_t b, p, page, e0, n, row, pos;  // pos: of the first row
};

// What slot x of the grid has to do (n == 0: nothing).
__device__ inline PageTokens find_page(const AppendFp8Args& a, uint32_t x) {
  const uint32_t lane = __lane_id();
  const int32_t T = (int32_t)a.T;
  // the last sequence whose slots begin at x or before: 64 are tried at a time
  uint32_t lo = 0u, n = a.B;
  for (;;) {
    const uint32_t stride = (n + kWave - 1u) / kWave;
    const bool in = lane * stride < n;
    const uint32_t i = lo + (in ? lane * stride : 0u);
    const uint32_t r = (uint32_t)min(max(a.tok_indptr[i], 0), T);
    const uint64_t le = __builtin_amdgcn_ballot_w64(in && r / a.S + 2u * i <= x);
    if (le == 0u) return PageTokens{};
    const uint32_t j = 63u - (uint32_t)__builtin_clzll(le);
    lo += j * stride;
    if (stride == 1u) break;
    const uint32_t left = n - j * stride;
    n = left < stride ? left : stride;
  }
  const uint32_t b = (uint32_t)__builtin_amdgcn_readfirstlane((int)lo);
  const int32_t r0 = min(max(a.tok_indptr[b], 0), T), r1 = min(a.tok_indptr[b + 1u], T);
  const int32_t p0 = a.kv_indptr[b], P = a.kv_indptr[b + 1u] - p0;
  const int32_t S = (int32_t)a.S, last = min(max(a.kv_last_page_len[b], 1), S);
  const int32_t N = r1 - r0;
  if (N <= 0 || P <= 0) return PageTokens{};
  const int64_t L = (int64_t)(P - 1) * S + last;
  const int64_t off = L - N, start = off > 0 ? off : 0;  // (rows before the sequence: dropped)
  const int64_t p = start / S + (int64_t)(x - ((uint32_t)r0 / a.S + 2u * b));
  const int64_t e0 = start > p * S ? start - p * S : 0;
  const int64_t e1 = L - p * S < S ? L - p * S : S;
  if (e1 <= e0) return PageTokens{};
  PageTokens t;
  t.b = b;
  t.p = (uint32_t)p;
  t.page = (uint32_t)a.kv_indices[p0 + (int32_t)p];
  t.e0 = (uint32_t)e0;
  t.n = (uint32_t)(e1 - e0);
  t.row = (uint32_t)(r0 + (p * S + e0 - off));
  t.pos = (uint32_t)(p * S + e0);
  return t;
}

// max over the N lanes of a head
template <uint32_t N>
__device__ inline uint32_t lanes_max(uint32_t x) {
#pragma unroll
  for (uint32_t m = 1; m < N; m <<= 1) {
    const uint32_t y = (uint32_t)__shfl_xor((int)x, (int)m, kWave);
    x = y > x ? y : x;
  }
  return x;
}

// 8 dims of a head turned: c, s of their angles, the partner dims in lane l ^ N / 2
template <uint32_t N>
__device__ inline H8 turn(const H8& x, const float2* cs, uint32_t l) {
  const uint4 u = __builtin_bit_cast(uint4, x);
  uint4 pu;
  if constexpr (N == 16u) {
    pu.x = (uint32_t)__builtin_amdgcn_mov_dpp((int)u.x, 0x128, 0xF, 0xF, false);  // row_ror:8
    pu.y = (uint32_t)__builtin_amdgcn_mov_dpp((int)u.y, 0x128, 0xF, 0xF, false);
    pu.z = (uint32_t)__builtin_amdgcn_mov_dpp((int)u.z, 0x128, 0xF, 0xF, false);
    pu.w = (uint32_t)__builtin_amdgcn_mov_dpp((int)u.w, 0x128, 0xF, 0xF, false);
  } else {
    pu.x = (uint32_t)__shfl_xor((int)u.x, (int)(N / 2u), kWave);
    pu.y = (uint32_t)__shfl_xor((int)u.y, (int)(N / 2u), kWave);
    pu.z = (uint32_t)__shfl_xor((int)u.z, (int)(N / 2u), kWave);
    pu.w = (uint32_t)__shfl_xor((int)u.w, (int)(N / 2u), kWave);
  }
  const H8 p = __builtin_bit_cast(H8, pu);
  const bool low = l < N / 2u;
  H8 y;
#pragma unroll
  for (int j = 0; j < kVec; ++j) {
    const float2 t = cs[j];
    const float v = (float)p.v[j] * t.y;
    y.v[j] = r16(__builtin_fmaf((float)x.v[j], t.x, low ? -v : v));
  }
  return y;
}

template <int D, int TOK, bool ROPE>
__global__ __launch_bounds__(kApThreads) void append_fp8_kernel(AppendFp8Args a) {
  constexpr uint32_t N = D / 8, kHeads = kApThreads / N;  // lanes per head, heads per workgroup
  __shared__ float2 s_cs[ROPE ? TOK : 1][D / 2];
  const PageTokens t = find_page(a, blockIdx.x);
  if (t.n == 0u) return;  // uniform
  const uint32_t l = threadIdx.x % N, S = a.S;
  const uint32_t kv_blocks = (a.H + kHeads - 1u) / kHeads;
  const bool turns_q = ROPE && blockIdx.y >= kv_blocks;  // uniform
  const uint32_t h = (turns_q ? blockIdx.y - kv_blocks : blockIdx.y) * kHeads + threadIdx.x / N;
  if constexpr (ROPE) {  // cosine and sine of the page's tokens, once per workgroup
    for (uint32_t i = threadIdx.x; i < t.n * (D / 2); i += kApThreads) {
      const uint64_t f = a.rope.turns[i % (D / 2)] * (uint64_t)(t.pos + i / (D / 2));
      const float x = (float)(int32_t)(f >> 32) * 0x1p-32f;  // of a turn, -1/2 .. 1/2
      s_cs[i / (D / 2)][i % (D / 2)] =
          float2{__builtin_amdgcn_cosf(x), __builtin_amdgcn_sinf(x)};
    }
    __syncthreads();
  }
  const float2* cs = &s_cs[0][(l * kVec) % (D / 2)];
  if (turns_q) {
    if (h >= a.Hq) return;
    f16* q = a.q + ((size_t)t.row * a.Hq + h) * D + l * kVec;
    for (uint32_t i = 0; i < t.n; ++i) {
      f16* x = q + (size_t)i * a.Hq * D;
      st16(x, turn<N>(ld16(x), cs + i * (D / 2), l));
    }
    return;
  }
  if (h >= a.H) return;  // whole heads

  const size_t in = ((size_t)t.row * a.H + h) * D + l * kVec, step = (size_t)a.H * D;
  // K, then V
  auto block = [&](auto kind) {
    constexpr uint32_t which = decltype(kind)::value;
    const f16* src = (which == 0u ? a.k : a.v) + in;
    H8 x[TOK];
#pragma unroll
    for (int i = 0; i < TOK; ++i)
      if ((uint32_t)i < t.n) x[i] = ld16(src + i * step);
    uint32_t top = 0u;
#pragma unroll
    for (int i = 0; i < TOK; ++i)
      if ((uint32_t)i < t.n) {
        if constexpr (ROPE && which == 0u) x[i] = turn<N>(x[i], cs + i * (D / 2), l);
        top = finite_top(x[i], top);
      }
    int e = block_exp(lanes_max<N>(top));
    int8_t* ep = a.kv_exp + ((size_t)t.page * 2u + which) * a.H + h;
    uint8_t* out = a.kv + elem_off(a.g, t.page, which, h, t.e0) + l * kVec;
    if (t.e0 != 0u) {  // the page holds tokens: the block's exponent only grows
      int old = *ep;
      old = old < kMinExp ? kMinExp : old > kMaxExp ? kMaxExp : old;
      if (e > old) {
        for (uint32_t i = 1; i <= t.e0; ++i) {
          uint2* c = reinterpret_cast<uint2*>(out - (size_t)i * a.g.tok);
          *c = encode8(decode8(*c, exp_scale(old)), e);
        }
      } else {
        e = old;
      }
    }
    if (l == 0u) *ep = (int8_t)e;
#pragma unroll
    for (int i = 0; i < TOK; ++i)
      if ((uint32_t)i < t.n) *reinterpret_cast<uint2*>(out + (size_t)i * a.g.tok) = encode8(x[i], e);
    if (a.meta == nullptr) return;

    if constexpr (which == 0u) {
      const uint32_t mpage = (uint32_t)a.meta_indices[(uint32_t)a.meta_indptr[t.b] + t.p / S];
      f16* kmax_p = a.meta + elem_off(a.g, mpage, 0, h, t.p % S) + l * kVec;
      f16* kmin_p = a.meta + elem_off(a.g, mpage, 1, h, t.p % S) + l * kVec;
      H8 kmax, kmin;
      if (t.e0 != 0u) {
        kmax = ld16(kmax_p);
        kmin = ld16(kmin_p);
      } else {
#pragma unroll
        for (int j = 0; j < kVec; ++j) {
          kmax.v[j] = (f16)-65504.0f;
          kmin.v[j] = (f16)65504.0f;
        }
      }
#pragma unroll
      for (int i = 0; i < TOK; ++i)
        if ((uint32_t)i < t.n)
#pragma unroll
          for (int j = 0; j < kVec; ++j) {
            kmax.v[j] = x[i].v[j] > kmax.v[j] ? x[i].v[j] : kmax.v[j];
            kmin.v[j] = x[i].v[j] < kmin.v[j] ? x[i].v[j] : kmin.v[j];
          }
      st16(kmax_p, kmax);
      st16(kmin_p, kmin);
    } else {  // (the mean of a page that begins empty, else the running mean)
      const size_t at = (size_t)t.page * a.H + h;
      f16* mean_p = a.v_mean + at * D + l * kVec;
      H8 mean;
      if (t.e0 == 0u) {
        float sum[kVec] = {};
#pragma unroll
        for (int i = 0; i < TOK; ++i)
          if ((uint32_t)i < t.n)
#pragma unroll
            for (int j = 0; j < kVec; ++j) sum[j] = sum[j] + (float)x[i].v[j];
#pragma unroll
        for (int j = 0; j < kVec; ++j) mean.v[j] = r16(sum[j] / (float)t.n);
      } else {
        mean = ld16(mean_p);
#pragma unroll
        for (int i = 0; i < TOK; ++i)
          if ((uint32_t)i < t.n)
#pragma unroll
            for (int j = 0; j < kVec; ++j)
              mean.v[j] = running_mean(mean.v[j], x[i].v[j], t.e0 + (uint32_t)i);
      }
      st16(mean_p, mean);
      const f16 norm = N == 16u ? log_norm_row(mean) : grp_log_norm<N>(mean, l);
      if (l == 0u) a.v_log_norm[at] = norm;
    }
  };
  block(std::integral_constant<uint32_t, 0u>{});
  block(std::integral_constant<uint32_t, 1u>{});
}

template <int D>
__global__ __launch_bounds__(kApThreads) void read_fp8_kernel(AppendFp8Args a) {
  constexpr uint32_t N = D / 8, kHeads = kApThreads / N;
  const PageTokens t = find_page(a, blockIdx.x);
  const uint32_t l = threadIdx.x % N, h = blockIdx.y * kHeads + threadIdx.x / N;
  if (t.n == 0u || h >= a.H) return;
  const size_t to = ((size_t)t.row * a.H + h) * D + l * kVec, step = (size_t)a.H * D;
#pragma unroll
  for (int which = 0; which < 2; ++which) {
    const float scale = exp_scale(a.kv_exp[((size_t)t.page * 2u + which) * a.H + h]);
    const uint8_t* src = a.kv + elem_off(a.g, t.page, which, h, t.e0) + l * kVec;
    f16* out = (which == 0 ? a.k_out : a.v_out) + to;
    for (uint32_t i = 0; i < t.n; ++i)
      st16(out + i * step,
           decode8(*reinterpret_cast<const uint2*>(src + (size_t)i * a.g.tok), scale));
  }
}

uint32_t page_slots(const AppendFp8Args& a) { return a.T / a.S + 2u * a.B; }

template <int D, int TOK>
hipError_t launch(const AppendFp8Args& a, hipStream_t s) {
  constexpr uint32_t kHeads = kApThreads / (D / 8);
  dim3 grid(page_slots(a), (a.H + kHeads - 1u) / kHeads);
  if (a.q != nullptr) {
    grid.y += (a.Hq + kHeads - 1u) / kHeads;
    hipLaunchKernelGGL((append_fp8_kernel<D, TOK, true>), grid, dim3(kApThreads), 0, s, a);
  } else {
    hipLaunchKernelGGL((append_fp8_kernel<D, TOK, false>), grid, dim3(kApThreads), 0, s, a);
  }
  return hipGetLastError();
}
template <int D>
hipError_t launch(const AppendFp8Args& a, hipStream_t s) {
  return a.S <= 16u ? launch<D, 16>(a, s) : launch<D, 32>(a, s);
}

}  // namespace

hipError_t launch_append_fp8(const AppendFp8Args& a, uint32_t head_dim, hipStream_t s) {
  switch (head_dim) {
    case 64: return launch<64>(a, s);
    case 128: return launch<128>(a, s);
    default: return launch<256>(a, s);
  }
}

hipError_t launch_read_fp8(const AppendFp8Args& a, uint32_t head_dim, hipStream_t s) {
  const uint32_t heads = kApThreads / (head_dim / 8u);
  const dim3 grid(page_slots(a), (a.H + heads - 1u) / heads), block(kApThreads);
  switch (head_dim) {
    case 64: hipLaunchKernelGGL(read_fp8_kernel<64>, grid, block, 0, s, a); break;
    case 128: hipLaunchKernelGGL(read_fp8_kernel<128>, grid, block, 0, s, a); break;
    default: hipLaunchKernelGGL(read_fp8_kernel<256>, grid, block, 0, s, a); break;
  }
  return hipGetLastError();
}

}  // namespace aoakv
