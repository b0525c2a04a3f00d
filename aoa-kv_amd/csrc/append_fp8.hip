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
// Work.  A workgroup takes one page of one sequence, and of K's, V's and q's heads, one
// after the other, those that its lanes hold: D / 8 lanes per head, 8 dims a lane.  Lengths
// are known on the device alone, so the grid has a slot for every page that n_b new tokens
// may touch: sequence b's begin at q_indptr[b] / S + 2 b, room for n_b / S + 2 pages,
// whatever the lengths.
//
// Bounds.  K and V are read as fp16 and written as codes, q is read and written; a page's
// rows stay in registers from the load to the store, so each of their bytes passes once.
// 8192 tokens of 32 heads, rotated, with statistics: 65 us alone, 5.4 TB/s with the reading
// back of its codes (a large copy: 5.15).  16 chunks of 400 tokens and less: 21 us, where
// angles, turning and loads of a page follow each other in a workgroup.  One token of 16
// sequences: 4.6 us, a launch and the chain of lengths, page id, rows, exponent and codes.
// (With the reading back 102 to 111, 27 and 10 us; 131, 45 and 12 when a workgroup took K, V
// and q of its heads in turn, stores between the loads.)
// A block whose exponent grows has its older codes read and written again, token after
// token: a load does not pass the store before it, so the chain of one block's is what such a
// step takes, however few grow.  A token each, 8 kv heads, caches restored before each call:
// 16 sequences 6.4 us where no exponent grows, 10.8 where a tenth does, 12 where all do; 64
// behind 14 tokens of a page 5.8, 13 and 14, behind 30 6.4, 22 and 23.
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

typedef uint32_t u32x2 __attribute__((ext_vector_type(2)));
template <class V>
__device__ inline void st_nt(void* p, const V& v) {
  __builtin_nontemporal_store(v, static_cast<V*>(p));
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

// sine and cosine of f / 2^64 turns: a polynomial in fp64 on half a quadrant (the first
// term left out is 1.2e-10), for a rounding to fp32 that is the values' own
__device__ inline float2 cos_sin(uint64_t f) {
  const int32_t x = (int32_t)(f >> 32);                 // of 2^32, -1/2 .. 1/2 turn
  const int32_t q = ((x >> 29) + 1) >> 1;               // nearest quadrant, -2 .. 2
  const double a = (double)(int32_t)((uint32_t)x - ((uint32_t)q << 30)) *
                   (6.283185307179586 / 4294967296.0);
  const double z = a * a;
  double s = __builtin_fma(z, -1.0 / 39916800.0, 1.0 / 362880.0);
  s = __builtin_fma(z, s, -1.0 / 5040.0);
  s = __builtin_fma(z, s, 1.0 / 120.0);
  s = __builtin_fma(z, s, -1.0 / 6.0);
  s = __builtin_fma(a * z, s, a);
  double c = __builtin_fma(z, -1.0 / 3628800.0, 1.0 / 40320.0);
  c = __builtin_fma(z, c, -1.0 / 720.0);
  c = __builtin_fma(z, c, 1.0 / 24.0);
  c = __builtin_fma(z, c, -0.5);
  c = __builtin_fma(z, c, 1.0);
  const float fs = (float)s, fc = (float)c;
  const float y = q & 1 ? fc : fs, w = q & 1 ? fs : fc;
  return float2{(q + 1) & 2 ? -w : w, q & 2 ? -y : y};
}

template <int D, int TOK, bool ROPE>
__global__ __launch_bounds__(kApThreads) void append_fp8_kernel(AppendFp8Args a) {
  constexpr uint32_t N = D / 8, kHeads = kApThreads / N;  // lanes and heads of a workgroup
  __shared__ float2 s_cs[ROPE ? TOK : 1][D / 2];
  const uint32_t group = blockIdx.y;
  const PageTokens t = find_page(a, blockIdx.x);
  if (t.n == 0u) return;  // uniform
  const uint32_t l = threadIdx.x % N, S = a.S;
  // what the lanes of a head do: K of a.H heads, V of them, q of a.Hq
  uint32_t h = group * kHeads + threadIdx.x / N;
  const bool turns = ROPE && (group * kHeads < a.H || (group + 1u) * kHeads > 2u * a.H);
  if (turns) {  // (uniform) cosine and sine of the page's tokens, once per workgroup
    for (uint32_t i = threadIdx.x; i < t.n * (D / 2); i += kApThreads)
      s_cs[i / (D / 2)][i % (D / 2)] =
          cos_sin(a.rope.turns[i % (D / 2)] * (uint64_t)(t.pos + i / (D / 2)));
    __syncthreads();
  }
  const float2* cs = &s_cs[0][(l * kVec) % (D / 2)];
  const uint32_t kind = h < a.H ? 0u : h < 2u * a.H ? 1u : 2u;
  h -= kind * a.H;
  const uint32_t heads = kind == 2u ? a.Hq : a.H;
  if (h >= heads) return;  // whole heads
  const f16* src = (kind == 0u ? a.k : kind == 1u ? a.v : a.q) + ((size_t)t.row * heads + h) * D +
                   l * kVec;
  const size_t step = (size_t)heads * D;
  // all tokens' loads together: before the first store, which they could not pass
  H8 x[TOK];
  if (a.stream) {
#pragma unroll
    for (int i = 0; i < TOK; ++i)
      if ((uint32_t)i < t.n) x[i] = ld16_nt(src + i * step);
  } else {
#pragma unroll
    for (int i = 0; i < TOK; ++i)
      if ((uint32_t)i < t.n) x[i] = ld16(src + i * step);
  }
  if (ROPE && kind != 1u) {
#pragma unroll
    for (int i = 0; i < TOK; ++i)
      if ((uint32_t)i < t.n) x[i] = turn<N>(x[i], cs + i * (D / 2), l);
  }
  if (kind == 2u) {
    f16* q = const_cast<f16*>(src);  // (a.q)
    if (a.stream) {
#pragma unroll
      for (int i = 0; i < TOK; ++i)
        if ((uint32_t)i < t.n) st_nt(q + i * step, __builtin_bit_cast(u32x4, x[i]));
    } else {
#pragma unroll
      for (int i = 0; i < TOK; ++i)
        if ((uint32_t)i < t.n) st16(q + i * step, x[i]);
    }
    return;
  }

  uint32_t top = 0u;
#pragma unroll
  for (int i = 0; i < TOK; ++i)
    if ((uint32_t)i < t.n) top = pair_top(x[i], top);
  top = top >> 16 > (top & 0xFFFFu) ? top >> 16 : top & 0xFFFFu;
  if (top >= 0x7C00u) {  // (inf or NaN among them: the largest of the others)
    top = 0u;
#pragma unroll
    for (int i = 0; i < TOK; ++i)
      if ((uint32_t)i < t.n) top = finite_top(x[i], top);
  }
  int e = block_exp(lanes_max<N>(top));
  int8_t* ep = a.kv_exp + ((size_t)t.page * 2u + kind) * a.H + h;
  uint8_t* out = a.kv + elem_off(a.g, t.page, kind, h, t.e0) + l * kVec;
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
  if (a.stream) {
#pragma unroll
    for (int i = 0; i < TOK; ++i)
      if ((uint32_t)i < t.n)
        st_nt(out + (size_t)i * a.g.tok, __builtin_bit_cast(u32x2, encode8(x[i], e)));
  } else {
#pragma unroll
    for (int i = 0; i < TOK; ++i)
      if ((uint32_t)i < t.n)
        *reinterpret_cast<uint2*>(out + (size_t)i * a.g.tok) = encode8(x[i], e);
  }
  if (a.meta == nullptr) return;

  if (kind == 0u) {
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
}

// As the append, K and V of a head by lanes of their own; kRead tokens' loads together.
// Whole batches are bound by HBM (4 sequences of 8192 tokens, 32 heads: 98 to 107 us, 5.0
// to 5.4 TB/s), a page of each of 16 sequences by the chain of lengths, page id, codes (3.8).
template <int D>
__global__ __launch_bounds__(kApThreads) void read_fp8_kernel(AppendFp8Args a) {
  constexpr uint32_t N = D / 8, kHeads = kApThreads / N, kRead = 8u;
  const PageTokens t = find_page(a, blockIdx.x);
  const uint32_t l = threadIdx.x % N;
  uint32_t h = blockIdx.y * kHeads + threadIdx.x / N;
  if (t.n == 0u || h >= 2u * a.H) return;
  const uint32_t kind = h < a.H ? 0u : 1u;
  h -= kind * a.H;
  const float scale = exp_scale(a.kv_exp[((size_t)t.page * 2u + kind) * a.H + h]);
  const uint8_t* src = a.kv + elem_off(a.g, t.page, kind, h, t.e0) + l * kVec;
  const size_t step = (size_t)a.H * D;
  f16* out = (kind == 0u ? a.k_out : a.v_out) + ((size_t)t.row * a.H + h) * D + l * kVec;
  for (uint32_t i0 = 0; i0 < t.n; i0 += kRead) {
    uint2 c[kRead];
#pragma unroll
    for (uint32_t u = 0; u < kRead; ++u) {
      const uint32_t i = i0 + u < t.n ? i0 + u : t.n - 1u;
      c[u] = *reinterpret_cast<const uint2*>(src + (size_t)i * a.g.tok);
    }
#pragma unroll
    for (uint32_t u = 0; u < kRead; ++u)
      if (i0 + u < t.n) st16(out + (i0 + u) * step, decode8(c[u], scale));
  }
}

uint32_t page_slots(const AppendFp8Args& a) { return a.T / a.S + 2u * a.B; }

// Rows of so many bytes pass the caches by (non-temporal loads and stores).  Three
// prompts in turn, and their codes read back, us without / with: 8192 tokens x 32 heads
// (201 MB of rows) 122 / 101, 4096 (the append alone) 45 / 38, 2048 22 / 22; a batch of
// 40 MB 29 / 35, which the memory-side cache holds from call to call as it would hold what
// a projection has just written.
constexpr uint64_t kStreamBytes = 64u << 20;

template <int D, int TOK>
hipError_t launch(const AppendFp8Args& args, hipStream_t s) {
  constexpr uint32_t kHeads = kApThreads / (D / 8);
  AppendFp8Args a = args;
  // (pages side by side: a prompt of 8192 tokens x 32 heads 81 us, and 85 with the heads
  // of a page so)
  const uint32_t heads = 2u * a.H + (a.q != nullptr ? a.Hq : 0u);
  a.stream = (uint64_t)a.T * heads * D * sizeof(f16) >= kStreamBytes ? 1u : 0u;
  const dim3 grid(page_slots(a), (heads + kHeads - 1u) / kHeads);
  if (a.q != nullptr) {
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
  const dim3 grid(page_slots(a), (2u * a.H + heads - 1u) / heads), block(kApThreads);
  switch (head_dim) {
    case 64: hipLaunchKernelGGL(read_fp8_kernel<64>, grid, block, 0, s, a); break;
    case 128: hipLaunchKernelGGL(read_fp8_kernel<128>, grid, block, 0, s, a); break;
    default: hipLaunchKernelGGL(read_fp8_kernel<256>, grid, block, 0, s, a); break;
  }
  return hipGetLastError();
}

}  // namespace aoakv
