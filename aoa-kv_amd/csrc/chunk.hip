// Attention of a ragged batch of chunks of new tokens over the paged cache, and
// the attention weight that each cached token received from them (gfx950).
//
// Query i of sequence b (n_b new tokens, the last of its L_b cached ones) is at
// position pos = L_b - n_b + i and scores key j
//   t = q_i . k_j / sqrt(D),  t = c tanh(t / c)  (soft cap),
//   t -= slope_h |pos - j|    (distance bias),
// where it sees it: j < L_b, and j <= pos (causal), j > pos - window, or j <
// prefix_len[b] whatever these say.  lse = log sum_j exp(t), o = sum_j exp(t -
// lse) v_j; a query that sees no key has o = 0 and lse = -inf.  The weight of
// key j in a kv head is the sum of exp(t - lse) over the queries of its group.
#include "kernels.hpp"

namespace aoakv {
namespace {

constexpr uint32_t kChThreads = 256;

// What the device tables say of sequence b, held to the sizes of the call.
struct Seq {
  int32_t q0, n, L, off, prefix;  // first row, new tokens, cached tokens, L - n
  uint32_t page0;                 // first entry of kv_indices
};
__device__ inline Seq load_seq(const ChunkArgs& a, uint32_t b) {
  Seq s;
  const int32_t T = (int32_t)a.T;
  s.q0 = min(max(a.q_indptr[b], 0), T);
  s.n = max(min(a.q_indptr[b + 1], T) - s.q0, 0);
  const int32_t p0 = a.kv_indptr[b];
  int32_t P = max(a.kv_indptr[b + 1] - p0, 0);
  int32_t last = min(max(a.kv_last_page_len[b], 1), (int32_t)a.S);
  if (P > (int32_t)a.max_pages) {
    flag_error(a.error, kErrTruncated);
    P = (int32_t)a.max_pages;
    last = (int32_t)a.S;
  }
  s.page0 = (uint32_t)p0;
  s.L = P > 0 ? (P - 1) * (int32_t)a.S + last : 0;
  s.off = s.L - s.n;
  s.prefix = a.prefix_len != nullptr ? a.prefix_len[b] : 0;
  return s;
}

__device__ inline bool sees(const ChunkArgs& a, const Seq& s, int32_t pos, int32_t j) {
  return j < s.L && (j < s.prefix || ((!a.causal || j <= pos) &&
                                      (a.window == 0u || pos - j < (int32_t)a.window)));
}

__device__ inline float score(const ChunkArgs& a, float dot, uint32_t h, int32_t pos, int32_t j) {
  float t = dot * a.sm_scale;
  if (a.soft_cap > 0.f) t = a.soft_cap * tanhf(t / a.soft_cap);
  if (a.slopes != nullptr) t -= a.slopes[h] * (float)abs(pos - j);
  return t;
}

// the sequence that row t belongs to (B: none)
__device__ inline uint32_t seq_of(const ChunkArgs& a, int32_t t) {
  uint32_t lo = 0u, hi = a.B;
  while (lo < hi) {
    const uint32_t mid = (lo + hi) / 2u;
    if (a.q_indptr[mid + 1u] <= t) lo = mid + 1u;
    else hi = mid;
  }
  return lo;
}

__device__ inline float wave_max(float x) {
#pragma unroll
  for (int m = 32; m; m >>= 1) x = fmaxf(x, __shfl_xor(x, m));
  return x;
}
__device__ inline float wave_sum(float x) {
#pragma unroll
  for (int m = 32; m; m >>= 1) x += __shfl_xor(x, m);
  return x;
}

// One wave per (row, query head): 64 keys at a time, a key per lane for the
// scores, D / 64 dims per lane for the values.
template <int D>
__global__ __launch_bounds__(kChThreads) void chunk_attn_kernel(ChunkArgs a) {
  const uint32_t lane = __lane_id(), wave = threadIdx.x / kWave;
  const uint64_t item = (uint64_t)blockIdx.x * (kChThreads / kWave) + wave;
  if (item >= (uint64_t)a.T * a.Hq) return;
  const uint32_t t = (uint32_t)(item / a.Hq), h = (uint32_t)(item % a.Hq), hk = h / (a.Hq / a.H);
  if ((int32_t)t < a.q_indptr[0]) return;
  const uint32_t b = seq_of(a, (int32_t)t);
  if (b >= a.B) return;
  const Seq s = load_seq(a, b);
  const int32_t pos = s.off + (int32_t)t - s.q0;
  const f16* q = a.q + ((size_t)t * a.Hq + h) * D;
  constexpr int kN = D / kWave;
  float acc[kN] = {}, m = -INFINITY, l = 0.f;
  for (int32_t j0 = 0; j0 < s.L; j0 += kWave) {
    const int32_t j = j0 + (int32_t)lane;
    const bool ok = sees(a, s, pos, j);
    uint64_t live = __ballot(ok);
    if (live == 0u) continue;
    uint32_t page = 0u, slot = 0u;
    float x = -INFINITY;
    if (ok) {
      page = (uint32_t)a.kv_indices[s.page0 + (uint32_t)j / a.S];
      slot = (uint32_t)j % a.S;
      const f16* k = a.kv + elem_off(a.g, page, 0, hk, slot);
      float dot = 0.f;
      for (int d = 0; d < D; ++d) dot += (float)q[d] * (float)k[d];
      x = score(a, dot, h, pos, j);
    }
    const float top = fmaxf(m, wave_max(x));
    const float base = top == -INFINITY ? 0.f : top;
    const float p = ok ? expf(x - base) : 0.f, w = expf(m - base);
    l = l * w + wave_sum(p);
    for (int i = 0; i < kN; ++i) acc[i] *= w;
    m = top;
    for (; live != 0u; live &= live - 1u) {
      const int src = __ffsll((unsigned long long)live) - 1;
      const float pj = __shfl(p, src);
      const f16* v = a.kv + elem_off(a.g, __shfl(page, src), 1, hk, __shfl(slot, src));
      for (int i = 0; i < kN; ++i) acc[i] += pj * (float)v[lane * kN + i];
    }
  }
  f16* o = a.o + ((size_t)t * a.Hq + h) * D;
  for (int i = 0; i < kN; ++i) o[lane * kN + i] = r16(l > 0.f ? acc[i] / l : l == 0.f ? 0.f : l);
  if (a.lse != nullptr && lane == 0u) a.lse[(size_t)t * a.Hq + h] = l == 0.f ? -INFINITY : m + logf(l);
}

// One thread per (sequence, kv head, key): the sum over the queries in order.
template <int D>
__global__ __launch_bounds__(kChThreads) void attn_weights_kernel(ChunkArgs a) {
  const uint32_t b = blockIdx.z, hk = blockIdx.y, G = a.Hq / a.H;
  const Seq s = load_seq(a, b);
  for (int32_t j = (int32_t)(blockIdx.x * kChThreads + threadIdx.x); j < s.L;
       j += (int32_t)(gridDim.x * kChThreads)) {
    const uint32_t page = (uint32_t)a.kv_indices[s.page0 + (uint32_t)j / a.S];
    const uint32_t slot = (uint32_t)j % a.S;
    const f16* k = a.kv + elem_off(a.g, page, 0, hk, slot);
    float sum = 0.f;
    for (int32_t i = 0; i < s.n; ++i) {
      const int32_t pos = s.off + i;
      if (!sees(a, s, pos, j)) continue;
      for (uint32_t gi = 0; gi < G; ++gi) {
        const uint32_t h = hk * G + gi;
        const size_t row = (size_t)(s.q0 + i) * a.Hq + h;
        float dot = 0.f;
        for (int d = 0; d < D; ++d) dot += (float)a.q[row * D + d] * (float)k[d];
        const float lse = a.lse[row];
        sum += lse == -INFINITY ? 0.f : expf(score(a, dot, h, pos, j) - lse);
      }
    }
    float* w = a.weights + ((size_t)page * a.H + hk) * a.S + slot;
    const int32_t start = a.start != nullptr ? a.start[b] : s.off;
    *w = (j < start ? *w : 0.f) + sum;
  }
}

}  // namespace

hipError_t launch_chunk_attn(const ChunkArgs& a, uint32_t head_dim, hipStream_t s) {
  const dim3 grid((uint32_t)(((uint64_t)a.T * a.Hq + 3u) / 4u)), block(kChThreads);
  switch (head_dim) {
    case 64: hipLaunchKernelGGL(chunk_attn_kernel<64>, grid, block, 0, s, a); break;
    case 128: hipLaunchKernelGGL(chunk_attn_kernel<128>, grid, block, 0, s, a); break;
    default: hipLaunchKernelGGL(chunk_attn_kernel<256>, grid, block, 0, s, a); break;
  }
  return hipGetLastError();
}

hipError_t launch_attn_weights(const ChunkArgs& a, uint32_t head_dim, hipStream_t s) {
  const uint64_t blocks = ((uint64_t)a.max_pages * a.S + kChThreads - 1u) / kChThreads;
  const dim3 grid((uint32_t)(blocks < 1024u ? blocks : 1024u), a.H, a.B), block(kChThreads);
  switch (head_dim) {
    case 64: hipLaunchKernelGGL(attn_weights_kernel<64>, grid, block, 0, s, a); break;
    case 128: hipLaunchKernelGGL(attn_weights_kernel<128>, grid, block, 0, s, a); break;
    default: hipLaunchKernelGGL(attn_weights_kernel<256>, grid, block, 0, s, a); break;
  }
  return hipGetLastError();
}

}  // namespace aoakv
