// Eviction from the paged cache (gfx950): which tokens each kv head keeps by
// the attention weight they received, and the cache packed down to them with
// its page statistics.
#include "kernels.hpp"

namespace aoakv {
namespace {

constexpr uint32_t kEvThreads = 1024;

// tokens of sequence b, held to the call's page bound
__device__ inline uint32_t seq_tokens(const int32_t* indptr, const int32_t* last_page_len,
                                      uint32_t b, uint32_t max_pages, uint32_t S,
                                      uint32_t* error) {
  const int32_t P = indptr[b + 1] - indptr[b];
  const int32_t last = min(max(last_page_len[b], 1), (int32_t)S);
  if (P <= 0) return 0u;
  if ((uint32_t)P > max_pages) {
    flag_error(error, kErrTruncated);
    return max_pages * S;
  }
  return (uint32_t)(P - 1) * S + (uint32_t)last;
}

// the sum of x over the workgroup's threads before this one, and the total
__device__ inline uint32_t block_scan(uint32_t x, uint32_t* s_wave, uint32_t& total) {
  const uint32_t lane = __lane_id(), wave = threadIdx.x / kWave;
  uint32_t y = x;
#pragma unroll
  for (uint32_t d = 1; d < (uint32_t)kWave; d <<= 1) {
    const uint32_t z = __shfl_up(y, d);
    if (lane >= d) y += z;
  }
  __syncthreads();
  if (lane == kWave - 1u) s_wave[wave] = y;
  __syncthreads();
  uint32_t before = 0u;
  total = 0u;
  for (uint32_t w = 0; w < kEvThreads / kWave; ++w) {
    if (w < wave) before += s_wave[w];
    total += s_wave[w];
  }
  return before + y - x;
}

// One workgroup per (kv head, sequence).  The order of two weights is that of
// their keys (NaN lowest, -0 as 0); 8 bits of the key at a time, a histogram
// finds the key of the last token kept, and how many of the tokens with just
// that key (the lowest positions) are kept with it.
__global__ __launch_bounds__(kEvThreads) void keep_kernel(KeepArgs a) {
  __shared__ uint32_t s_hist[256], s_wave[kEvThreads / kWave], s_pick[2];
  const uint32_t h = blockIdx.x, b = blockIdx.y, tid = threadIdx.x;
  const uint32_t L = seq_tokens(a.kv_indptr, a.kv_last_page_len, b, a.max_pages, a.S, a.error);
  const uint32_t page0 = (uint32_t)a.kv_indptr[b];
  int32_t* out = a.kept + ((size_t)b * a.H + h) * a.stride;
  if (L <= a.keep) {
    for (uint32_t j = tid; j < L; j += kEvThreads) out[j] = (int32_t)j;
    return;
  }
  const uint32_t lo = a.sink, hi = L - a.recent;  // the tokens that compete (lo <= hi)
  auto key_of = [&](uint32_t j) {
    const uint32_t page = (uint32_t)a.kv_indices[page0 + j / a.S];
    const float w = a.weights[((size_t)page * a.H + h) * a.S + j % a.S] + 0.f;
    return w == w ? order_key(w) : 0u;
  };
  uint32_t need = a.keep - a.sink - a.recent, prefix = 0u, mask = 0u;
  for (int shift = 24; shift >= 0 && need != 0u; shift -= 8) {
    if (tid < 256u) s_hist[tid] = 0u;
    __syncthreads();
    for (uint32_t j = lo + tid; j < hi; j += kEvThreads) {
      const uint32_t k = key_of(j);
      if ((k & mask) == prefix) atomicAdd(&s_hist[(k >> shift) & 255u], 1u);
    }
    __syncthreads();
    if (tid == 0u) {
      uint32_t left = need, bin = 255u;
      while (s_hist[bin] < left) left -= s_hist[bin--];
      s_pick[0] = bin;
      s_pick[1] = left;
    }
    __syncthreads();
    prefix |= s_pick[0] << shift;
    mask |= 255u << shift;
    need = s_pick[1];
    __syncthreads();
  }
  // need: tokens with the key `prefix` that are kept
  uint32_t at = 0u, ties = 0u;
  const bool any = a.keep > a.sink + a.recent;
  for (uint32_t j0 = 0; j0 < L; j0 += kEvThreads) {
    const uint32_t j = j0 + tid;
    bool take = false, tie = false;
    if (j < L) {
      if (j < lo || j >= hi) take = true;
      else if (any) {
        const uint32_t k = key_of(j);
        take = k > prefix;
        tie = k == prefix;
      }
    }
    uint32_t n;
    const uint32_t t = block_scan(tie ? 1u : 0u, s_wave, n);
    take = take || (tie && ties + t < need);
    ties += n;
    const uint32_t p = block_scan(take ? 1u : 0u, s_wave, n);
    if (take) out[at + p] = (int32_t)j;
    at += n;
  }
}

// One workgroup per (kv head, sequence), page by page in order: a token's new
// slot is never behind its old one, so a page's tokens are loaded before any
// slot that a later page still reads is written.
template <int D>
__global__ __launch_bounds__(D) void compact_kernel(CompactArgs a) {
  const uint32_t h = blockIdx.x, b = blockIdx.y, d = threadIdx.x, S = a.S;
  __shared__ f16 s_mean[D];
  const uint32_t L = seq_tokens(a.kv_indptr, a.kv_last_page_len, b, a.max_pages, S, a.error);
  const uint32_t n = L < a.keep ? L : a.keep;
  const int32_t* kept = a.kept + ((size_t)b * a.H + h) * a.stride;
  const uint32_t page0 = (uint32_t)a.kv_indptr[b], new0 = (uint32_t)a.new_indptr[b];
  const uint32_t meta0 = (uint32_t)a.meta_indptr[b];
  for (uint32_t p = 0; p * S < n; ++p) {
    const uint32_t c = n - p * S < S ? n - p * S : S;
    f16 k[kMaxPageSize], v[kMaxPageSize];
    float w[kMaxPageSize];
    for (uint32_t e = 0; e < c; ++e) {
      uint32_t j = (uint32_t)kept[p * S + e];
      j = j < L ? j : L - 1u;
      const uint32_t page = (uint32_t)a.kv_indices[page0 + j / S];
      k[e] = a.kv[elem_off(a.g, page, 0, h, j % S) + d];
      v[e] = a.kv[elem_off(a.g, page, 1, h, j % S) + d];
      if (a.weights != nullptr) w[e] = a.weights[((size_t)page * a.H + h) * S + j % S];
    }
    __syncthreads();
    const uint32_t to = (uint32_t)a.new_indices[new0 + p];
    f16 kmax = (f16)-65504.0f, kmin = (f16)65504.0f;  // as a bulk append's
    float sum = 0.f;
    for (uint32_t e = 0; e < c; ++e) {
      kmax = k[e] > kmax ? k[e] : kmax;
      kmin = k[e] < kmin ? k[e] : kmin;
      sum += (float)v[e];
      a.kv[elem_off(a.g, to, 0, h, e) + d] = k[e];
      a.kv[elem_off(a.g, to, 1, h, e) + d] = v[e];
      if (a.weights != nullptr && d == 0u) a.weights[((size_t)to * a.H + h) * S + e] = w[e];
    }
    const uint32_t mp = (uint32_t)a.meta_indices[meta0 + p / S];
    a.meta[elem_off(a.g, mp, 0, h, p % S) + d] = kmax;
    a.meta[elem_off(a.g, mp, 1, h, p % S) + d] = kmin;
    const f16 mean = r16(sum / (float)c);
    a.v_mean[((size_t)to * a.H + h) * D + d] = mean;
    s_mean[d] = mean;
    __syncthreads();
    if (d == 0u) {
      float acc = 0.f;
      for (int i = 0; i < D; ++i) acc += (float)s_mean[i] * (float)s_mean[i];
      f16 nrm = r16((float)__builtin_sqrt((double)acc));
      nrm = r16((float)nrm + 1e-8f);
      a.v_log_norm[(size_t)to * a.H + h] = r16((float)log((double)(float)nrm));
    }
    __syncthreads();
  }
}

}  // namespace

hipError_t launch_keep(const KeepArgs& a, uint32_t batch, hipStream_t s) {
  hipLaunchKernelGGL(keep_kernel, dim3(a.H, batch), dim3(kEvThreads), 0, s, a);
  return hipGetLastError();
}

hipError_t launch_compact(const CompactArgs& a, uint32_t batch, uint32_t head_dim, hipStream_t s) {
  const dim3 grid(a.H, batch);
  switch (head_dim) {
    case 64: hipLaunchKernelGGL(compact_kernel<64>, grid, dim3(64), 0, s, a); break;
    case 128: hipLaunchKernelGGL(compact_kernel<128>, grid, dim3(128), 0, s, a); break;
    default: hipLaunchKernelGGL(compact_kernel<256>, grid, dim3(256), 0, s, a); break;
  }
  return hipGetLastError();
}

}  // namespace aoakv
