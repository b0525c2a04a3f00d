// Eviction from the paged cache (gfx950): which tokens each kv head keeps by
// the attention weight they received, and the cache packed down to them with
// its page statistics.
#include <type_traits>

#include "kernels.hpp"

namespace aoakv {
namespace {

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

// ---------------------------------------------------------------- choice
constexpr uint32_t kKeepThreads = 1024;
constexpr uint32_t kKeepWaves = kKeepThreads / kWave;
constexpr uint32_t kRun = 4u * kKeepThreads;  // tokens a workgroup takes at once, 4 per thread
constexpr uint32_t kBins = 2048u, kCopies = 4u;

// One workgroup per (kv head, sequence).  Two weights are ordered as the
// integers that order_key makes of them (NaN lowest, -0 as 0); the first `sink`
// and last `recent` tokens have the largest integer of all, so the choice is
// that of the `keep` largest, ties to the lower position.  Eleven bits at a time
// from the top, a histogram of the tokens that agree so far finds where the
// last kept one lies, until that bin is kept whole; then a token's place in the
// row is the number of larger tokens before it plus that of kept equal ones.
//
// Bound by the chain of steps in one workgroup (the weights are read once:
// they are held in registers, 4 x RUNS per thread, and only longer sequences
// load them again in each step).  2048 of up to 32768 tokens, 4 x 32 heads: 143
// us with a token per thread and loop trip, 37 from registers in four steps of
// 8 bits, 22 so (24 with caches in turn).  The histogram has 4 copies, by lane, because
// equal weights (many are exactly 0) would otherwise add to one word one after the
// other.  Slots behind a sequence's end count as the lowest weight in the first step,
// so 5000 tokens take what 32768 do (22 us; up to 4096, with RUNS = 1, 6.6 to 7.8).
template <int RUNS, bool VEC>
__global__ __launch_bounds__(kKeepThreads) void keep_kernel(KeepArgs a) {
  __shared__ uint32_t s_hist[kBins * kCopies];
  __shared__ uint32_t s_wave[RUNS][kKeepWaves];
  __shared__ uint32_t s_pick[3];
  const uint32_t h = blockIdx.x, b = blockIdx.y, tid = threadIdx.x;
  const uint32_t lane = __lane_id(), wave = tid / kWave;
  const uint32_t L = seq_tokens(a.kv_indptr, a.kv_last_page_len, b, a.max_pages, a.S, a.error);
  const int32_t* ids = a.kv_indices + (uint32_t)a.kv_indptr[b];
  int32_t* out = a.kept + ((size_t)b * a.H + h) * a.stride;
  if (L <= a.keep) {
    for (uint32_t j = tid; j < L; j += kKeepThreads) out[j] = (int32_t)j;
    return;
  }
  const uint32_t lo = a.sink, hi = L - a.recent;  // the tokens that compete (lo <= hi)
  const uint32_t S = a.S, segment = kRun * RUNS;

  uint32_t key[RUNS][4];
  auto load = [&](uint32_t seg) {
    float w[RUNS][4];
    if constexpr (VEC) {  // 4 tokens of a thread lie in one page
      uint32_t page[RUNS], slot[RUNS];
#pragma unroll
      for (int i = 0; i < RUNS; ++i) {
        uint32_t j = seg + (uint32_t)i * kRun + 4u * tid;
        j = j < L ? j : 0u;
        const uint32_t p = div_page(j, a.page_rcp);
        slot[i] = j - p * S;
        page[i] = (uint32_t)ids[p];
      }
#pragma unroll
      for (int i = 0; i < RUNS; ++i) {
        const float4 x = *reinterpret_cast<const float4*>(
            a.weights + ((size_t)page[i] * a.H + h) * S + slot[i]);
        w[i][0] = x.x, w[i][1] = x.y, w[i][2] = x.z, w[i][3] = x.w;
      }
    } else {
#pragma unroll
      for (int i = 0; i < RUNS; ++i)
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          uint32_t j = seg + (uint32_t)i * kRun + 4u * tid + (uint32_t)e;
          j = j < L ? j : 0u;
          const uint32_t p = div_page(j, a.page_rcp);
          w[i][e] = a.weights[((size_t)(uint32_t)ids[p] * a.H + h) * S + (j - p * S)];
        }
    }
#pragma unroll
    for (int i = 0; i < RUNS; ++i)
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        const uint32_t j = seg + (uint32_t)i * kRun + 4u * tid + (uint32_t)e;
        const float x = w[i][e] + 0.f;
        uint32_t k = x == x ? order_key(x) : 0u;
        k = j < lo || j >= hi ? 0xFFFFFFFFu : k;
        key[i][e] = j < L ? k : 0u;  // (behind every token, so never kept)
      }
  };

  uint32_t need = a.keep, prefix = 0u, mask = 0u;
  const bool one = L <= segment;
  if (one) load(0u);
  for (int step = 0; step < 3; ++step) {
    const int shift = step == 0 ? 21 : step == 1 ? 10 : 0;
    const uint32_t digit = step == 2 ? 1023u : 2047u;
#pragma unroll
    for (uint32_t i = 0; i < kBins * kCopies / kKeepThreads; ++i)
      s_hist[i * kKeepThreads + tid] = 0u;
    __syncthreads();
    for (uint32_t seg = 0; seg < L; seg += segment) {
      if (!one) load(seg);
#pragma unroll
      for (int i = 0; i < RUNS; ++i)
#pragma unroll
        for (int e = 0; e < 4; ++e)
          if ((key[i][e] & mask) == prefix)
            atomicAdd(&s_hist[(key[i][e] >> shift & digit) * kCopies + lane % kCopies], 1u);
    }
    __syncthreads();
    // thread t has bins 2047 - 2 t and the one below
    const uint4 x = reinterpret_cast<const uint4*>(s_hist)[kBins - 1u - 2u * tid];
    const uint4 y = reinterpret_cast<const uint4*>(s_hist)[kBins - 2u - 2u * tid];
    const uint32_t n0 = x.x + x.y + x.z + x.w, n1 = y.x + y.y + y.z + y.w;
    uint32_t upto = n0 + n1;
#pragma unroll
    for (uint32_t d = 1; d < (uint32_t)kWave; d <<= 1) {
      const uint32_t z = __shfl_up(upto, d);
      if (lane >= d) upto += z;
    }
    if (lane == kWave - 1u) s_wave[0][wave] = upto;
    __syncthreads();
    for (uint32_t i = 0; i < kKeepWaves; ++i) upto += i < wave ? s_wave[0][i] : 0u;
    const uint32_t before = upto - n0 - n1;
    if (before < need && need <= upto) {
      const bool second = need > before + n0;
      s_pick[0] = kBins - 1u - 2u * tid - (second ? 1u : 0u);
      s_pick[1] = need - before - (second ? n0 : 0u);
      s_pick[2] = second ? n1 : n0;
    }
    __syncthreads();
    prefix |= s_pick[0] << shift;
    mask |= digit << shift;
    need = s_pick[1];
    if (need == s_pick[2]) break;  // the bin is kept whole
  }

  // kept: the tokens above `prefix` under `mask`, and the first `need` at it
  uint32_t above = 0u, ties = 0u;  // in the runs before
  for (uint32_t seg = 0; seg < L; seg += segment) {
    if (!one) load(seg);
    uint32_t mine[RUNS], upto[RUNS];  // tokens above (low half) and ties of the run
#pragma unroll
    for (int i = 0; i < RUNS; ++i) {
      mine[i] = 0u;
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        const uint32_t k = key[i][e] & mask;
        mine[i] += k > prefix ? 1u : k == prefix ? 1u << 16 : 0u;
      }
      upto[i] = mine[i];
    }
#pragma unroll
    for (uint32_t d = 1; d < (uint32_t)kWave; d <<= 1)
#pragma unroll
      for (int i = 0; i < RUNS; ++i) {
        const uint32_t x = __shfl_up(upto[i], d);
        if (lane >= d) upto[i] += x;
      }
    __syncthreads();
    if (lane == kWave - 1u) {
#pragma unroll
      for (int i = 0; i < RUNS; ++i) s_wave[i][wave] = upto[i];
    }
    __syncthreads();
#pragma unroll
    for (int i = 0; i < RUNS; ++i) {
      uint32_t before = 0u, all = 0u;
#pragma unroll
      for (uint32_t x = 0; x < kKeepWaves; ++x) {
        before += x < wave ? s_wave[i][x] : 0u;
        all += s_wave[i][x];
      }
      before += upto[i] - mine[i];
      uint32_t n = above + (before & 0xFFFFu), t = ties + (before >> 16);
      if (mine[i] != 0u) {
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          const uint32_t j = seg + (uint32_t)i * kRun + 4u * tid + (uint32_t)e;
          const uint32_t k = key[i][e] & mask;
          if (k > prefix || (k == prefix && t < need))
            out[n + (t < need ? t : need)] = (int32_t)j;
          n += k > prefix ? 1u : 0u;
          t += k == prefix ? 1u : 0u;
        }
      }
      above += all & 0xFFFFu;
      ties += all >> 16;
    }
  }
}

// ---------------------------------------------------------------- packing
// threads: in place, where one workgroup takes all of a head, many; else few, so
// that the steps of several workgroups overlap on a CU (2048 tokens of 4 x 32
// heads to new pages, 285 MB: 512 threads 79 us, 256 68; 59 with K and V as code of
// their own below, 4.8 TB/s, and 70 to 73 with caches in turn).  In place 66 where
// there are many heads; 2048 of 16384 tokens of one sequence at 32 and 8 heads 33 and
// 30 us, to new pages 16 and 9.
constexpr int kPackThreadsInPlace = 512, kPackThreads = 256;

// A workgroup takes steps of K or of V of one (kv head, sequence): each lane
// group of D / 8 lanes holds MOST tokens at a time (whole pages where a page is
// shorter, else one page), so all of a step's loads are in flight together and
// a page's statistics need no other group.  In place one workgroup takes a
// head's steps in order: a token's new slot is never behind its old one, so
// a step that has been loaded whole overwrites no later step's tokens.  Else
// the steps of a head are dealt to gridDim.z / 2 workgroups.
template <int D, int MOST, int THREADS>
__global__ __launch_bounds__(THREADS) void compact_kernel(CompactArgs a) {
  constexpr uint32_t kLanes = D / 8, kGroups = THREADS / kLanes;
  constexpr uint32_t kTokens = kGroups * MOST;  // of a step, at most
  __shared__ uint32_t s_page[kTokens], s_slot[kTokens];
  const uint32_t h = blockIdx.x, b = blockIdx.y, which = blockIdx.z % 2u;
  const uint32_t tid = threadIdx.x, l = tid % kLanes, grp = tid / kLanes, S = a.S;
  const uint32_t L = seq_tokens(a.kv_indptr, a.kv_last_page_len, b, a.max_pages, S, a.error);
  const uint32_t n = L < a.keep ? L : a.keep;
  const int32_t* kept = a.kept + ((size_t)b * a.H + h) * a.stride;
  const int32_t* ids = a.kv_indices + (uint32_t)a.kv_indptr[b];
  const int32_t* new_ids = a.new_indices + (uint32_t)a.new_indptr[b];
  const int32_t* meta_ids = a.meta_indices + (uint32_t)a.meta_indptr[b];
  const uint32_t pages = S < (uint32_t)MOST ? (uint32_t)MOST / S : 1u;  // per group
  const uint32_t per = pages * S, step = kGroups * per;

  for (uint32_t j0 = blockIdx.z / 2u * step; j0 < n; j0 += gridDim.z / 2u * step) {
    __syncthreads();  // the step before is stored
    float w[(kTokens + THREADS - 1) / THREADS];
#pragma unroll
    for (uint32_t i = 0; i < kTokens; i += THREADS) {
      const uint32_t t = i + tid;
      if (t < step && j0 + t < n) {
        uint32_t j = (uint32_t)kept[j0 + t];
        j = j < L ? j : L - 1u;
        const uint32_t p = div_page(j, a.page_rcp);
        const uint32_t page = (uint32_t)ids[p], slot = j - p * S;
        s_page[t] = page;
        s_slot[t] = slot;
        if (which == 0u && a.weights != nullptr)
          w[i / THREADS] = a.weights[((size_t)page * a.H + h) * S + slot];
      }
    }
    __syncthreads();
    const uint32_t first = j0 + grp * per;  // the group's first token
    const uint32_t c = first < n ? (n - first < per ? n - first : per) : 0u;
    H8 x[MOST];
#pragma unroll
    for (uint32_t t = 0; t < (uint32_t)MOST; ++t)
      if (t < c)
        x[t] = ld16(a.kv + elem_off(a.g, s_page[grp * per + t], which, h, s_slot[grp * per + t]) +
                    l * kVec);
    const uint32_t p0 = div_page(first, a.page_rcp);  // the group's first new page
    uint32_t to = c != 0u ? (uint32_t)new_ids[p0] : 0u;
    if (a.in_place) {  // every load of the step is back before its first store
      asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
      __syncthreads();
    }
    H8 kmax, kmin, mean;
    float sum[kVec];
    // (K and V each with their own code: half as many instructions to fetch)
    auto store = [&](auto is_v) {
      constexpr bool kV = is_v.value;
      uint32_t e = 0u, p = p0;
#pragma unroll
      for (uint32_t t = 0; t < (uint32_t)MOST; ++t) {
        if (t >= c) continue;
        if (e == 0u) {
#pragma unroll
          for (int j = 0; j < kVec; ++j) {
            kmax.v[j] = (f16)-65504.0f;  // as a bulk append starts a page
            kmin.v[j] = (f16)65504.0f;
            sum[j] = 0.f;
          }
        }
#pragma unroll
        for (int j = 0; j < kVec; ++j) {
          if constexpr (!kV) {
            kmax.v[j] = x[t].v[j] > kmax.v[j] ? x[t].v[j] : kmax.v[j];
            kmin.v[j] = x[t].v[j] < kmin.v[j] ? x[t].v[j] : kmin.v[j];
          } else {
            sum[j] = sum[j] + (float)x[t].v[j];
          }
        }
        st16(a.kv + elem_off(a.g, to, which, h, e) + l * kVec, x[t]);
        if (++e == S || t + 1u == c) {  // the page's last token
          if constexpr (!kV) {
            const uint32_t mp = div_page(p, a.page_rcp), me = p - mp * S;
            const uint32_t page = (uint32_t)meta_ids[mp];
            st16(a.meta + elem_off(a.g, page, 0, h, me) + l * kVec, kmax);
            st16(a.meta + elem_off(a.g, page, 1, h, me) + l * kVec, kmin);
          } else {
#pragma unroll
            for (int j = 0; j < kVec; ++j) mean.v[j] = r16(sum[j] / (float)e);
            st16(a.v_mean + ((size_t)to * a.H + h) * D + l * kVec, mean);
          }
          e = 0u;
          ++p;
          if (t + 1u < c) to = (uint32_t)new_ids[p];
        }
      }
    };
    if (which == 0u) store(std::false_type{});
    else store(std::true_type{});
    // the log-norms (in a loop of their own: once per token above would be
    // most of the code); several pages' means are this lane's own stores
    if (which == 1u) {
#pragma nounroll
      for (uint32_t q = 0; q * S < c; ++q) {
        const size_t at = (size_t)(pages == 1u ? to : (uint32_t)new_ids[p0 + q]) * a.H + h;
        if (pages != 1u) mean = ld16(a.v_mean + at * D + l * kVec);
        f16 norm;
        if constexpr (kLanes == (uint32_t)kLanesPerRow) norm = log_norm_row(mean);
        else norm = grp_log_norm<kLanes>(mean, l);
        if (l == 0u) a.v_log_norm[at] = norm;
      }
    }
    if (which == 0u && a.weights != nullptr) {
#pragma unroll
      for (uint32_t i = 0; i < kTokens; i += THREADS) {
        const uint32_t t = i + tid;
        if (t < step && j0 + t < n) {
          const uint32_t q = div_page(j0 + t, a.page_rcp);
          a.weights[((size_t)(uint32_t)new_ids[q] * a.H + h) * S + (j0 + t - q * S)] =
              w[i / THREADS];
        }
      }
    }
  }
}

template <int D, int THREADS>
void launch_pack(const CompactArgs& a, uint32_t batch, hipStream_t s) {
  const uint32_t most = a.S > 16u ? 32u : 16u;
  const uint32_t step = THREADS / (D / 8) * (a.S < most ? most / a.S * a.S : a.S);
  const uint64_t steps = ((uint64_t)a.keep + step - 1u) / step;
  const uint32_t z = a.in_place ? 1u : (uint32_t)(steps < 16384u ? steps : 16384u);
  const dim3 grid(a.H, batch, 2u * z), block(THREADS);
  if (most == 16u) hipLaunchKernelGGL((compact_kernel<D, 16, THREADS>), grid, block, 0, s, a);
  else hipLaunchKernelGGL((compact_kernel<D, 32, THREADS>), grid, block, 0, s, a);
}
template <int D>
void launch_pack(const CompactArgs& a, uint32_t batch, hipStream_t s) {
  if (a.in_place) launch_pack<D, kPackThreadsInPlace>(a, batch, s);
  else launch_pack<D, kPackThreads>(a, batch, s);
}

uint32_t rcp_of(uint32_t S) { return S == 1u ? 0u : (uint32_t)((1ull << 32) / S) + 1u; }

}  // namespace

hipError_t launch_keep(const KeepArgs& args, uint32_t batch, hipStream_t s) {
  KeepArgs a = args;
  a.page_rcp = rcp_of(a.S);
  const dim3 grid(a.H, batch), block(kKeepThreads);
  // 4096 tokens per sequence at most: 4 per thread; else 32
  const bool few = (uint64_t)a.max_pages * a.S <= kRun;
  const bool vec = a.S % 4u == 0u && reinterpret_cast<uintptr_t>(a.weights) % 16u == 0u;
  if (few && vec) hipLaunchKernelGGL((keep_kernel<1, true>), grid, block, 0, s, a);
  else if (few) hipLaunchKernelGGL((keep_kernel<1, false>), grid, block, 0, s, a);
  else if (vec) hipLaunchKernelGGL((keep_kernel<8, true>), grid, block, 0, s, a);
  else hipLaunchKernelGGL((keep_kernel<8, false>), grid, block, 0, s, a);
  return hipGetLastError();
}

hipError_t launch_compact(const CompactArgs& args, uint32_t batch, uint32_t head_dim,
                          hipStream_t s) {
  CompactArgs a = args;
  a.page_rcp = rcp_of(a.S);
  switch (head_dim) {
    case 64: launch_pack<64>(a, batch, s); break;
    case 128: launch_pack<128>(a, batch, s); break;
    default: launch_pack<256>(a, batch, s); break;
  }
  return hipGetLastError();
}

}  // namespace aoakv
