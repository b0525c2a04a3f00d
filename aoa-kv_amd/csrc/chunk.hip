// Attention of a ragged batch of chunks of new tokens over the paged cache
// (chunk_attn.hpp), and the attention weight that each cached token received from
// them (gfx950).
#include "chunk_attn.hpp"

namespace aoakv {
namespace {

// ---------------------------------------------------------------- weights
constexpr uint32_t kSumsLeast = 4u;

// tanh(y): near 0, where 1 - 2 / (e^2y + 1) has no relative precision left, the
// odd series to y^9 (its next term is 0.0089 y^10 of the result: 1.5e-8 at y =
// 0.27)
__device__ inline float tanh_f32(float y) {
  const float y2 = y * y;
  float s = __builtin_fmaf(y2, 62.f / 2835.f, -17.f / 315.f);
  s = __builtin_fmaf(y2, s, 2.f / 15.f);
  s = __builtin_fmaf(y2, s, -1.f / 3.f);
  s = __builtin_fmaf(y * y2, s, y);
  const float e = __builtin_amdgcn_exp2f(y * (2.f * kLog2e));
  const float f = 1.f - 2.f * __builtin_amdgcn_rcpf(1.f + e);
  return __builtin_fabsf(y) < 0.27f ? s : f;
}

__device__ inline void store_weight(const ChunkArgs& a, const Seq& s, uint32_t b, uint32_t hk,
                                    int32_t j, float sum) {
  if (j >= s.L) return;
  const uint32_t p = div_page((uint32_t)j, a.page_rcp);
  const uint32_t page = (uint32_t)a.kv_indices[s.page0 + p];
  float* w = a.weights + ((size_t)page * a.H + hk) * a.S + ((uint32_t)j - p * a.S);
  const int32_t start = a.start != nullptr ? a.start[b] : s.off;
  *w = (j < start ? *w : 0.f) + sum;
}

// position of a row that counts nothing (no row of the call, or one that sees no
// key): outside of every range of positions
constexpr int32_t kNoPos = INT32_MIN;

// How the weights are cut.  BIG, where a sequence has many rows: a wave holds 2 x
// 32 keys (64 registers at D = 128; each halves the reads of query rows per
// product), tiles of 128 rows, two workgroups per CU.  Else the keys' own way
// from memory is what takes the time: 32 keys, tiles of 32 rows, and as many
// workgroups per CU with their keys in flight as registers allow (the last 32
// rows of 16384 tokens x 32 heads, one cache over and over: 2 per CU 38 us, 3 32,
// 4, spilling, 41).
template <int D, bool BIG>
struct SumShape {
  static constexpr int kSets = BIG && D != 256 ? 2 : 1;  // of 32 keys per wave
  static constexpr int32_t kKeys = 4 * 32 * kSets;       // of an item
  static constexpr int32_t kRows = BIG ? (D == 256 ? 64 : 128) : 32;  // of a tile
  static constexpr uint32_t kPerCu = BIG || D == 256 ? 2u : D == 128 ? 3u : 4u;
};
constexpr int32_t kMostKeys = 256;
constexpr uint32_t kMostSums = 4u;
constexpr uint32_t kWholeTiles = 4u;

// One workgroup's share of the items.  Scores are S = Q K^T: a wave holds its
// keys in registers (lane l: keys l % 32, + 32) and reads 32 query rows at a time
// from LDS, so a key's sum is a sum over a lane's own registers.  Each 32 rows are
// added up by themselves first: one chain of single additions over 16384 rows was
// 2e-6 off.
//
// Bound by the exponentials and the products where rows are many (4096 tokens of
// 16 heads of 128: 57 us, of 256 97, of 64 43; the products alone would take 29, 58
// and 14 at a large product's rate, the exponentials with their multiply and add
// about 20, so the two hardly overlap), and where they are few by the keys' way from
// memory, an item's after the other's: 32 rows after 16384 tokens x 32 heads 41 us,
// 3.3 TB/s, with caches in turn, and 32 where one stays in the memory-side cache; a
// decode step of 16 sequences 87, 3.8 TB/s.
template <int D, int MOD, bool BIG>
__global__ __launch_bounds__(kChThreads, (SumShape<D, BIG>::kPerCu)) void attn_weights_kernel(
    ChunkArgs a) {
  using Sh = PfShape<D>;
  using Cut_ = SumShape<D, BIG>;
  constexpr int32_t kRows = Cut_::kRows;
  __shared__ __attribute__((aligned(16))) char s_q0[kRows * Sh::kRowBytes];
  __shared__ __attribute__((aligned(16))) char s_q1[kRows * Sh::kRowBytes];
  // of a tile's rows: -lse in units of log 2 (-inf: the row counts nothing),
  // position, slope
  __shared__ __attribute__((aligned(16))) float s_neg[2][kRows];
  __shared__ __attribute__((aligned(16))) int32_t s_pos[2][kRows];
  __shared__ __attribute__((aligned(16))) float s_slope[2][kRows];
  __shared__ PlanLds s_plan;
  const int tid = threadIdx.x;
  const int lane = (int)__lane_id();
  const int wave = __builtin_amdgcn_readfirstlane(tid / kWave);
  const int g = lane / 32, c = lane % 32;

  constexpr int kSets = Cut_::kSets;
  constexpr int32_t kKeys = Cut_::kKeys;
  using By = ByKeys<kKeys, kRows>;
  Walk<By> w(a, s_plan);
  const uint64_t per_head = w.total(), units = per_head * a.H;
  const uint64_t share = share_of(a, units, kSumsLeast);
  uint64_t u = list_place() * share;
  const uint64_t u1 = min(u + share, units);
  if (u >= u1) {
    if (tid == 0 && !a.whole) reinterpret_cast<Cut*>(a.cuts)[list_place()].n = 0u;
    return;
  }
  w.seek(u, per_head);
  if (a.whole) {  // the items that begin in the share, whole
    if (w.at != 0u) {
      u += (uint32_t)By::item(a, w.seq(), w.x).count + kItemUnits - w.at;
      if (u >= u1) return;
      w.next();
    }
  } else if (tid == 0) {
    reinterpret_cast<Cut*>(a.cuts)[list_place()] = cut_of(w, list_place(), share);
  }

  constexpr int kWaveRows = kRows / 4;  // rows that a wave loads
  constexpr int kNI = kWaveRows / Sh::kRPI;
  constexpr int kRow32 = 32 * Sh::kRowBytes;
  const int lrow = lane / Sh::kCh, lslot = lane % Sh::kCh;
  // (offsets as in the attention kernel: with slopes they are made where they are used)
  constexpr bool kXor = (MOD & kBias) != 0;
  int q_off[kXor ? 1 : Sh::kKS];
#pragma unroll
  for (int s8 = 0; s8 < (kXor ? 1 : Sh::kKS); ++s8) q_off[s8] = tile_off<D>(c, 2 * s8 + g);
  const float scale = MOD == 0 ? a.sm_scale * kLog2e : 1.f;
  const float cap2 = a.soft_cap * kLog2e;
  const float cap_in = MOD & kCap ? a.sm_scale / a.soft_cap : 0.f;
  const int32_t window = a.window != 0u ? (int32_t)a.window : 1 << 30;

  for (;;) {
    const Seq s = w.seq();
    const Item item = By::item(a, s, w.x);
    const uint32_t hk = w.h;
    const uint32_t ue = (uint32_t)item.count + kItemUnits;
    const uint32_t ua = w.at, ub = a.whole ? ue : (uint32_t)min((uint64_t)ue, ua + (u1 - u));
    const int32_t t0 = max((int32_t)(ua - kItemUnits), 0), t1 = max((int32_t)(ub - kItemUnits), 0);
    const int32_t R = s.n * group(a);
    constexpr int32_t kWaveKeys = 32 * kSets;
    const int32_t k0 = w.x * kKeys + wave * kWaveKeys;  // the wave's first key

    half8 kf[kSets][Sh::kKS];
#pragma unroll
    for (int z = 0; z < kSets; ++z) {
      const uint32_t j = (uint32_t)min(k0 + 32 * z + c, s.L - 1), p = div_page(j, a.page_rcp);
      const uint32_t page = (uint32_t)a.kv_indices[s.page0 + p];
      const f16* k = a.kv + elem_off(a.g, page, 0, hk, j - p * a.S) + 8 * g;
#pragma unroll
      for (int s8 = 0; s8 < Sh::kKS; ++s8) kf[z][s8] = *reinterpret_cast<const half8*>(k + 16 * s8);
    }

    // row r of the packed rows lies at r * D + token * (Hq - G) * D of this
    const f16* q0 = a.q + ((size_t)s.q0 * a.Hq + (size_t)hk * a.G) * D;
    const uint32_t tok_step = (a.Hq - a.G) * D;
    auto load_tile = [&](char* buf, int32_t tile) {
#pragma unroll
      for (int i = 0; i < kNI; ++i) {
        const int tr = kWaveRows * wave + Sh::kRPI * i + lrow;
        const int32_t r = min(tile * kRows + tr, R - 1);
        load_lds16(q0 + (size_t)(uint32_t)r * D + (size_t)(uint32_t)token_of(a, r) * tok_step +
                       8 * (lslot ^ k_swz<Sh::kCh>(tr)),
                   buf + (kWaveRows * wave + Sh::kRPI * i) * Sh::kRowBytes);
      }
    };
    // what s_neg, s_pos and s_slope get: fetched a tile ahead, stored after the
    // tile before it is done (waiting for them no earlier)
    struct RowData {
      float lse, slope;
      int32_t pos;
      bool live;
    };
    auto fetch_row = [&](int32_t tile) {
      RowData d{};
      if (tid < kRows) {
        const int32_t r = tile * kRows + tid;
        const Row row = row_of(a, hk, min(r, R - 1));
        d.lse = a.lse[(size_t)(s.q0 + row.tok) * a.Hq + row.h];
        if constexpr (MOD & kBias) d.slope = a.slopes[row.h];
        d.pos = s.off + row.tok;
        d.live = r < R;
      }
      return d;
    };
    auto store_rows = [&](int v, const RowData& d) {
      if (tid < kRows) {
        const bool counts = d.live && d.lse != -INFINITY;
        s_neg[v][tid] = counts ? -d.lse * kLog2e : -INFINITY;
        s_pos[v][tid] = counts ? d.pos : kNoPos;
        if constexpr (MOD & kBias) s_slope[v][tid] = d.slope * kLog2e;
      }
    };
    // rows 32 half .. + 31 of a tile: their query fragments, -lse, and what MOD
    // and the masks need
    struct Rows {
      float neg[16], slope[16];
      int32_t pos[16];
    };
    auto read_q = [&](const lds_char* sQ, int half, half8 (&q)[Sh::kKS]) {
      if constexpr (kXor) asm volatile("" : "+v"(q_off[0]));
#pragma unroll
      for (int s8 = 0; s8 < Sh::kKS; ++s8)
        q[s8] = *reinterpret_cast<const __attribute__((address_space(3))) half8*>(
            sQ + (kXor ? q_off[0] ^ (32 * s8) : q_off[s8 % Sh::kKS]) + half * kRow32);
    };
    auto read_quad = [&](int v, int half, Rows& x, bool pos, int q4) {
      const int at = 32 * half + 8 * q4 + 4 * g;  // rows crow(4 q4, g) ..
      const float4 n = *reinterpret_cast<const float4*>(&s_neg[v][at]);
      x.neg[4 * q4] = n.x, x.neg[4 * q4 + 1] = n.y, x.neg[4 * q4 + 2] = n.z,
      x.neg[4 * q4 + 3] = n.w;
      if (MOD & kBias || pos) {
        const int4 y = *reinterpret_cast<const int4*>(&s_pos[v][at]);
        x.pos[4 * q4] = y.x, x.pos[4 * q4 + 1] = y.y, x.pos[4 * q4 + 2] = y.z,
        x.pos[4 * q4 + 3] = y.w;
      }
      if constexpr (MOD & kBias) {
        const float4 y = *reinterpret_cast<const float4*>(&s_slope[v][at]);
        x.slope[4 * q4] = y.x, x.slope[4 * q4 + 1] = y.y, x.slope[4 * q4 + 2] = y.z,
        x.slope[4 * q4 + 3] = y.w;
      }
    };
    auto read_rows = [&](int v, int half, Rows& x, bool pos) {
#pragma unroll
      for (int q4 = 0; q4 < 4; ++q4) read_quad(v, half, x, pos, q4);
    };
    // probability of register i of a product
    auto weight = [&](float t, const Rows& x, int i, int32_t key) {
      if constexpr (MOD & kCap) t = cap2 * tanh_f32(t * cap_in);
      else if constexpr (MOD != 0) t *= a.sm_scale * kLog2e;
      if constexpr (MOD & kBias)
        t = __builtin_fmaf(-x.slope[i], __builtin_fabsf((float)(x.pos[i] - key)), t);
      return __builtin_amdgcn_exp2f(__builtin_fmaf(t, scale, x.neg[i]));
    };
    float sum[kSets] = {};
    // A tile that the wave's keys are seen by whole.  The products of 32 rows and
    // a set of keys follow each other, and the exponentials of one are issued
    // between the matrix instructions of the next (held there by the scheduling
    // barriers): with all products first, the two waves of a SIMD did the same
    // thing at the same time and neither unit was busy more than half.
    auto whole_tile = [&](const lds_char* sQ, int v) {
      constexpr int kPer = 16 / Sh::kKS;  // elements per matrix instruction
      constexpr int kN = kRows / 32 * kSets;  // products
      // (slopes and positions take the registers of a buffer, and at D = 256 are
      // read four rows at a time: none is spilled)
      constexpr int kQ = MOD & kBias ? 1 : 2;
      constexpr bool kQuads = MOD & kBias && D == 256;
      half8 q[kQ][Sh::kKS];
      Rows x;
      read_q(sQ, 0, q[0]);
      floatx16 acc[2];
      float part = 0.f;
#pragma unroll
      for (int n = 0; n <= kN; ++n) {  // product n, exponentials of product n - 1
        const int half = n / kSets, z = n % kSets, pz = (n + kSets - 1) % kSets;
        if (kQ == 2 && n < kN && z == 0 && half + 1 < kRows / 32)
          read_q(sQ, half + 1, q[(half + 1) % kQ]);
        if (kQ == 1 && n > 0 && n < kN && z == 0) read_q(sQ, half, q[0]);
        if (n > 0 && kQuads) read_quad(v, (n - 1) / kSets, x, false, 0);
        if (n > 0 && !kQuads && pz == 0) read_rows(v, (n - 1) / kSets, x, false);
        if (n < kN) acc[n % 2] = floatx16{};
#pragma unroll
        for (int s8 = 0; s8 < Sh::kKS; ++s8) {
          if (n < kN) acc[n % 2] = mfma32(q[half % kQ][s8], kf[z][s8], acc[n % 2]);
          if (n > 0) {
            const int q4 = s8 * kPer / 4 + 1;  // (needed four elements on)
            if (kQuads && s8 * kPer % 4 == 0 && q4 < 4) read_quad(v, (n - 1) / kSets, x, false, q4);
#pragma unroll
            for (int e = 0; e < kPer; ++e)
              part += weight(acc[(n + 1) % 2][s8 * kPer + e], x, s8 * kPer + e,
                             k0 + 32 * pz + c);
          }
          if (n > 0 && n < kN) __builtin_amdgcn_sched_barrier(0);
        }
        if (n > 0) {
          sum[pz] += part;
          part = 0.f;
        }
      }
    };
    // ... or in part: a key is seen from a range of positions (one subtraction and
    // one unsigned comparison per element; a chain of && became branches here and
    // took 30 us per tile)
    auto masked_half = [&](const lds_char* sQ, int v, int half, int32_t p0, int32_t p1) {
      half8 q[Sh::kKS];
      Rows x;
      read_q(sQ, half, q);
      read_rows(v, half, x, true);
#pragma unroll
      for (int z = 0; z < kSets; ++z) {
        const int32_t kz = k0 + 32 * z;  // (none of these keys is seen)
        if (kz >= s.prefix && ((a.causal && kz > p1) || p0 - (kz + 31) >= window)) continue;
        floatx16 acc = floatx16{};
#pragma unroll
        for (int s8 = 0; s8 < Sh::kKS; ++s8) acc = mfma32(q[s8], kf[z][s8], acc);
        const int32_t key = kz + c;
        const int32_t from = key >= s.L                      ? INT32_MAX
                             : key < s.prefix || !a.causal ? kNoPos + 1
                                                             : key;
        const int32_t to = key >= s.L ? INT32_MAX
                           : key < s.prefix ? INT32_MAX
                                            : key + (window - 1);
        const uint32_t span = (uint32_t)to - (uint32_t)from;
        float part = 0.f;
#pragma unroll
        for (int i = 0; i < 16; ++i) {
          const float p = weight(acc[i], x, i, key);
          part += (uint32_t)x.pos[i] - (uint32_t)from <= span ? p : 0.f;
        }
        sum[z] += part;
      }
    };

    __syncthreads();  // the item before is done with the buffers
    if (t0 < t1) {
      const RowData d = fetch_row(item.tile(t0));
      load_tile(s_q0, item.tile(t0));
      store_rows(0, d);
    }
    for (int32_t it = t0; it < t1; it += 2) {
#pragma unroll
      for (int v = 0; v < 2; ++v) {
        const int32_t i = it + v;
        if (i >= t1) break;  // uniform
        const lds_char* sQ = (const lds_char*)(v == 0 ? s_q0 : s_q1);
        asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
        __syncthreads();
        RowData next{};
        if (i + 1 < t1) {
          next = fetch_row(item.tile(i + 1));
          load_tile(v == 0 ? s_q1 : s_q0, item.tile(i + 1));
        }
        // the tile's rows at positions p0 .. p1: all see all of the wave's keys,
        // or some see some
        const int32_t r0 = item.tile(i) * kRows;
        const int32_t p0 = s.off + token_of(a, r0),
                      p1 = s.off + token_of(a, min(r0 + kRows - 1, R - 1));
        if (r0 + kRows <= R && k0 + kWaveKeys <= s.L &&
            (k0 + kWaveKeys <= s.prefix ||
             ((!a.causal || k0 + kWaveKeys - 1 <= p0) && p1 - k0 < window))) {
          whole_tile(sQ, v);
        } else if (k0 < s.prefix ||
                   ((!a.causal || k0 <= p1) && p0 - (k0 + kWaveKeys - 1) < window)) {
#pragma nounroll
          for (int half = 0; half < kRows / 32; ++half) {
            const int32_t rh = r0 + 32 * half;
            if (rh >= R) break;
            masked_half(sQ, v, half, s.off + token_of(a, rh),
                        s.off + token_of(a, min(rh + 31, R - 1)));
          }
        }
        if (i + 1 < t1) store_rows(v ^ 1, next);
      }
    }
    float* part =
        a.parts + (2u * (size_t)list_place() + (ua == 0u ? 1u : 0u)) * kMostKeys + wave * kWaveKeys;
#pragma unroll
    for (int z = 0; z < kSets; ++z) {
      const float x = pair_sum(sum[z]);
      if (g != 0) continue;
      if (ua == 0u && ub == ue) store_weight(a, s, w.b, hk, k0 + 32 * z + c, x);
      else part[32 * z + c] = x;
    }
    u += ub - ua;
    if (u >= u1) return;
    w.next();
  }
}

// Joins an item's parts: a thread per key.
__global__ __launch_bounds__(kMostKeys) void weights_join_kernel(ChunkArgs a) {
  const Cut cut = reinterpret_cast<const Cut*>(a.cuts)[blockIdx.x + 1u];
  if (cut.n == 0u) return;
  float sum = 0.f;
  for (uint32_t i = 0; i < cut.n; ++i) sum += a.parts[cut.slot(i) * kMostKeys + threadIdx.x];
  store_weight(a, load_seq(a, cut.b), cut.b, cut.h,
               cut.x * (int32_t)blockDim.x + (int32_t)threadIdx.x, sum);
}

template <int D, bool BIG>
hipError_t launch_sums(const ChunkArgs& args, hipStream_t s) {
  using Shape = SumShape<D, BIG>;
  const uint64_t G = args.Hq / args.H;
  const uint64_t tiles = (args.T * G) / Shape::kRows + 2u;  // of an item, at most
  const uint32_t n = workgroups(
      args, (uint64_t)args.B * (((uint64_t)args.max_pages * args.S) / Shape::kKeys + 1u), tiles,
      kCus * Shape::kPerCu, kSumsLeast);
  ChunkArgs a = with_rcps(args, n);
  // Items of a few tiles are not worth cutting, nor a launch to join them: 32, 64,
  // 128, 256 and 512 rows of one sequence of 8000 keys, 8 kv heads, whole / cut 12 /
  // 14, 13 / 17, 12 / 16, 15 / 18 and 30 / 25 us.  The bound is the call's rows,
  // because a sequence's are known on the device alone: a decode step of 16
  // sequences of 4 heads a group is whole (57.5; cut 59.2) and one of 17 is cut (69.6;
  // whole 67.5), 64 273 (270).
  a.whole = tiles <= kWholeTiles ? 1u : 0u;
  const dim3 grid(n), block(kChThreads);
  switch ((a.soft_cap > 0.f ? kCap : 0) | (a.slopes != nullptr ? kBias : 0)) {
    case 0: hipLaunchKernelGGL((attn_weights_kernel<D, 0, BIG>), grid, block, 0, s, a); break;
    case kCap:
      hipLaunchKernelGGL((attn_weights_kernel<D, kCap, BIG>), grid, block, 0, s, a);
      break;
    case kBias:
      hipLaunchKernelGGL((attn_weights_kernel<D, kBias, BIG>), grid, block, 0, s, a);
      break;
    default:
      hipLaunchKernelGGL((attn_weights_kernel<D, (kCap | kBias), BIG>), grid, block, 0, s, a);
      break;
  }
  if (hipError_t e = hipGetLastError(); e != hipSuccess || a.whole) return e;
  hipLaunchKernelGGL(weights_join_kernel, dim3(n - 1u), dim3(Shape::kKeys), 0, s, a);
  return hipGetLastError();
}

// The BIG cut (SumShape) goes by the batch's rows per sequence, the longest being
// known on the device alone.  4 sequences of 4096 keys, 8 kv heads, small / big: 64
// rows each 20.6 / 22.6 us, 128 22 / 26, 256 30 / 31, 512 38 / 40, 1024 59 / 59, 2048
// 100 / 88, 4096 172 / 153.  The border is below their crossing because an average
// of 256 is often a long chunk among short ones (one of 4096 rows beside 31 of one:
// 113 / 94, and with 129 on average still the small cut's).
template <int D>
hipError_t launch_sums(const ChunkArgs& a, hipStream_t s) {
  const uint64_t rows = (uint64_t)a.T * (a.Hq / a.H);
  return rows >= 256u * (uint64_t)a.B ? launch_sums<D, true>(a, s) : launch_sums<D, false>(a, s);
}

}  // namespace

size_t chunk_attn_workspace(uint32_t T, uint32_t B, uint32_t Hq, uint32_t H, uint32_t head_dim,
                            uint32_t max_pages, uint32_t S) {
  ChunkArgs a{};
  a.T = T;
  a.B = B;
  a.Hq = Hq;
  a.H = H;
  a.max_pages = max_pages;
  a.S = S;
  const uint32_t slots = head_dim == 256u ? attn_slots<256>() : attn_slots<128>();
  const uint32_t n = lists_items(a, slots) ? slots : share_workgroups(a, slots);
  return kCutBytes + list_bytes(a, slots) +
         2u * (size_t)n * part_floats((int)head_dim) * sizeof(float);
}
size_t attn_weights_workspace() {
  return kCutBytes + 2u * kCus * kMostSums * kMostKeys * sizeof(float);
}

hipError_t launch_chunk_attn(const ChunkArgs& a, uint32_t head_dim, hipStream_t s) {
  switch (head_dim) {
    case 64: return launch_attn<64, false>(a, s);
    case 128: return launch_attn<128, false>(a, s);
    default: return launch_attn<256, false>(a, s);
  }
}

hipError_t launch_attn_weights(const ChunkArgs& a, uint32_t head_dim, hipStream_t s) {
  switch (head_dim) {
    case 64: return launch_sums<64>(a, s);
    case 128: return launch_sums<128>(a, s);
    default: return launch_sums<256>(a, s);
  }
}

}  // namespace aoakv
