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
//
// Rows.  A kv head's queries of one sequence are packed token by token, the
// group's heads of a token side by side: row r is token r / G, head r % G.  A
// tile of K/V in LDS then serves the whole group, and a few tokens fill a tile
// of rows better.
//
// Work.  An item is 128 rows (attention) or 128 keys (weights) of one kv head
// and sequence, and walks tiles of 64 keys (or rows) that any of its rows sees
// (or that see any of its keys).  Lengths are known on the device alone, so
// every workgroup adds up the tiles of all items (kItemUnits more per item, for
// its start and end) and takes an equal, contiguous share of them, whatever
// items that cuts: a long sequence beside many short ones, few rows over a long
// context and a long prompt all end at the same time.  An item that lies in one
// share is finished there; the parts of one that does not go to the workspace,
// two slots per workgroup (the part that its share begins with, and the one it
// ends with), and a second launch joins them in order.  Where the call's rows make
// an item for every workgroup that the GPU holds, the attention's items are listed
// by a launch of one workgroup instead, the longest first, a workgroup each, and
// only those longer than an equal share are cut.  Nothing depends on timing: equal
// calls give equal bits.
//
// Registers.  No kernel here may spill a vector register: the allocator, keeping
// part of a spilled 128-bit tuple in an accumulation register, lost its fourth
// dword (head dim 256, odd pages, listed: every score was wrong).  Fragments are
// read in batches, and offsets made where they are used, as far as that takes.
// (Scalar registers are spilled, into lanes of a vector register.)
#include "kernels.hpp"
#include "mfma_tile.hpp"

namespace aoakv {
namespace {

constexpr uint32_t kChThreads = 256;
constexpr int32_t kChRows = 128;  // rows of an item (attention)
constexpr int32_t kChTile = 64;   // keys (attention) or rows (weights) of a tile
constexpr float kLn2 = 0.6931471805599453f;
constexpr uint32_t kItemUnits = 1u;

// What the device tables say of a sequence, held to the sizes of the call.
struct Seq {
  int32_t q0, n, L, off, prefix;  // first row of q, new tokens, cached tokens, L - n
  uint32_t page0;                 // first entry of kv_indices
};
__device__ inline Seq load_seq(const ChunkArgs& a, uint32_t b) {
  Seq s;
  const int32_t T = (int32_t)a.T;
  const int32_t r0 = a.q_indptr[b], r1 = a.q_indptr[b + 1], p0 = a.kv_indptr[b],
                p1 = a.kv_indptr[b + 1];
  int32_t last = a.kv_last_page_len[b];
  s.prefix = a.prefix_len != nullptr ? a.prefix_len[b] : 0;
  s.q0 = min(max(r0, 0), T);
  s.n = max(min(r1, T) - s.q0, 0);
  last = min(max(last, 1), (int32_t)a.S);
  int32_t P = max(p1 - p0, 0);
  if (P > (int32_t)a.max_pages) {
    flag_error(a.error, kErrTruncated);
    P = (int32_t)a.max_pages;
    last = (int32_t)a.S;
  }
  s.page0 = (uint32_t)p0;
  s.L = P > 0 ? (P - 1) * (int32_t)a.S + last : 0;
  s.off = s.L - s.n;
  s.prefix = min(max(s.prefix, 0), s.L);
  return s;
}

// A value that is the same in all lanes, in a scalar register (what comes from
// LDS or a scan is not known to be: loops and tests on it would run in masks).
__device__ inline uint32_t scalar(uint32_t x) {
  return (uint32_t)__builtin_amdgcn_readfirstlane((int)x);
}
__device__ inline int32_t scalar(int32_t x) { return __builtin_amdgcn_readfirstlane(x); }
__device__ inline uint64_t scalar(uint64_t x) {
  return (uint64_t)scalar((uint32_t)(x >> 32)) << 32 | scalar((uint32_t)x);
}
__device__ inline Seq scalar(const Seq& s) {
  return Seq{scalar(s.q0), scalar(s.n), scalar(s.L), scalar(s.off), scalar(s.prefix),
             scalar(s.page0)};
}

// An item's tiles: tile i of its list is tile i < cut ? i : i - cut + first.
struct Item {
  int32_t cut, first, count;
  __device__ int32_t tile(int32_t i) const { return i < cut ? i : i - cut + first; }
};

__device__ inline int32_t group(const ChunkArgs& a) { return (int32_t)a.G; }
// r / G of a packed row (group_rcp = ceil(2^31 / G): exact for powers of two, and
// for r * G < 2^31; r < 2^30)
__device__ inline int32_t token_of(const ChunkArgs& a, int32_t r) {
  return (int32_t)__umulhi(2u * (uint32_t)r, a.group_rcp);
}
__device__ inline int32_t div_up(int32_t x, int32_t y) { return (x + y - 1) / y; }

// Items of 128 rows, tiles of 64 keys.
struct ByRows {
  static __device__ int32_t items(const ChunkArgs& a, const Seq& s) {
    return div_up(s.n * group(a), kChRows);
  }
  static __device__ Item item(const ChunkArgs& a, const Seq& s, int32_t x) {
    const int32_t i0 = token_of(a, x * kChRows),
                  i1 = min(s.n - 1, token_of(a, x * kChRows + kChRows - 1));
    const int32_t hi = a.causal ? min(max(s.off + i1 + 1, 0), s.L) : s.L;
    const int32_t lo = a.window != 0u ? max(s.off + i0 - (int32_t)a.window + 1, 0) : 0;
    const int32_t he = div_up(hi, kChTile), pe = div_up(s.prefix, kChTile), lt = lo / kChTile;
    if (pe >= lt) return Item{0, 0, max(pe, he)};
    return Item{pe, lt, pe + max(he - lt, 0)};
  }
};
// Items of KEYS keys, tiles of ROWS rows.
template <int32_t KEYS, int32_t ROWS>
struct ByKeys {
  static __device__ int32_t items(const ChunkArgs& a, const Seq& s) { return div_up(s.L, KEYS); }
  static __device__ Item item(const ChunkArgs& a, const Seq& s, int32_t x) {
    const int32_t k0 = x * KEYS;
    int32_t i0 = 0, i1 = s.n;
    if (k0 >= s.prefix) {
      if (a.causal) i0 = min(max(k0 - s.off, 0), s.n);
      if (a.window != 0u) i1 = min(max((int32_t)a.window + k0 + KEYS - 1 - s.off, 0), s.n);
    }
    const int32_t G = group(a), t0 = i0 * G / ROWS, t1 = div_up(i1 * G, ROWS);
    return Item{0, t0, i1 > i0 ? t1 - t0 : 0};
  }
};

// ---------------------------------------------------------------- shares
struct PlanLds {
  Seq seq[kChThreads];           // of the sequences base .. base + 255
  uint64_t start[kChThreads];    // units before each of them
  uint64_t wave[kChThreads / kWave];
  uint64_t off;
  uint32_t pick;
};

// the sum of x over the threads before this one, and over all
__device__ inline uint64_t scan_units(uint64_t x, PlanLds& l, uint64_t& total) {
  const uint32_t lane = __lane_id(), wave = threadIdx.x / kWave;
  uint64_t y = x;
#pragma nounroll  // (run once: its instructions are fetched cold)
  for (uint32_t d = 1; d < (uint32_t)kWave; d <<= 1) {
    const uint64_t z = __shfl_up((unsigned long long)y, d);
    if (lane >= d) y += z;
  }
  __syncthreads();
  if (lane == kWave - 1u) l.wave[wave] = y;
  __syncthreads();
  uint64_t before = 0u;
  total = 0u;
#pragma unroll
  for (uint32_t w = 0; w < kChThreads / kWave; ++w) {
    if (w < wave) before += l.wave[w];
    total += l.wave[w];
  }
  return before + y - x;
}

// A place in the list of all items' units: head by head, in it sequence by
// sequence, in it item by item.
template <class By>
struct Walk {
  const ChunkArgs& a;
  PlanLds& l;
  uint32_t base;    // first sequence in l.seq
  uint64_t before;  // units of the sequences before it
  uint64_t inside;  // ... and of those in l.seq
  uint32_t h, b;
  int32_t x;        // item of sequence b
  uint32_t at;      // unit of the item

  __device__ Walk(const ChunkArgs& args, PlanLds& lds) : a(args), l(lds), base(0u), before(0u),
                                                         inside(0u), h(0u), b(0u), x(0), at(0u) {}
  __device__ Seq seq() const { return scalar(l.seq[b - base]); }
  __device__ void load(uint32_t first) {
    __syncthreads();
    if (first + threadIdx.x < a.B) l.seq[threadIdx.x] = load_seq(a, first + threadIdx.x);
    __syncthreads();
    base = first;
  }
  // loads the sequences from `first` on and counts their units (several
  // threads share a sequence's items where the batch is small)
  __device__ void count(uint32_t first, uint64_t units_before) {
    load(first);
    const uint32_t nb = min(a.B - first, kChThreads);
    const uint32_t per = kChThreads >> (nb > 1u ? 32 - __clz(nb - 1u) : 0);
    const uint32_t sb = threadIdx.x / per, k = threadIdx.x % per;
    uint64_t u = 0u;
    if (sb < nb) {
      const Seq s = l.seq[sb];
      const int32_t n = By::items(a, s);
      for (int32_t i = (int32_t)k; i < n; i += (int32_t)per)
        u += (uint32_t)By::item(a, s, i).count + kItemUnits;
    }
    before = units_before;
    uint64_t sum;
    const uint64_t p = scan_units(u, l, sum);
    inside = scalar(sum);
    if (sb < nb && k == 0u) l.start[sb] = before + p;
    __syncthreads();
  }
  // units of one head
  __device__ uint64_t total() {
    uint64_t t = 0u;
    for (uint32_t first = 0u; first < a.B; first += kChThreads) {
      count(first, t);
      t += inside;
    }
    return t;
  }
  // goes to unit u of all heads, total() units each (u < H * total); total()
  // was called before
  __device__ void seek(uint64_t u, uint64_t per_head) {
    // u / per_head < 256: a quotient in fp32 is off by one at most
    h = scalar((uint32_t)((float)u * __builtin_amdgcn_rcpf((float)per_head)));
    h -= (uint64_t)h * per_head > u ? 1u : 0u;
    h += (uint64_t)(h + 1u) * per_head <= u ? 1u : 0u;
    const uint64_t y = u - (uint64_t)h * per_head;
    if (a.B > kChThreads) {
      uint64_t t = 0u;
      for (uint32_t first = 0u;; first += kChThreads) {
        count(first, t);
        t += inside;
        if (y < t) break;
      }
    }
    const uint32_t nb = min(a.B - base, kChThreads), i = threadIdx.x;
    if (i < nb) {
      const uint64_t s = l.start[i], e = i + 1u < nb ? l.start[i + 1u] : before + inside;
      if (s <= y && y < e) l.pick = i;
    }
    __syncthreads();
    b = base + scalar(l.pick);
    uint64_t rest = y - scalar(l.start[b - base]);
    const Seq s = seq();
    const int32_t n = By::items(a, s);
    __syncthreads();
    for (int32_t first = 0;; first += (int32_t)kChThreads) {
      const int32_t j = first + (int32_t)i;
      const uint64_t v = j < n ? (uint32_t)By::item(a, s, j).count + kItemUnits : 0u;
      uint64_t sum;
      const uint64_t p = scan_units(v, l, sum);
      sum = scalar(sum);
      if (rest < sum) {
        if (p <= rest && rest < p + v) {
          l.pick = (uint32_t)j;
          l.off = rest - p;
        }
        __syncthreads();
        break;
      }
      rest -= sum;
    }
    x = (int32_t)scalar(l.pick);
    at = (uint32_t)scalar(l.off);
    __syncthreads();
  }
  // the next item (there is one)
  __device__ void next() {
    at = 0u;
    ++x;
    while (x >= By::items(a, seq())) {
      x = 0;
      if (++b == a.B) {
        b = 0u;
        ++h;
      }
      if (b / kChThreads * kChThreads != base) load(b / kChThreads * kChThreads);
    }
  }
};

// The share of workgroup w: units [w * share, (w + 1) * share) of them
// (at least units / workgroups; the factor's rounding is below the 1 added).
__device__ inline uint64_t share_of(const ChunkArgs& a, uint64_t units, uint32_t least) {
  const uint64_t s = scalar((uint64_t)((double)units * a.share_rcp)) + 1u;
  return s > least ? s : least;
}

// An item in parts, for the launch that joins them: n parts (0: nothing to join),
// the first in slot `first`, the others in every step-th slot from first + 1 on.
struct Cut {
  uint32_t n, h, b;
  int32_t x, q0, rows;
  uint32_t first, step;
  __device__ size_t slot(uint32_t i) const {
    return i == 0u ? first : first + 1u + (i - 1u) * step;
  }
};
// The item that the border before workgroup `place`'s share cuts, where that is
// its first cut: slot 1 of the workgroup before, slot 0 of the following ones.
template <class By>
__device__ inline Cut cut_of(const Walk<By>& w, uint32_t place, uint64_t share) {
  Cut c{};
  if (w.at == 0u || w.at > share) return c;  // (at == share: it begins where the share before does)
  const Seq s = w.seq();
  const uint32_t after = (uint32_t)By::item(w.a, s, w.x).count + kItemUnits - w.at;
  c.n = 2u + (share >= after ? 0u : (after - 1u) / (uint32_t)share);
  c.h = w.h;
  c.b = w.b;
  c.x = w.x;
  c.q0 = s.q0;
  c.rows = s.n * group(w.a);
  c.first = 2u * place - 1u;
  c.step = 2u;
  return c;
}

// Workgroup b runs on XCD b % 8: neighbours in the list share an XCD (and its L2).
__device__ inline uint32_t list_place() {
  return blockIdx.x % kXcds * (gridDim.x / kXcds) + blockIdx.x / kXcds;
}

// ---------------------------------------------------------------- attention
constexpr int kCap = 1, kBias = 2;  // MOD bits

// floats of a part: O [D / 4][128 rows][4], m [128], l [128]
__host__ __device__ constexpr size_t part_floats(int D) { return (size_t)kChRows * (D + 2); }
// workgroups per CU (LDS: two buffers of K and V tiles; see prefill.hip)
template <int D>
constexpr uint32_t attn_per_cu() { return D == 256 ? 1u : 2u; }
constexpr uint32_t kCus = 256u;
// Probabilities are rounded to fp16 for the second product (products of 32-bit
// operands run at a sixteenth of the rate).  Beside the running maximum they are
// 2^8 at most (see `up` below) and fp16 holds 2^15, so all of them, and the sum
// and O that they make, are held 2^7 times as large: down to 2^-21 of that
// maximum the rounding is 2^-11 of a probability, as the values' own, and below
// it 2^-32 of the maximum.  (Without the factor, those below 2^-25 were missing
// in O and counted in the sum: 16384 keys of e^-17.5 beside one of 1, 4e-4 of the
// weight.)
constexpr float kLift = 7.f, kLiftInv = 1.f / 128.f;
constexpr size_t kCutBytes = kCus * 4u * sizeof(Cut);  // (4 workgroups per CU at most)
constexpr uint32_t kAttnLeast = 2u;  // units of a share at least

// Row r of a sequence's packed rows.
struct Row {
  int32_t tok;  // token of the chunk
  uint32_t h;   // query head
};
__device__ inline Row row_of(const ChunkArgs& a, uint32_t hk, int32_t r) {
  const int32_t tok = token_of(a, r);
  return Row{tok, hk * a.G + (uint32_t)r - (uint32_t)tok * a.G};
}

// o and lse of a row: O dims 32 t + crow(i, g) of the lane's row; l and O are
// lifted
template <int D>
__device__ inline void store_row(const ChunkArgs& a, const Seq& s, const Row& r, int g, float m2,
                                 float l, const floatx16 (&acc)[PfShape<D>::kDB]) {
  const size_t row = (size_t)(s.q0 + r.tok) * a.Hq + r.h;
  const float inv = l == 0.f ? 0.f : 1.f / l;
  f16* o = a.o + row * D;
#pragma unroll
  for (int t = 0; t < PfShape<D>::kDB; ++t)
#pragma unroll
    for (int i0 = 0; i0 < 16; i0 += 4) {
      half4 v;
#pragma unroll
      for (int e = 0; e < 4; ++e) v[e] = (f16)(acc[t][i0 + e] * inv);
      *reinterpret_cast<half4*>(o + t * 32 + crow(i0, g)) = v;
    }
  if (a.lse != nullptr && g == 0)
    a.lse[row] = l == 0.f ? -INFINITY : (m2 + __builtin_amdgcn_logf(l * kLiftInv)) * kLn2;
}

// A call of many items: a launch before lists them (and the parts of those
// longer than an equal share), the longest first, for one workgroup each.
// Walking the keys of a head from its first on, side by side, the workgroups of
// an XCD find them in its L2, and few items are cut.  The listing takes 5 us;
// 8192 tokens of 32 heads take 680 us in shares and 574 so.
struct Entry {
  uint32_t b;
  int32_t x, t0, t1;
  uint32_t slot;  // of the head's parts, or kWhole
};
struct ListHead {
  uint32_t entries, parts, cuts;  // of each head
};
constexpr uint32_t kWhole = 0xFFFFFFFFu;
constexpr size_t kListHeadBytes = 64;
constexpr int32_t kListBins = 1024;

__global__ __launch_bounds__(kChThreads) void chunk_list_kernel(ChunkArgs a, uint32_t slots,
                                                                  uint32_t room) {
  __shared__ PlanLds s_plan;
  __shared__ uint32_t s_bin[kListBins], s_parts, s_cuts, s_wave[kChThreads / kWave];
  const uint32_t tid = threadIdx.x;
  Walk<ByRows> w(a, s_plan);
  const uint64_t per_head = w.total();
  const uint64_t share64 = per_head * a.H / slots + 1u;
  const uint32_t share = (uint32_t)(share64 < 0x7FFFFFFFu ? share64 : 0x7FFFFFFFu);
  for (uint32_t i = tid; i < (uint32_t)kListBins; i += kChThreads) s_bin[i] = 0u;
  if (tid == 0u) s_parts = s_cuts = 0u;
  __syncthreads();
  // twice over all items: how many entries there are of each length (bins from
  // the longest on), then their places
  Entry* list = static_cast<Entry*>(a.list);
  Cut* cuts = reinterpret_cast<Cut*>(static_cast<char*>(a.cuts) + kListHeadBytes);
  for (int pass = 0; pass < 2; ++pass) {
    for (uint32_t first = 0u; first < a.B; first += kChThreads) {
      if (a.B > kChThreads) w.load(first);
      const uint32_t nb = min(a.B - first, kChThreads);
      const uint32_t per = kChThreads >> (nb > 1u ? 32 - __clz(nb - 1u) : 0);
      const uint32_t sb = tid / per;
      if (sb >= nb) continue;
      const Seq s = s_plan.seq[sb];
      const int32_t n = ByRows::items(a, s);
      for (int32_t x = (int32_t)(tid % per); x < n; x += (int32_t)per) {
        const uint32_t count = (uint32_t)ByRows::item(a, s, x).count;
        const uint32_t units = count + kItemUnits;
        const uint32_t parts = units > share ? (units + share - 1u) / share : 1u;
        const int32_t length = (int32_t)((count + parts - 1u) / parts);
        const uint32_t bin = (uint32_t)(kListBins - 1 - min(length, kListBins - 1));
        const uint32_t at = atomicAdd(&s_bin[bin], parts);
        if (pass == 0) continue;
        uint32_t slot = kWhole;
        if (parts > 1u) {
          slot = atomicAdd(&s_parts, parts);
          Cut c{};
          c.n = parts;
          c.b = first + sb;
          c.x = x;
          c.q0 = s.q0;
          c.rows = s.n * group(a);
          c.first = slot;
          c.step = 1u;
          cuts[atomicAdd(&s_cuts, 1u)] = c;
        }
        // (room: what rows of a q_indptr that counts none twice can fill)
        for (uint32_t i = 0; i < parts && at + i < room; ++i)
          list[at + i] = Entry{first + sb, x, (int32_t)((uint64_t)count * i / parts),
                               (int32_t)((uint64_t)count * (i + 1u) / parts),
                               parts > 1u ? slot + i : kWhole};
      }
    }
    __syncthreads();
    if (pass == 0) {  // bins to their first places
      constexpr uint32_t kN = kListBins / kChThreads;
      uint32_t v[kN], sum = 0u;
      for (uint32_t i = 0; i < kN; ++i) sum += v[i] = s_bin[tid * kN + i];
      uint32_t upto = sum;
      for (uint32_t d = 1; d < (uint32_t)kWave; d <<= 1) {
        const uint32_t y = __shfl_up(upto, d);
        if (__lane_id() >= d) upto += y;
      }
      if (__lane_id() == kWave - 1u) s_wave[tid / kWave] = upto;
      __syncthreads();
      for (uint32_t i = 0; i < tid / kWave; ++i) upto += s_wave[i];
      uint32_t before = upto - sum;
      if (tid == kChThreads - 1u) reinterpret_cast<ListHead*>(a.cuts)->entries = min(upto, room);
      for (uint32_t i = 0; i < kN; ++i) {
        s_bin[tid * kN + i] = before;
        before += v[i];
      }
      __syncthreads();
    }
  }
  if (tid == 0u) {
    reinterpret_cast<ListHead*>(a.cuts)->parts = s_parts;
    reinterpret_cast<ListHead*>(a.cuts)->cuts = s_cuts;
  }
}

// One workgroup's share, or its entry of the list.  The tile loop is that of
// prefill.hip (S^T = K Q^T, lane l holds row l % 32 of its wave's 32); scores are
// kept in units of log 2.
//
// What bounds it: a tile's K and V fragments pass from LDS to the matrix cores at
// 128 bytes a clock and CU, the rate at which the products consume them, and the
// exponentials take as long again; two workgroups per CU run one beside the other.
// 8192 tokens over themselves, causal: 32 heads of 128 572 us (960 TFLOP/s; 8 kv
// heads the same), with slopes 620, a cap 693; 16 heads of 256 722, 859 and 795; 32
// of 64 347, 371 and 474 (smallest of 5 x 20 calls, normal inputs; with a few large
// channels 637 to 648 with slopes).  Few rows over a long cache pass 5.3 TB/s.  64
// rows per wave, which halves the fragments, left one wave per SIMD and took 920 us
// (650 then).
template <int D, int MOD, bool S16, bool LIST>
__global__ __launch_bounds__(kChThreads, attn_per_cu<D>()) void chunk_attn_kernel(ChunkArgs a) {
  using Sh = PfShape<D>;
  __shared__ __attribute__((aligned(16))) char s_buf0[2 * Sh::kTileBytes];
  __shared__ __attribute__((aligned(16))) char s_buf1[2 * Sh::kTileBytes];
  __shared__ PlanLds s_plan;
  const int tid = threadIdx.x;
  const int wave = __builtin_amdgcn_readfirstlane(tid / kWave);

  Walk<ByRows> w(a, s_plan);
  uint64_t u = 0u, u1 = 0u;
  if constexpr (!LIST) {
    const uint64_t per_head = w.total(), units = per_head * a.H;
    const uint64_t share = share_of(a, units, kAttnLeast);
    u = list_place() * share;
    u1 = min(u + share, units);
    if (u >= u1) {
      if (tid == 0 && !a.whole) reinterpret_cast<Cut*>(a.cuts)[list_place()].n = 0u;
      return;
    }
    w.seek(u, per_head);
    if (a.whole) {  // no workspace: the items that begin in the share, whole
      if (w.at != 0u) {
        u += (uint32_t)ByRows::item(a, w.seq(), w.x).count + kItemUnits - w.at;
        if (u >= u1) return;
        w.next();
      }
    } else if (tid == 0) {
      reinterpret_cast<Cut*>(a.cuts)[list_place()] = cut_of(w, list_place(), share);
    }
  }

  // Slopes alone begin the scores with their distances, and the products are added
  // to these (the step took 4 and 6 % off 8192 tokens of 32 heads of 128 and of 64;
  // at head dim 256 the tile's start held more registers than there are).
  constexpr bool kBegin = MOD == kBias && D != 256;
  const float scale = MOD == 0 || kBegin ? a.sm_scale * kLog2e : 1.f;
  // cap: c tanh(x / c) = c - 2 c / (1 + e^(2 x / c))
  const float cap2 = a.soft_cap * kLog2e;
  const float cap_in = MOD & kCap ? 2.f * kLog2e * a.sm_scale / a.soft_cap : 0.f;
  const int32_t window = a.window != 0u ? (int32_t)a.window : 1 << 30;

  for (;;) {
    // (the offsets below are made anew for each item: kept over the loop, their
    // registers would be missing at an item's end)
    int lane = (int)__lane_id();
    asm volatile("" : "+v"(lane));
    const int g = lane / 32, c = lane % 32;
    constexpr int kNI = 16 / Sh::kRPI;  // load instructions per wave and tile
    constexpr int kRow16 = 16 * Sh::kRowBytes;
    const int lrow = lane / Sh::kCh;
    // lane-constant offsets into a tile (see prefill.hip)
    const int vm = (lane % 16) / 4, va4 = lane % 4, vG = lane / 16;
    auto v_off = [&](int t, int key0) {
      const int row = key0 + vm;
      const int dim = 32 * t + 16 * (vG % 2) + 4 * va4;
      return row * Sh::kRowBytes + 16 * ((dim / 8) ^ v_swz<Sh::kCh>(row)) + 2 * (dim % 8);
    };
    // (the swizzles are XORs above the bits of s8 and t, so each offset is the
    // first one XOR a constant: at D = 256, where 32 registers of offsets would
    // be spilled, they are made where they are used)
    constexpr bool kXor = D == 256;
    int k_off[kXor ? 1 : Sh::kKS], v_lo[kXor ? 1 : Sh::kDB], v_hi[kXor ? 1 : Sh::kDB];
#pragma unroll
    for (int s8 = 0; s8 < (kXor ? 1 : Sh::kKS); ++s8) k_off[s8] = tile_off<D>(c, 2 * s8 + g);
#pragma unroll
    for (int t = 0; t < (kXor ? 1 : Sh::kDB); ++t) {
      v_lo[t] = v_off(t, 4 * g);
      v_hi[t] = v_off(t, 4 * g + 8);
    }
    auto k_at = [&](int s8) { return kXor ? k_off[0] ^ (32 * s8) : k_off[s8 % Sh::kKS]; };
    auto lo_at = [&](int t) { return kXor ? v_lo[0] ^ (64 * t) : v_lo[t]; };
    auto hi_at = [&](int t) { return kXor ? v_hi[0] ^ (64 * t) : v_hi[t]; };

    // ---- the work: tiles t0 .. t1 - 1 of item ix of a sequence and kv head hk,
    // whole or for a slot of the workspace
    Seq s;
    int32_t ix, t0, t1;
    uint32_t hk, slot, units = 0u;
    Item item;
    if constexpr (LIST) {
      // (an entry per workgroup, the longest of all heads first; heads as in
      // prefill.hip: each XCD its own, walking their keys side by side)
      const ListHead* head = reinterpret_cast<const ListHead*>(a.cuts);
      const uint32_t k = blockIdx.x / a.H, hs = blockIdx.x % a.H;
      if (k >= head->entries) return;
      hk = a.H % kXcds == 0u ? hs % kXcds * (a.H / kXcds) + hs / kXcds : hs;
      const Entry e = static_cast<const Entry*>(a.list)[k];
      s = scalar(load_seq(a, e.b));
      ix = e.x;
      t0 = e.t0;
      t1 = e.t1;
      item = ByRows::item(a, s, ix);
      slot = e.slot == kWhole ? kWhole : hk * head->parts + e.slot;
    } else {
      s = w.seq();
      ix = w.x;
      item = ByRows::item(a, s, ix);
      hk = w.h;
      const uint32_t ue = (uint32_t)item.count + kItemUnits;
      const uint32_t ua = w.at, ub = a.whole ? ue : (uint32_t)min((uint64_t)ue, ua + (u1 - u));
      units = ub - ua;
      t0 = (int32_t)((uint64_t)ua * (uint32_t)item.count / ue);
      t1 = (int32_t)((uint64_t)ub * (uint32_t)item.count / ue);
      slot = ua == 0u && ub == ue ? kWhole : 2u * list_place() + (ua == 0u ? 1u : 0u);
    }

    // ---- this lane's row
    const int32_t R = s.n * group(a);
    const int32_t r0 = ix * kChRows + wave * 32;  // the wave's first row
    const int32_t r = r0 + c;
    const bool live = r < R;
    const Row row = row_of(a, hk, live ? r : R - 1);
    const int32_t pos = s.off + row.tok;
    half8 qreg[Sh::kKS];
    {
      const f16* q = a.q + ((size_t)(s.q0 + row.tok) * a.Hq + row.h) * D + 8 * g;
#pragma unroll
      for (int s8 = 0; s8 < Sh::kKS; ++s8) qreg[s8] = *reinterpret_cast<const half8*>(q + 16 * s8);
    }
    const float slope = MOD & kBias ? a.slopes[row.h] * kLog2e / scale : 0.f;
    // keys the row sees: below s.prefix, and [lo, hi)
    const int32_t hi = a.causal ? min(pos + 1, s.L) : s.L, lo = pos - window + 1;
    // first and last position of the wave's rows and of the item's
    const int32_t wp0 = s.off + token_of(a, min(r0, R - 1)),
                  wp1 = s.off + token_of(a, min(r0 + 31, R - 1));
    // whether rows at positions p0 .. p1 all see the 64 keys from k0 on
    auto all_see = [&](int32_t k0, int32_t p0, int32_t p1) {
      return k0 + kChTile <= s.prefix ||
             (k0 + kChTile <= s.L && (!a.causal || k0 + kChTile - 1 <= p0) && p1 - k0 < window);
    };
    // ... or any of the wave's sees one
    auto any_sees = [&](int32_t k0) {
      return r0 < R && (k0 < s.prefix || ((!a.causal || k0 <= wp1) &&
                                          wp0 - (k0 + kChTile - 1) < window));
    };

    // ---- tile loads: wave w fills rows 16 w .. 16 w + 15 of K and V
    struct PageIds {
      uint32_t id[S16 ? 1 : kNI];
    };
    const uint32_t npages = div_page((uint32_t)s.L + a.S - 1u, a.page_rcp);
    const __attribute__((address_space(4))) int32_t* kv_idx =
        (const __attribute__((address_space(4))) int32_t*)(a.kv_indices + s.page0);
    // (a page past the sequence reads the last one: its keys are masked)
    auto page_of = [&](int32_t tile) {
      const uint32_t key0 = (uint32_t)(tile * kChTile + 16 * wave);
      PageIds ph;
      if constexpr (S16) {  // the wave's 16 rows lie in one page
        const uint32_t p = div_page(key0, a.page_rcp);
        ph.id[0] = (uint32_t)kv_idx[p < npages ? p : npages - 1u];
      } else {
#pragma unroll
        for (int i = 0; i < kNI; ++i) {
          const uint32_t p = div_page(key0 + (uint32_t)(Sh::kRPI * i + lrow), a.page_rcp);
          ph.id[i] = (uint32_t)a.kv_indices[s.page0 + (p < npages ? p : npages - 1u)];
        }
      }
      return ph;
    };
    auto load_tile = [&](char* buf, const PageIds& ph, int32_t tile) {
      int ln = lane;
      if constexpr (kXor) asm volatile("" : "+v"(ln));  // (as the offsets above)
      const int lrow = ln / Sh::kCh, lslot = ln % Sh::kCh;
      const uint32_t key0 = (uint32_t)(tile * kChTile + 16 * wave);
#pragma unroll
      for (int i = 0; i < kNI; ++i) {
        const int tr = 16 * wave + Sh::kRPI * i + lrow;
        const uint32_t key = key0 + (uint32_t)(Sh::kRPI * i + lrow);
        const uint32_t slot = S16 ? key & (a.S - 1u) : key - div_page(key, a.page_rcp) * a.S;
        const size_t e = elem_off(a.g, ph.id[S16 ? 0 : i], 0, hk, slot);
        load_lds16(a.kv + e + 8 * (lslot ^ k_swz<Sh::kCh>(tr)),
                   buf + (16 * wave + Sh::kRPI * i) * Sh::kRowBytes);
        load_lds16(a.kv + e + a.g.kv + 8 * (lslot ^ v_swz<Sh::kCh>(tr)),
                   buf + Sh::kTileBytes + (16 * wave + Sh::kRPI * i) * Sh::kRowBytes);
      }
    };

    floatx16 acc_o[Sh::kDB];
#pragma unroll
    for (int t = 0; t < Sh::kDB; ++t) acc_o[t] = floatx16{};
    float m_run = kPfNoMax, l_run = 0.f;
    // At head dim 64 a row's two lanes each keep the sum of their own keys until the
    // item's end (with slopes 393 -> 371 us, a cap 512 -> 481; at 128 it spilled).
    constexpr bool kHalves = D == 64;
    // O elements that a value of +inf / -inf / NaN (both) reaches, bit 16 t + i
    constexpr int kFlags = D == 256 ? 2 : 1;
    uint64_t inf_pos[kFlags] = {}, inf_neg[kFlags] = {};

    auto vfrag = [&](const lds_char* sV, int t, int kk) {
      const int rows = kk * kRow16;
      const half4 x = __builtin_bit_cast(
          half4, __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_short4*)(sV + lo_at(t) + rows)));
      const half4 y = __builtin_bit_cast(
          half4, __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_short4*)(sV + hi_at(t) + rows)));
      return __builtin_shufflevector(x, y, 0, 1, 2, 3, 4, 5, 6, 7);
    };

    // A value of inf or NaN that some rows of the wave do not see: a probability of
    // 0 times it would be NaN in the product.  So where a tile that is masked in
    // part holds any (rare; found in the fragments on their way), they are 0 in
    // the product, and this notes the O elements that they reach.
    auto note_values = [&](const lds_char* sV, int32_t k0) {
      const int end = min(kChTile, s.L - k0) * Sh::kCh;  // (slots behind the end are nobody's)
#pragma nounroll
      for (int j = 0; j < end; j += kWave) {
        const int at = j + lane;
        bool odd = false;
        if (at < end) {
          const half8 x = *reinterpret_cast<const __attribute__((address_space(3))) half8*>(
              sV + 16 * at);
#pragma unroll
          for (int e = 0; e < 8; ++e) odd |= !__builtin_isfinite((float)x[e]);
        }
#pragma nounroll
        for (uint64_t left = __builtin_amdgcn_ballot_w64(odd); left != 0u; left &= left - 1u) {
          const int src = __builtin_ctzll(left);
          const int tr = (j + src) / Sh::kCh;
          const int d0 = 8 * (((j + src) % Sh::kCh) ^ v_swz<Sh::kCh>(tr));
          const int32_t key = k0 + tr;
          const bool seen = key < s.prefix || (key < hi && key >= lo);
#pragma nounroll
          for (int e = 0; e < 8; ++e) {
            const uint32_t y = *reinterpret_cast<const __attribute__((address_space(3))) uint16_t*>(
                sV + 16 * (j + src) + 2 * e);
            if ((y & 0x7C00u) != 0x7C00u) continue;
            // dim d0 + e is element 16 t + i of lane group dd / 4 % 2
            const int dd = (d0 + e) % 32, bit = 16 * ((d0 + e) / 32) + 4 * (dd / 8) + dd % 4;
            const uint64_t mask = seen && dd / 4 % 2 == g ? 1ull << (bit % 64) : 0u;
            const bool nan = (y & 0x3FFu) != 0u;
#pragma unroll
            for (int f = 0; f < kFlags; ++f) {
              if (bit / 64 != f) continue;
              if (nan || y == 0x7C00u) inf_pos[f] |= mask;
              if (nan || y == 0xFC00u) inf_neg[f] |= mask;
            }
          }
        }
      }
    };

    // what the products of a tile are added to
    auto begin_scores = [&](floatx16 (&x)[2], int32_t k0) {
      x[0] = x[1] = floatx16{};
      if constexpr (kBegin) {
        const float d0 = (float)(pos - k0 - 4 * g);  // crow(i, g) = crow(i, 0) + 4 g
        if (k0 + kChTile - 1 <= wp0) {  // no key behind a row: the distances need no |.|
          const float far = -slope * d0;
#pragma unroll
          for (int ks = 0; ks < 2; ++ks)
#pragma unroll
            for (int i = 0; i < 16; ++i)
              x[ks][i] = __builtin_fmaf(slope, (float)(ks * 32 + crow(i, 0)), far);
        } else {
#pragma unroll
          for (int ks = 0; ks < 2; ++ks)
#pragma unroll
            for (int i = 0; i < 16; ++i)
              x[ks][i] = -slope * __builtin_fabsf(d0 - (float)(ks * 32 + crow(i, 0)));
        }
      }
    };

    auto tile = [&](const lds_char* sK, const lds_char* sV, int32_t k0) {
      if constexpr (kXor) {
        asm volatile("" : "+v"(k_off[0]));
        asm volatile("" : "+v"(v_lo[0]));
        asm volatile("" : "+v"(v_hi[0]));
      }
      floatx16 acc_s[2];
      if constexpr (Sh::kKS <= 8) {
        half8 kf0[Sh::kKS], kf1[Sh::kKS];
#pragma unroll
        for (int s8 = 0; s8 < Sh::kKS; ++s8)
          kf0[s8] = *reinterpret_cast<const __attribute__((address_space(3))) half8*>(
              sK + k_at(s8));
#pragma unroll
        for (int s8 = 0; s8 < Sh::kKS; ++s8)
          kf1[s8] = *reinterpret_cast<const __attribute__((address_space(3))) half8*>(
              sK + k_at(s8) + 2 * kRow16);
        __builtin_amdgcn_sched_barrier(0);
        begin_scores(acc_s, k0);
#pragma unroll
        for (int s8 = 0; s8 < Sh::kKS; ++s8) acc_s[0] = mfma32(kf0[s8], qreg[s8], acc_s[0]);
#pragma unroll
        for (int s8 = 0; s8 < Sh::kKS; ++s8) acc_s[1] = mfma32(kf1[s8], qreg[s8], acc_s[1]);
      } else {
        constexpr int kB = 4, kNB = 2 * Sh::kKS / kB;  // batches of 4 fragments
        // (batches of 8 spilled up to 35 registers and took 755 us at 8192 tokens for 740)
        auto kread = [&](int bt, half8 (&kf)[kB]) {
#pragma unroll
          for (int j = 0; j < kB; ++j)
            kf[j] = *reinterpret_cast<const __attribute__((address_space(3))) half8*>(
                sK + k_at((bt % (kNB / 2)) * kB + j) + (bt / (kNB / 2)) * 2 * kRow16);
        };
        half8 kfa[kB], kfb[kB];
        begin_scores(acc_s, k0);
        kread(0, kfa);
#pragma unroll
        for (int bt = 0; bt < kNB; bt += 2) {
          kread(bt + 1, kfb);
          __builtin_amdgcn_sched_barrier(0);
#pragma unroll
          for (int j = 0; j < kB; ++j)
            acc_s[bt / (kNB / 2)] =
                mfma32(kfa[j], qreg[(bt % (kNB / 2)) * kB + j], acc_s[bt / (kNB / 2)]);
          if (bt + 2 < kNB) kread(bt + 2, kfa);
          __builtin_amdgcn_sched_barrier(0);
#pragma unroll
          for (int j = 0; j < kB; ++j)
            acc_s[(bt + 1) / (kNB / 2)] =
                mfma32(kfb[j], qreg[((bt + 1) % (kNB / 2)) * kB + j], acc_s[(bt + 1) / (kNB / 2)]);
        }
      }
      if constexpr (MOD != 0 && !kBegin) {
        const float d0 = (float)(pos - k0 - 4 * g);  // crow(i, g) = crow(i, 0) + 4 g
        const float pre = MOD & kCap ? 0.f : a.sm_scale * kLog2e;
        if (MOD & kCap) {
#pragma unroll
          for (int ks = 0; ks < 2; ++ks)
#pragma unroll
            for (int i = 0; i < 16; ++i)
              acc_s[ks][i] = __builtin_fmaf(
                  -2.f * cap2,
                  __builtin_amdgcn_rcpf(1.f + __builtin_amdgcn_exp2f(acc_s[ks][i] * cap_in)), cap2);
        }
        if constexpr (MOD & kBias) {
          if (k0 + kChTile - 1 <= wp0) {  // no key behind a row: the distances need no |.|
            const float far = -slope * d0;
#pragma unroll
            for (int ks = 0; ks < 2; ++ks)
#pragma unroll
              for (int i = 0; i < 16; ++i) {
                const float t = MOD & kCap ? acc_s[ks][i] + far
                                           : __builtin_fmaf(acc_s[ks][i], pre, far);
                acc_s[ks][i] = __builtin_fmaf(slope, (float)(ks * 32 + crow(i, 0)), t);
              }
          } else {
#pragma unroll
            for (int ks = 0; ks < 2; ++ks)
#pragma unroll
              for (int i = 0; i < 16; ++i) {
                const float d = __builtin_fabsf(d0 - (float)(ks * 32 + crow(i, 0)));
                const float t = MOD & kCap ? acc_s[ks][i] : acc_s[ks][i] * pre;
                acc_s[ks][i] = __builtin_fmaf(-slope, d, t);
              }
          }
        }
      }
      bool dirty = false;
      if (!all_see(k0, wp0, wp1)) {
        // (one unsigned comparison for the range, one for the prefix)
        uint32_t odd = 0u;  // values of inf or NaN (adding 1 to the exponent carries)
#pragma unroll
        for (int t = 0; t < Sh::kDB; ++t)
#pragma unroll
          for (int kk = 0; kk < 4; ++kk) {
            const u32x4 y = __builtin_bit_cast(u32x4, vfrag(sV, t, kk));
#pragma unroll
            for (int e = 0; e < 4; ++e) odd |= (y[e] & 0x7C007C00u) + 0x04000400u;
          }
        dirty = __builtin_amdgcn_ballot_w64((odd & 0x80008000u) != 0u) != 0u;
        if (dirty) note_values(sV, k0);
        const int32_t first = k0 + 4 * g, pre = s.prefix - first;
        const uint32_t begin = (uint32_t)(lo - first), span = (uint32_t)max(hi - lo, 0);
#pragma unroll
        for (int ks = 0; ks < 2; ++ks)
#pragma unroll
          for (int i = 0; i < 16; ++i) {
            const int32_t key = ks * 32 + crow(i, 0);
            const bool see = (int)(key < pre) | (int)((uint32_t)key - begin < span);
            acc_s[ks][i] = see ? acc_s[ks][i] : -INFINITY;
          }
      }
      float mt = acc_s[0][0];
#pragma unroll
      for (int ks = 0; ks < 2; ++ks)
#pragma unroll
        for (int i = 0; i < 16; ++i) mt = fmaxf(mt, acc_s[ks][i]);
      mt = pair_max(mt);
      // lazy rescaling (see prefill.hip): a row's running max moves only where a
      // probability would pass 2^8 (each row by itself: what other rows of the
      // wave see does not touch its bits)
      const bool up = (mt - m_run) * scale > 8.f;
      const bool move = __builtin_amdgcn_ballot_w64(up) != 0;
      const float m_new = up ? mt : m_run;
      const float neg_m = __builtin_fmaf(-m_new, scale, kLift);
      float lt = 0.f;
      half8 pb[2][2];
#pragma unroll
      for (int ks = 0; ks < 2; ++ks)
#pragma unroll
        for (int i = 0; i < 16; ++i) {
          const float p = __builtin_amdgcn_exp2f(__builtin_fmaf(acc_s[ks][i], scale, neg_m));
          lt += p;
          // (the sum l has them unrounded; kLift)
          pb[ks][i / 8][i % 8] = (f16)p;
        }
      if constexpr (!kHalves) lt = pair_sum(lt);
      if (move) {
        const float alpha = __builtin_amdgcn_exp2f((m_run - m_new) * scale);
        l_run = l_run * alpha;
#pragma unroll
        for (int t = 0; t < Sh::kDB; ++t)
#pragma unroll
          for (int i = 0; i < 16; ++i) acc_o[t][i] *= alpha;
      }
      l_run = l_run + lt;
      m_run = m_new;
      auto frags = [&](int t, half8 (&f)[4]) {
#pragma unroll
        for (int kk = 0; kk < 4; ++kk) f[kk] = vfrag(sV, t, kk);
        if (dirty) {  // (uniform; a copy of the loop below for it spilled registers)
#pragma unroll
          for (int kk = 0; kk < 4; ++kk)
#pragma unroll
            for (int e = 0; e < 8; ++e)
              f[kk][e] = __builtin_isfinite((float)f[kk][e]) ? f[kk][e] : (f16)0.f;
        }
      };
      half8 vfa[4], vfb[4];
      frags(0, vfa);
#pragma unroll
      for (int t = 0; t < Sh::kDB; t += 2) {
        frags(t + 1, vfb);
        __builtin_amdgcn_sched_barrier(0);
#pragma unroll
        for (int kk = 0; kk < 4; ++kk) acc_o[t] = mfma32(vfa[kk], pb[kk / 2][kk % 2], acc_o[t]);
        if (t + 2 < Sh::kDB) frags(t + 2, vfa);
        __builtin_amdgcn_sched_barrier(0);
#pragma unroll
        for (int kk = 0; kk < 4; ++kk)
          acc_o[t + 1] = mfma32(vfb[kk], pb[kk / 2][kk % 2], acc_o[t + 1]);
      }
    };

    // ---- the tiles of this part
    __syncthreads();  // the item before is done with the buffers
    PageIds ids{};
    if (t0 < t1) {
      load_tile(s_buf0, page_of(item.tile(t0)), item.tile(t0));
      if (t0 + 1 < t1) ids = page_of(item.tile(t0 + 1));
    }
    for (int32_t it = t0; it < t1; it += 2) {
#pragma unroll
      for (int v = 0; v < 2; ++v) {
        const int32_t i = it + v;
        if (i >= t1) break;  // uniform
        char* buf = v == 0 ? s_buf0 : s_buf1;
        asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
        __syncthreads();
        if (i + 1 < t1) {
          load_tile(v == 0 ? s_buf1 : s_buf0, ids, item.tile(i + 1));
          if (i + 2 < t1) ids = page_of(item.tile(i + 2));
        }
        const int32_t k0 = item.tile(i) * kChTile;
        if (any_sees(k0)) tile((const lds_char*)buf, (const lds_char*)(buf + Sh::kTileBytes), k0);
      }
    }

#pragma unroll
    for (int t = 0; t < Sh::kDB; ++t)
      if (inf_pos[t / 4] != 0u || inf_neg[t / 4] != 0u) {
#pragma unroll
        for (int i = 0; i < 16; ++i) {
          const int bit = (16 * t + i) % 64;
          if (inf_pos[t / 4] >> bit & 1u) acc_o[t][i] += INFINITY;
          if (inf_neg[t / 4] >> bit & 1u) acc_o[t][i] -= INFINITY;
        }
      }
    if constexpr (kHalves) l_run = pair_sum(l_run);
    // (in units of log 2, as the exponents had it)
    const float m2 = kLift - __builtin_fmaf(-m_run, scale, kLift);
    if (slot == kWhole) {
      if (live) store_row<D>(a, s, row, g, m2, l_run, acc_o);
    } else if (live) {  // a part: O lifted, l not
      float* part = a.parts + (size_t)slot * part_floats(D);
      float4* po = reinterpret_cast<float4*>(part) + wave * 32 + c;
#pragma unroll
      for (int j = 0; j < Sh::kDB * 4; ++j) {
        const floatx16& x = acc_o[j / 4];
        const int i0 = 4 * (j % 4);
        po[(8 * (j / 4) + 2 * (j % 4) + g) * kChRows] =
            float4{x[i0], x[i0 + 1], x[i0 + 2], x[i0 + 3]};
      }
      if (g == 0) {
        float* pm = part + kChRows * D + wave * 32 + c;
        pm[0] = m2;
        pm[kChRows] = l_run * kLiftInv;
      }
    }
    if constexpr (LIST) return;
    u += units;
    if (u >= u1) return;
    w.next();
  }
}

// Joins an item's parts: workgroup (cut, sub) takes 32 of its rows, a thread one
// row and D / 8 dims.
template <int D, bool LIST>
__global__ __launch_bounds__(kChThreads) void chunk_join_kernel(ChunkArgs a) {
  const uint32_t place = blockIdx.x / 4u, sub = blockIdx.x % 4u;
  Cut cut;
  if constexpr (LIST) {
    const ListHead* head = reinterpret_cast<const ListHead*>(a.cuts);
    if (place / a.H >= head->cuts) return;
    cut = reinterpret_cast<const Cut*>(static_cast<const char*>(a.cuts) +
                                       kListHeadBytes)[place / a.H];
    cut.h = place % a.H;
    cut.first += cut.h * head->parts;
  } else {
    cut = reinterpret_cast<const Cut*>(a.cuts)[place + 1u];
    if (cut.n == 0u) return;
  }
  const int32_t r = (int32_t)(sub * 32u + threadIdx.x % 32u);
  if (cut.x * kChRows + r >= cut.rows) return;
  const Row row = row_of(a, cut.h, cut.x * kChRows + r);
  const uint32_t j0 = threadIdx.x / 32u;
  // kAt parts at a time, their loads together: a part after the other, few rows
  // over many parts took 17 us
  constexpr int kV = D / 32, kAt = D == 256 ? 4 : 8;
  float m = kPfNoMax, l = 0.f;
  float4 acc[kV] = {};
  for (uint32_t i0 = 0; i0 < cut.n; i0 += kAt) {
    float pm[kAt], pl[kAt];
    float4 po[kAt][kV];
#pragma unroll
    for (int i = 0; i < kAt; ++i) {
      pm[i] = kPfNoMax;
      if (i0 + (uint32_t)i >= cut.n) continue;  // uniform
      const float* p = a.parts + cut.slot(i0 + (uint32_t)i) * part_floats(D);
      pm[i] = p[kChRows * D + r];
      pl[i] = p[kChRows * (D + 1) + r];
#pragma unroll
      for (int v = 0; v < kV; ++v)
        po[i][v] = reinterpret_cast<const float4*>(p)[(kV * j0 + v) * kChRows + r];
    }
    float top = m;
#pragma unroll
    for (int i = 0; i < kAt; ++i) top = fmaxf(top, pm[i]);
    const float keep = __builtin_amdgcn_exp2f(m - top);
    m = top;
    l *= keep;
#pragma unroll
    for (int v = 0; v < kV; ++v) {
      acc[v].x *= keep;
      acc[v].y *= keep;
      acc[v].z *= keep;
      acc[v].w *= keep;
    }
#pragma unroll
    for (int i = 0; i < kAt; ++i) {
      if (i0 + (uint32_t)i >= cut.n) break;  // uniform
      const float f = __builtin_amdgcn_exp2f(pm[i] - m);
      l += pl[i] * f;
#pragma unroll
      for (int v = 0; v < kV; ++v) {
        acc[v].x += po[i][v].x * f;
        acc[v].y += po[i][v].y * f;
        acc[v].z += po[i][v].z * f;
        acc[v].w += po[i][v].w * f;
      }
    }
  }
  const float inv = l == 0.f ? 0.f : kLiftInv / l;
  const size_t at = (size_t)(cut.q0 + row.tok) * a.Hq + row.h;
  f16* o = a.o + at * D + 4 * kV * j0;
#pragma unroll
  for (int v = 0; v < kV; ++v)
    *reinterpret_cast<half4*>(o + 4 * v) = half4{(f16)(acc[v].x * inv), (f16)(acc[v].y * inv),
                                                 (f16)(acc[v].z * inv), (f16)(acc[v].w * inv)};
  if (a.lse != nullptr && j0 == 0u)
    a.lse[at] = l == 0.f ? -INFINITY : (m + __builtin_amdgcn_logf(l)) * kLn2;
}

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

// Workgroups of a call: those that fit on the chip at once, fewer where the
// call's bounds say that shares of `least` units need no more.
uint32_t workgroups(const ChunkArgs& a, uint64_t items, uint64_t tiles, uint32_t fit,
                    uint32_t least) {
  const uint64_t units = items * (tiles + kItemUnits) * a.H;
  const uint64_t n = (units + least - 1u) / least;
  const uint64_t m = n < fit ? n : fit;
  return (uint32_t)((m + kXcds - 1u) / kXcds * kXcds);
}

// The factors that divide by the page size, the group and n workgroups; the
// workspace holds the cuts, then the parts (there may be none: a.whole).
ChunkArgs with_rcps(const ChunkArgs& args, uint32_t n) {
  ChunkArgs a = args;
  a.G = a.Hq / a.H;
  a.page_rcp = a.S == 1u ? 0u : (uint32_t)((1ull << 32) / a.S) + 1u;
  a.group_rcp = ((1u << 31) + a.G - 1u) / a.G;
  a.share_rcp = 1.0 / (double)n;
  if (a.cuts != nullptr)
    a.parts = reinterpret_cast<float*>(static_cast<char*>(a.cuts) + kCutBytes);
  return a;
}

template <int D, int MOD, bool LIST>
hipError_t launch_attn(const ChunkArgs& a, uint32_t n, hipStream_t s) {
  if (a.S % 16u == 0u)
    hipLaunchKernelGGL((chunk_attn_kernel<D, MOD, true, LIST>), dim3(n), dim3(kChThreads), 0, s, a);
  else
    hipLaunchKernelGGL((chunk_attn_kernel<D, MOD, false, LIST>), dim3(n), dim3(kChThreads), 0, s,
                       a);
  return hipGetLastError();
}

template <int D, bool LIST>
hipError_t launch_attn(const ChunkArgs& a, uint32_t n, hipStream_t s) {
  switch ((a.soft_cap > 0.f ? kCap : 0) | (a.slopes != nullptr ? kBias : 0)) {
    case 0: return launch_attn<D, 0, LIST>(a, n, s);
    case kCap: return launch_attn<D, kCap, LIST>(a, n, s);
    case kBias: return launch_attn<D, kBias, LIST>(a, n, s);
    default: return launch_attn<D, kCap | kBias, LIST>(a, n, s);
  }
}

// Entries of a head's list at most: its items, and the parts of those cut (a
// part is longer than half a share, and all heads' shares fill the slots).
uint64_t list_entries(const ChunkArgs& a, uint32_t slots) {
  return (uint64_t)a.T * (a.Hq / a.H) / kChRows + a.B + 2u * slots / a.H + 1u;
}
// Whether a call has rows for so many items that they are listed (and a grid of
// 32-bit work-items holds their workgroups).  Both ways, us in shares / listed, at x
// items per workgroup that the GPU holds:
//                                        x = 0.5       1          1.5        2          4
//   prompt, 32 heads of 128              38 / 37     74 / 67   125 / 107  202 / 159  679 / 574
//   prompt, 16 of 256                    50 / 48    100 / 89   164 / 142  259 / 205  850 / 722
//   chunk after 8000, 32 / 8 of 128     170 / 193   333 / 388  516 / 542  710 / 679 1710 / 1615
//   chunk after 8000, 16 of 256         217 / 269   434 / 542  688 / 752  952 / 845 2269 / 2035
//   chunk after 8000, 32 of 64          114 / 117   227 / 224  359 / 311  487 / 445 1152 / 982
// So the list starts where prompts want it; chunks after a long context would have
// it from 2 on at 8 kv heads or head dim 256.  Fewer rows: a windowed batch of prompts, chunks and single
// tokens 110 / 134 in the kernel, drafted tokens after 16384 60 / 73.
bool lists_items(const ChunkArgs& a, uint32_t slots) {
  return (uint64_t)a.T * (a.Hq / a.H) / kChRows * a.H >= slots &&
         list_entries(a, slots) * a.H < (1u << 24);
}
template <int D>
constexpr uint32_t attn_slots() { return kCus * attn_per_cu<D>(); }
size_t list_bytes(const ChunkArgs& a, uint32_t slots) {
  return lists_items(a, slots) ? (list_entries(a, slots) * sizeof(Entry) + 255u) / 256u * 256u : 0u;
}

// Workgroups of a call whose items are not listed.
uint32_t share_workgroups(const ChunkArgs& a, uint32_t slots) {
  const uint64_t G = a.Hq / a.H;
  return workgroups(a, (a.T * G) / kChRows + a.B, ((uint64_t)a.max_pages * a.S) / kChTile + 2u,
                    slots, kAttnLeast);
}

template <int D>
hipError_t launch_attn(const ChunkArgs& args, hipStream_t s) {
  constexpr uint32_t kSlots = attn_slots<D>();
  if (!args.whole && lists_items(args, kSlots)) {
    const uint64_t n = list_entries(args, kSlots) * args.H;
    ChunkArgs a = with_rcps(args, kSlots);
    a.list = a.parts;
    a.parts = reinterpret_cast<float*>(reinterpret_cast<char*>(a.parts) + list_bytes(a, kSlots));
    hipLaunchKernelGGL(chunk_list_kernel, dim3(1), dim3(kChThreads), 0, s, a, kSlots,
                       (uint32_t)(n / a.H));
    if (hipError_t e = hipGetLastError(); e != hipSuccess) return e;
    if (hipError_t e = launch_attn<D, true>(a, (uint32_t)n, s); e != hipSuccess) return e;
    hipLaunchKernelGGL((chunk_join_kernel<D, true>), dim3((kSlots / a.H + 1u) * a.H * 4u),
                       dim3(kChThreads), 0, s, a);
    return hipGetLastError();
  }
  const uint32_t n = share_workgroups(args, kSlots);
  const ChunkArgs a = with_rcps(args, n);
  if (hipError_t e = launch_attn<D, false>(a, n, s); e != hipSuccess || a.whole) return e;
  hipLaunchKernelGGL((chunk_join_kernel<D, false>), dim3((n - 1u) * 4u), dim3(kChThreads), 0, s, a);
  return hipGetLastError();
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
    case 64: return launch_attn<64>(a, s);
    case 128: return launch_attn<128>(a, s);
    default: return launch_attn<256>(a, s);
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
