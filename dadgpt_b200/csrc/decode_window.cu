// Decode attention over part of a cache, over an 8-bit cache, and with the attention weights added up.
//
//   out = sum_j p_j v_j,  p_j = exp(s_j - m) / l,  s_j = scale q.k_j,  m = max s_j,  l = sum exp(s_j - m)
//
// over the rows j that the token at row L (the sequence's length) sees: j <= L and (L - j < window or j < sinks). One pass
// over the visible rows with a running maximum and sum; the others are not read. It is decode.cu's kernel in another
// form: a producer thread per CTA streams the rows through a ring of 16 KB stages, four consumer warps compute, persistent
// CTAs or clusters, a counter that hands out items and tickets for the lengths. What differs is that an item is a list of
// tiles, so that the rows need not be one range:
//   bf16 cache    tiles of the first rows, then of the window's
//   8-bit cache   the same from blocks of 64 tokens (fp8_block.cuh), whose scales travel with the tile, then the open
//                 block's rows, which are bf16, from the tail buffer. The token goes to the tail; where it fills it, the
//                 CTA that appended it turns it into a block behind the item's arithmetic: every block is rounded once,
//                 from bf16, and holds the same bytes whether a prompt filled it or single tokens did.
// Weights: a row's score is written to scratch as it is formed; once the item's m and l are known the CTA that formed it
// adds exp(s - m) / l to the row's weight. 16 bytes a row (the score out and, from L2, in again; the weight in and out) beside
// 4 D of K and V.
//
// Measured in a graph of such calls on rotating caches (us; 64 x 12 heads of 64, 4 x 24 of 128):
//   64 sequences of 9 .. 1017 rows   bf16 21.8 (4.6 TB/s), with weights 25.3, 8 bits 18.5 (2.7 TB/s)
//   64 of 1000                       bf16 35.7 (5.5 TB/s), with weights 42.0; 8 bits, 1024 rows, 26.2 (3.8 TB/s)
//   64 of 600, window 256            13.3 (3.8 TB/s)
//   4 of 4000                        bf16 34.3 (5.7 TB/s), with weights 38.8, 8 bits 25.2 (3.9 TB/s); one of 650: 4.7 either way
// The 8-bit form is at no unit's limit (HBM 41 %, issue slots 53 %): its time is the start and end of a call, 4.4 us of the
// 18.5 to the first tile, and in between waits of few warps for their own earlier steps (2.4 cycles an instruction for memory,
// 1.4 for results). It executes 5.8 instructions for a cached element, where two conversions to a pair and the product are 2 to
// 2.5: tiles whose last rows are missing are computed whole, and every item is merged and ranked. Its persistent instances
// spill (94 registers, 128 bytes out and 160 in). Tried for it and not faster: rings of every warp's own filled by 16-byte
// copies (20-22 us), both products by warp-wide matrix instructions (20-29) or K's alone (19.7), even shares of all rows for
// every CTA with partial results in memory (25-34), two consumer warps with 4 KB tiles (26).
#include <cuda_bf16.h>

#include <cfloat>
#include <climits>
#include <cstddef>

#include <algorithm>
#include <initializer_list>
#include <type_traits>

#include "common.cuh"
#include "decode_common.cuh"
#include "fp8_block.cuh"
#include "sm100_ptx.cuh"

namespace dadattn {
namespace {

using namespace ptx;
using bf16 = __nv_bfloat16;

constexpr int kWarps = 4;                     // consumer warps
constexpr int kThreads = (kWarps + 1) * 32;   // and one producer warp
constexpr int kTileBytes = 8192;              // K (and V) bytes of one ring stage
constexpr int kFewStages = 4, kFewPerSm = 3;
constexpr int kManyStages = 3, kManyPerSm = 4;
constexpr int kMaxStages = 4;
constexpr int kItemRing = 2;                  // items a CTA's producer may be ahead
constexpr int kMaxCluster = 8;
constexpr int kMaxPaired = 64;                // sequences of a call up to which clusters share two

// The workspace: the item counter and 1 + kTicketGroups counters of the lengths' tickets (uint32, zero between calls), in
// the space that decode.cu has for its own, so that the calls of both can share a workspace; with weights, the scores
// [B, H, max_len] fp32 behind that.
size_t counter_bytes(int B, int H) {
  return (sizeof(uint32_t) * (static_cast<size_t>(B) * H + 1 + kTicketGroups) + 255) / 256 * 256;
}
size_t window_workspace_bytes(int B, int H, int max_len, bool weights) {
  return counter_bytes(B, H) + (weights ? static_cast<size_t>(B) * H * max_len * sizeof(float) : 0);
}

struct Shared {
  uint64_t full[kMaxStages], empty[kMaxStages];
  uint64_t item_ready[kItemRing], item_free[kItemRing];
  int item[kItemRing];
  int abort_flag;
  float scales[kMaxStages][4];           // 8-bit tiles: K, K of the second block, V, V of the second block
  float m[kWarps], l[kWarps];
  __align__(16) float acc[kWarps][128];   // (written as pairs)
  __align__(16) int lens[kMaxRanked];
  union {
    struct {
      int place[kMaxRanked];
      int order[kMaxRanked];
    };
    float record[kMaxCluster][130];      // clusters: every CTA's partial result, in the CTA that merges it
  };
  int2 member[2];                        // paired: (sequence or -1, length)
  float2 state[kMaxCluster];             // clusters with weights: every CTA's (m, l), in every CTA
};

static_assert(offsetof(Shared, acc) % 8 == 0 && offsetof(Shared, lens) % 16 == 0 && offsetof(Shared, state) % 8 == 0,
              "alignment of wide accesses");

struct Params {
  bf16* out;
  const bf16 *q, *k_new, *v_new;
  void *k, *v;               // caches [B, H, max_len, D]
  float *k_scale, *v_scale;  // 8-bit: [B, H, blocks]
  bf16 *k_tail, *v_tail;     // 8-bit: [B, H, 64, D]
  int32_t* lengths;
  float *weights, *scores;   // [B, H, max_len]
  unsigned* counters;
  int* status;
  int B, H, max_len, blocks, window, sinks;
  int ranks, stages, reorder, paired;
  float scale;
};

// Copies of 4 bytes that the calling thread makes, and its arrival at `bar` once all of them so far have landed (one of the
// arrivals that the barrier was set up for).
__device__ __forceinline__ void copy_4_bytes(void* smem_dst, const void* src) {
  asm volatile("cp.async.ca.shared.global [%0], [%1], 4;" ::"r"(smem_u32(smem_dst)), "l"(src) : "memory");
}
__device__ __forceinline__ void arrive_behind_copies(uint64_t* bar) {
  asm volatile("cp.async.mbarrier.arrive.noinc.shared::cta.b64 [%0];" ::"r"(smem_u32(bar)) : "memory");
}
__device__ __forceinline__ void consumers_sync() { asm volatile("bar.sync 1, %0;" ::"n"(kWarps * 32) : "memory"); }
// The same, and whether any consumer thread brought a true one.
__device__ __forceinline__ bool consumers_any(bool mine) {
  uint32_t any;
  asm volatile(
      "{\n\t.reg .pred p, q;\n\tsetp.ne.u32 p, %1, 0;\n\t"
      "bar.red.or.pred q, 2, %2, p;\n\tselp.u32 %0, 1, 0, q;\n\t}"
      : "=r"(any)
      : "r"(static_cast<uint32_t>(mine)), "n"(kWarps * 32)
      : "memory");
  return any != 0;
}

// Elements of a row that a lane holds, as float pairs: from a bf16 row 16 bytes (8 elements), from an 8-bit one 16 bytes
// (16 elements), and 32 bytes of bf16 for rows of the tail, so that a lane has the same elements of both.
template <bool FP8>
struct Lane {
  static constexpr int kElems = FP8 ? 16 : 8;
};
__device__ __forceinline__ void unpack_fp8(float2 (&f)[8], const uint4& raw) {
  const uint32_t w[4] = {raw.x, raw.y, raw.z, raw.w};
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    f[2 * i] = __half22float2(__half2(__nv_cvt_fp8x2_to_halfraw2(static_cast<__nv_fp8x2_storage_t>(w[i] & 0xffffu), __NV_E4M3)));
    f[2 * i + 1] = __half22float2(__half2(__nv_cvt_fp8x2_to_halfraw2(static_cast<__nv_fp8x2_storage_t>(w[i] >> 16), __NV_E4M3)));
  }
}

// The visible rows of a sequence of `len` rows as tiles.
template <bool FP8, int D>
struct View {
  static constexpr int kRows = kTileBytes / (FP8 ? D : 2 * D);   // rows of a tile of the cache
  static constexpr int kTailRows = kTileBytes / (2 * D);         // and of the tail
  int len, full;      // rows in all, rows that lie in the cache itself
  int first, sinks;   // the window begins at `first`; the rows below `sinks` <= first are seen as well
  int a, b, t;        // tiles of the first rows, of the window's, of the tail

  __device__ __forceinline__ View(int len_, int window, int sinks_) : len(len_) {
    full = FP8 ? len / kFp8Block * kFp8Block : len;
    first = window > 0 ? max(len + 1 - window, 0) : 0;
    sinks = min(sinks_, first);
    if (sinks == first) first = sinks = 0;   // no gap
    a = (min(sinks, full) + kRows - 1) / kRows;
    b = first < full ? (full - base_b() + kRows - 1) / kRows : 0;
    t = (len - full + kTailRows - 1) / kTailRows;
  }
  __device__ __forceinline__ int base_b() const { return FP8 ? first / kFp8Block * kFp8Block : first; }   // tiles hold whole blocks
  __device__ __forceinline__ int tiles() const { return a + b + t; }

  // Tile i: rows lo .. hi - 1, the first of its places being row `base`.
  struct Tile {
    int base, lo, hi;
    bool tail;
  };
  __device__ __forceinline__ Tile tile(int i) const {
    Tile r;
    r.tail = FP8 && i >= a + b;
    if (i < a) {
      r.base = r.lo = i * kRows;
      r.hi = min(r.base + kRows, min(sinks, full));
    } else if (!r.tail) {
      r.base = base_b() + (i - a) * kRows;
      r.lo = max(r.base, first);
      r.hi = min(r.base + kRows, full);
    } else {
      r.base = r.lo = full + (i - a - b) * kTailRows;
      r.hi = min(r.base + kTailRows, len);
    }
    return r;
  }
  __device__ __forceinline__ bool sees(const Tile& r, int row) const {
    return row >= r.lo && row < r.hi && (row < sinks || row >= first);
  }
};

template <bool FP8, int D, bool CLUSTER, bool WEIGHTS>
__global__ void __launch_bounds__(kThreads, kManyPerSm) decode_window_kernel(const __grid_constant__ Params p) {
  using V = View<FP8, D>;
  constexpr int EPL = Lane<FP8>::kElems;
  constexpr int LPK = D / EPL;            // lanes per row
  constexpr int KPI = 32 / LPK;           // rows per warp instruction
  constexpr int kGroups = V::kRows / (kWarps * KPI);           // row groups of a tile per warp
  constexpr int kTailGroups = V::kTailRows / (kWarps * KPI);   // and of a tail's tile
  constexpr int kRowBytes = FP8 ? D : 2 * D;
  static_assert(kGroups * kWarps * KPI == V::kRows && kTailGroups * kWarps * KPI == V::kTailRows, "tile split");
  static_assert(!FP8 || (V::kRows / kWarps <= kFp8Block && kFp8Block % (V::kRows / kWarps) == 0 && V::kRows <= 2 * kFp8Block),
                "a warp's rows of a tile are of one block");
  constexpr float kUnit = Elem<bf16>::kUnit;   // scores in log2 units

  extern __shared__ __align__(128) uint8_t smem[];
  const int ranks = CLUSTER ? p.ranks : 1, stages = p.stages;
  Shared& sh = *reinterpret_cast<Shared*>(smem + stages * 2 * kTileBytes);
  const int warp = __shfl_sync(0xffffffffu, static_cast<int>(threadIdx.x / 32), 0);
  const int lane = threadIdx.x % 32;
  const int rank = static_cast<int>(blockIdx.x) % ranks;
  const int B = p.B, H = p.H, max_len = p.max_len;

  if (threadIdx.x == 0) {
    for (int i = 0; i < stages; ++i) {
      mbar_init(&sh.full[i], FP8 ? 2 : 1);
      mbar_init(&sh.empty[i], kWarps);
    }
    for (int i = 0; i < kItemRing; ++i) {
      mbar_init(&sh.item_ready[i], 1);
      mbar_init(&sh.item_free[i], kWarps);
    }
    sh.abort_flag = 0;
    fence_mbar_init();
  }
  pdl_wait();
  pdl_launch_dependents();

  // Up to kMaxRanked lengths are copied first; nobody reads the caller's array after that.
  const bool snapshot = B <= kMaxRanked;
  if (snapshot)
    for (int i = threadIdx.x; i < kMaxRanked; i += kThreads) {
      sh.lens[i] = i < B ? p.lengths[i] : INT_MIN;
      if (!CLUSTER && p.reorder) sh.place[i] = 0;
    }
  if (CLUSTER && threadIdx.x < 2) sh.member[threadIdx.x] = make_int2(-1, 0);
  __syncthreads();
  if (!CLUSTER && p.reorder) rank_by_length(sh.lens, sh.place, sh.order, B, kThreads);
  if (CLUSTER) cluster_arrive();   // "this CTA has started": waited for before the first remote store

  // Item e of the call and this CTA's tiles t0 .. t1 - 1 of it. A sequence whose length is outside [0, max_len) is skipped
  // (no tiles, no token) and reported.
  struct Item {
    int b, h, len, t0, t1;
    bool good;
  };
  const int n_items = B * H, n_lanes = static_cast<int>(gridDim.x);
  // CTA `share` of the `shares` that share sequence b's head h
  auto share_of = [&](int b, int h, int len, int share, int shares) -> Item {
    Item s{b, h, len, 0, 0, len >= 0 && len < max_len};
    if (!s.good) {
      s.len = 0;
    } else {
      const int n = V(len, p.window, p.sinks).tiles();
      // (64 bits: not needed by any cache that fits the GPU, and free here)
      s.t0 = static_cast<int>(static_cast<long long>(n) * share / shares);
      s.t1 = static_cast<int>(static_cast<long long>(n) * (share + 1) / shares);
    }
    return s;
  };
  int share = rank, shares = ranks;             // this CTA among those that share its sequence
  int merges = rank == 0 ? 0 : -1, from = 0;    // clusters: which of its sequences a CTA merges, whose first CTA has rank `from`
  auto item = [&](int e) -> Item {
    const int place = e / H, b = !CLUSTER && p.reorder ? sh.order[place] : place;
    return share_of(b, e - place * H, snapshot ? sh.lens[b] : p.lengths[b], share, shares);
  };
  Item first, merged;
  bool second = false;                          // whether the CTA's share is of its cluster's second sequence
  if (!CLUSTER || !p.paired) {
    first = merged = item(static_cast<int>(blockIdx.x) / ranks);
  } else {
    // Cluster c takes head c % H of the c / H-th longest and the c / H-th shortest sequence (one, in the middle of an odd
    // number), as decode.cu's; its CTAs are divided by their tiles, so that the largest share is as small as it can be.
    const int e = static_cast<int>(blockIdx.x) / ranks, nth = e / H, h = e - nth * H, t = threadIdx.x;
    if (t < B) {
      const int mine = sh.lens[t];
      int place = 0;
#pragma unroll 4
      for (int j = 0; j < B; ++j)
        place += static_cast<int>(sh.lens[j] > mine) | (static_cast<int>(sh.lens[j] == mine) & static_cast<int>(j < t));
      if (place == nth) sh.member[0] = make_int2(t, mine);
      else if (place == B - 1 - nth) sh.member[1] = make_int2(t, mine);
    }
    __syncthreads();
    const int2 a = sh.member[0], b = sh.member[1];
    auto tiles_of = [&](const int2& x) { return x.x >= 0 && x.y >= 0 && x.y < max_len ? V(x.y, p.window, p.sinks).tiles() + 1 : 0; };
    const int tiles_a = tiles_of(a), tiles_b = tiles_of(b);
    int cut = b.x < 0 || tiles_b == 0 ? ranks : 0;   // CTAs for the first
    if (tiles_a > 0 && tiles_b > 0) {
      // the whole number below or above what is in proportion, whichever has the smaller largest share
      const float fa = static_cast<float>(tiles_a), fb = static_cast<float>(tiles_b);
      const int below = min(max(static_cast<int>(__fdividef(fa * ranks, fa + fb)), 1), ranks - 1), above = min(below + 1, ranks - 1);
      cut = fa * (ranks - above) <= fb * below ? below : above;
    }
    second = rank >= cut;
    share = second ? rank - cut : rank;
    shares = second ? ranks - cut : cut;
    first = second ? share_of(b.x, h, b.y, share, shares) : share_of(a.x, h, a.y, share, shares);
    merges = rank == 0 ? 0 : rank == 1 && b.x >= 0 ? 1 : -1;
    merged = merges == 1 ? share_of(b.x, h, b.y, 0, max(ranks - cut, 1)) : share_of(a.x, h, a.y, 0, max(cut, 1));
    from = merges == 1 ? cut : 0;
  }
  const int merged_shares = CLUSTER && p.paired ? (merges == 1 ? ranks - from : second ? 0 : shares) : ranks;

  const LengthTickets tickets{p.counters + 1};
  volatile int* abort_flag = &sh.abort_flag;
  if (warp == kWarps) {
    // ------------------------------ producer ------------------------------
    if (elect_one()) {
      bool ticket_due = snapshot;
      const unsigned ticket = ticket_due ? tickets.draw() : 0;
      auto settle_ticket = [&]() {
        if (ticket_due && tickets.is_last(ticket))
          for (int j = 0; j < B; ++j) {
            const int len = sh.lens[j];
            if (len >= 0 && len < max_len) p.lengths[j] = len + 1;   // a full or invalid sequence is left alone
          }
        ticket_due = false;
      };
      // One claim per item beyond the CTAs' first ones and one per CTA that finds nothing left: n_items in all, of which the
      // last returns the counter to zero.
      auto claim = [&]() -> int {
        if (CLUSTER || n_lanes >= n_items) return n_items;
        const unsigned c = atomicAdd(p.counters, 1u);
        if (c == static_cast<unsigned>(n_items - 1)) *p.counters = 0;
        return min(static_cast<int>(c) + n_lanes, n_items);
      };
      int st = 0, lap = 0, next = 0;
      Item s = first;
      bool ok = true;
      for (int n = 0; ok; ++n) {
        const size_t bh = static_cast<size_t>(s.b) * H + s.h;
        const V view(s.len, p.window, p.sinks);
        const uint8_t* kc = static_cast<const uint8_t*>(p.k) + bh * max_len * kRowBytes;
        const uint8_t* vc = static_cast<const uint8_t*>(p.v) + bh * max_len * kRowBytes;
        for (int t = s.t0; t < s.t1; ++t) {
          if (lap == 1 && st == 0) settle_ticket();
          if (lap > 0 && !(ok = mbar_wait(&sh.empty[st], (lap - 1) & 1, abort_flag))) break;
          const typename V::Tile r = view.tile(t);
          uint8_t* ks = smem + st * 2 * kTileBytes;
          if (r.tail) {
            const size_t at = (bh * kFp8Block + (r.lo - view.full)) * D;
            const uint32_t bytes = static_cast<uint32_t>(r.hi - r.lo) * 2 * D;
            mbar_arrive_expect_tx(&sh.full[st], 2 * bytes);
            bulk_load(ks, p.k_tail + at, bytes, &sh.full[st]);
            bulk_load(ks + kTileBytes, p.v_tail + at, bytes, &sh.full[st]);
            arrive_behind_copies(&sh.full[st]);
          } else {
            const uint32_t bytes = static_cast<uint32_t>(r.hi - r.lo) * kRowBytes, skip = static_cast<uint32_t>(r.lo - r.base) * kRowBytes;
            mbar_arrive_expect_tx(&sh.full[st], 2 * bytes);
            bulk_load(ks + skip, kc + static_cast<size_t>(r.lo) * kRowBytes, bytes, &sh.full[st]);
            bulk_load(ks + kTileBytes + skip, vc + static_cast<size_t>(r.lo) * kRowBytes, bytes, &sh.full[st]);
            if (FP8) {
              const size_t block = bh * p.blocks + r.base / kFp8Block;
#pragma unroll
              for (int i = 0; i < V::kRows / kFp8Block; ++i)
                if (r.base + i * kFp8Block < r.hi) {   // (a block that the tile has none of may not be there)
                  copy_4_bytes(&sh.scales[st][i], p.k_scale + block + i);
                  copy_4_bytes(&sh.scales[st][2 + i], p.v_scale + block + i);
                }
              arrive_behind_copies(&sh.full[st]);
            }
          }
          if (++st == stages) st = 0, ++lap;
        }
        // The item after this one is claimed only when this one's last rows are on their way (decode.cu).
        if (ok) next = claim();
        const int slot = n % kItemRing;
        ok = ok && (n < kItemRing || mbar_wait(&sh.item_free[slot], (n / kItemRing - 1) & 1, abort_flag));
        if (!ok) break;
        *reinterpret_cast<volatile int*>(&sh.item[slot]) = next;
        mbar_arrive(&sh.item_ready[slot]);
        if (next >= n_items) break;
        s = item(next);
      }
      // After a wait that ran out the claims are made all the same: the workspace stays usable.
      while (next < n_items) next = claim();
      settle_ticket();
      settle_ring(sh.full, stages, lap * stages + st);
    }
  } else {
    // ------------------------------ consumers ------------------------------
    const int slot = lane / LPK, part = lane % LPK;
    const float scale_unit = p.scale * kUnit;
    int st = 0;
    uint32_t phase = 0;
    bool ok = true;
    Item s = first, nxt = first;
    bool have = true;
    constexpr int kRaw = FP8 ? 2 : 1;   // 16-byte pieces of bf16 per lane and row
    // token vectors of an item: fetched an item ahead (k_new / v_new by the warp that appends)
    uint4 q_raw[kRaw], kn_raw[kRaw], vn_raw[kRaw];
#pragma unroll
    for (int i = 0; i < kRaw; ++i) kn_raw[i] = vn_raw[i] = make_uint4(0, 0, 0, 0);
    auto fetch_token = [&](const Item& t) {
      const size_t off = (static_cast<size_t>(t.b) * H + t.h) * D + part * EPL;
#pragma unroll
      for (int i = 0; i < kRaw; ++i) {
        q_raw[i] = reinterpret_cast<const uint4*>(p.q + off)[i];
        if (warp == 0 && slot == 0) {
          kn_raw[i] = reinterpret_cast<const uint4*>(p.k_new + off)[i];
          vn_raw[i] = reinterpret_cast<const uint4*>(p.v_new + off)[i];
        }
      }
    };
    fetch_token(s);
    for (int n = 0; have; ++n, s = nxt) {
      const size_t bh = static_cast<size_t>(s.b) * H + s.h;
      const V view(s.len, p.window, p.sinks);
      float m = -FLT_MAX, l = 0.f;
      float2 acc[EPL / 2], qf[EPL / 2];
      auto unpack_bf16 = [](float2 (&f)[EPL / 2], const uint4* raw) {
#pragma unroll
        for (int i = 0; i < kRaw; ++i) {
          float2 x[4];
          Elem<bf16>::unpack(x, raw[i]);
#pragma unroll
          for (int e = 0; e < 4; ++e) f[4 * i + e] = x[e];
        }
      };
      if (FP8) unpack_bf16(qf, q_raw);
      // q k of a lane's part of a row: bf16 without a conversion (64 x 12 heads of 64, 512 rows each: 23.1 -> 22.2 us, with
      // weights and 1000 rows 45.1 -> 42.0), 8-bit rows as fp32. (Those as f16, with q scaled to f16 once, was 2 % faster on
      // some calls and 3 % slower on others.)
      auto dot_of = [&](const auto& k, auto unpack) -> float {
        float2 dot = make_float2(0.f, 0.f);
        if constexpr (FP8) {
          float2 kf[EPL / 2];
          unpack(kf, k);
#pragma unroll
          for (int e = 0; e < EPL / 2; ++e) dot = ffma2(qf[e], kf[e], dot);
        } else {
          const uint4 &qx = q_raw[0], &kx = *reinterpret_cast<const uint4*>(&k.x);   // (one piece, whichever way it came)
          const uint32_t a[4] = {qx.x, qx.y, qx.z, qx.w}, b[4] = {kx.x, kx.y, kx.z, kx.w};
#pragma unroll
          for (int e = 0; e < 4; ++e) fma_bf16(dot, a[e], b[e]);
        }
        return dot.x + dot.y;
      };
#pragma unroll
      for (int e = 0; e < EPL / 2; ++e) acc[e] = make_float2(0.f, 0.f);
      float* scores = WEIGHTS ? p.scores + bh * max_len : nullptr;

      // NR row groups into the lane's state, without branches (decode.cu). `row(u)`: the lane's row of group u. Rows that do
      // not count come in as zeros. ks, vs: the block's scales.
      auto absorb = [&](const auto& kr, const auto& vr, auto unpack, const bool* valid, auto count, auto all, float ks, float vs,
                        auto row) {
        constexpr int NR = decltype(count)::value;
        constexpr bool ALL = decltype(all)::value;
        float sc[NR], pr[NR];
#pragma unroll
        for (int u = 0; u < NR; ++u) sc[u] = dot_of(kr[u], unpack);
#pragma unroll
        for (int o = LPK / 2; o > 0; o >>= 1)
#pragma unroll
          for (int u = 0; u < NR; ++u) sc[u] += __shfl_xor_sync(0xffffffffu, sc[u], o);
        float m_new = m;
#pragma unroll
        for (int u = 0; u < NR; ++u) {
          sc[u] = ALL || valid[u] ? sc[u] * ks : -FLT_MAX;
          m_new = fmaxf(m_new, sc[u]);
          if (WEIGHTS && part == 0 && (ALL || valid[u])) scores[row(u)] = sc[u];
        }
        // (while m_new is still -FLT_MAX the state is all zeros: corr = 1 leaves it so)
        const float corr = ex2(m - m_new);
        float sum = 0.f;
#pragma unroll
        for (int u = 0; u < NR; ++u) {
          pr[u] = ex2(sc[u] - m_new);
          if (!ALL && !valid[u]) pr[u] = 0.f;
          sum += pr[u];
        }
        l = fmaf(l, corr, sum);
#pragma unroll
        for (int e = 0; e < EPL / 2; ++e) acc[e] = fmul2(acc[e], make_float2(corr, corr));
#pragma unroll
        for (int u = 0; u < NR; ++u) {
          float2 vf[EPL / 2];
          unpack(vf, vr[u]);
          const float w = FP8 ? pr[u] * vs : pr[u];
#pragma unroll
          for (int e = 0; e < EPL / 2; ++e) acc[e] = ffma2(make_float2(w, w), vf[e], acc[e]);
        }
        m = m_new;
      };
      struct Raw {   // a lane's piece of a bf16 row
        uint4 x[kRaw];
      };
      auto unpack_raw = [&](float2 (&f)[EPL / 2], const Raw& r) { unpack_bf16(f, r.x); };
      using One = std::integral_constant<int, 1>;

      // the token being appended: its vectors are used and stored by the CTA of the last share
      if (warp == 0 && s.good && share == shares - 1) {
        const bool mine = slot == 0;
        Raw kr[1], vr[1];
#pragma unroll
        for (int i = 0; i < kRaw; ++i) kr[0].x[i] = kn_raw[i], vr[0].x[i] = vn_raw[i];
        if (mine) {
          const size_t at = FP8 ? (bh * kFp8Block + s.len % kFp8Block) * D : (bh * max_len + s.len) * D;
          bf16* kd = (FP8 ? p.k_tail : static_cast<bf16*>(p.k)) + at + part * EPL;
          bf16* vd = (FP8 ? p.v_tail : static_cast<bf16*>(p.v)) + at + part * EPL;
#pragma unroll
          for (int i = 0; i < kRaw; ++i) {
            reinterpret_cast<uint4*>(kd)[i] = kn_raw[i];
            reinterpret_cast<uint4*>(vd)[i] = vn_raw[i];
          }
        }
        absorb(kr, vr, unpack_raw, &mine, One{}, std::false_type{}, scale_unit, 1.f, [&](int) { return s.len; });
      }
      for (int t = s.t0; t < s.t1; ++t) {
        if (!ok || !(ok = mbar_wait(&sh.full[st], phase, abort_flag))) break;
        const typename V::Tile r = view.tile(t);
        const uint8_t* kt = smem + st * 2 * kTileBytes;
        const uint8_t* vt = kt + kTileBytes;
        if (FP8 && r.tail) {
          Raw kr[kTailGroups], vr[kTailGroups];
          bool valid[kTailGroups];
          auto row = [&](int u) { return r.base + (warp * kTailGroups + u) * KPI + slot; };
#pragma unroll
          for (int u = 0; u < kTailGroups; ++u) {
            const int at = ((warp * kTailGroups + u) * KPI + slot) * 2 * D + part * 32;
            valid[u] = view.sees(r, row(u));
#pragma unroll
            for (int i = 0; i < kRaw; ++i) {
              kr[u].x[i] = valid[u] ? *reinterpret_cast<const uint4*>(kt + at + 16 * i) : make_uint4(0, 0, 0, 0);
              vr[u].x[i] = valid[u] ? *reinterpret_cast<const uint4*>(vt + at + 16 * i) : make_uint4(0, 0, 0, 0);
            }
          }
          absorb(kr, vr, unpack_raw, valid, std::integral_constant<int, kTailGroups>{}, std::false_type{}, scale_unit, 1.f, row);
        } else {
          struct Row {
            uint4 x;
          };
          Row kr[kGroups], vr[kGroups];
          const int at = (warp * kGroups * 32 + lane) * 16;
#pragma unroll
          for (int u = 0; u < kGroups; ++u) kr[u].x = *reinterpret_cast<const uint4*>(kt + at + u * 512);
#pragma unroll
          for (int u = 0; u < kGroups; ++u) vr[u].x = *reinterpret_cast<const uint4*>(vt + at + u * 512);
          float ks = scale_unit, vs = 1.f;
          if (FP8) {
            const int i = warp * (V::kRows / kWarps) / kFp8Block;           // the warp's block within the tile
            if (V::kRows == kFp8Block || r.base + i * kFp8Block < r.hi) {   // (of one without a row no scale was loaded)
              ks *= sh.scales[st][i];
              vs = sh.scales[st][2 + i];
            }
          }
          auto unpack = [&](float2 (&f)[EPL / 2], const Row& w) {
            if constexpr (FP8) unpack_fp8(f, w.x);
            else unpack_bf16(f, &w.x);
          };
          auto row = [&](int u) { return r.base + (warp * kGroups + u) * KPI + slot; };
          using Count = std::integral_constant<int, kGroups>;
          if (r.hi - r.lo == V::kRows) {
            absorb(kr, vr, unpack, nullptr, Count{}, std::true_type{}, ks, vs, row);
          } else {   // what lies beside the rows loaded is left over from earlier tiles
            bool valid[kGroups];
#pragma unroll
            for (int u = 0; u < kGroups; ++u) {
              valid[u] = view.sees(r, row(u));
              if (!valid[u]) kr[u].x = vr[u].x = make_uint4(0, 0, 0, 0);
            }
            absorb(kr, vr, unpack, valid, Count{}, std::false_type{}, ks, vs, row);
          }
        }
        __syncwarp();
        if (lane == 0) mbar_arrive(&sh.empty[st]);
        if (++st == stages) st = 0, phase ^= 1;
      }

      // the next item; its token vectors arrive while this one is merged
      have = false;
      if (!CLUSTER) {
        const int slot_i = n % kItemRing;
        if (ok && (ok = mbar_wait(&sh.item_ready[slot_i], (n / kItemRing) & 1, abort_flag))) {
          const int e = *reinterpret_cast<volatile int*>(&sh.item[slot_i]);
          __syncwarp();
          if (lane == 0) mbar_arrive(&sh.item_free[slot_i]);
          if ((have = e < n_items)) {
            nxt = item(e);
            fetch_token(nxt);
          }
        }
      }

      // Merge the KPI row slots of the warp (lanes with equal `part`), then the warps.
#pragma unroll
      for (int o = LPK; o < 32; o <<= 1) {
        const float m_o = __shfl_xor_sync(0xffffffffu, m, o);
        const float l_o = __shfl_xor_sync(0xffffffffu, l, o);
        const float m_new = fmaxf(m, m_o);
        const float ca = m > -FLT_MAX ? ex2(m - m_new) : 0.f;
        const float cb = m_o > -FLT_MAX ? ex2(m_o - m_new) : 0.f;
        l = l * ca + l_o * cb;
#pragma unroll
        for (int e = 0; e < EPL / 2; ++e) {
          acc[e].x = acc[e].x * ca + __shfl_xor_sync(0xffffffffu, acc[e].x, o) * cb;
          acc[e].y = acc[e].y * ca + __shfl_xor_sync(0xffffffffu, acc[e].y, o) * cb;
        }
        m = m_new;
      }
      if (slot == 0) {
#pragma unroll
        for (int e = 0; e < EPL / 2; ++e)
          *reinterpret_cast<float2*>(&sh.acc[warp][part * EPL + 2 * e]) = acc[e];
        if (part == 0) {
          sh.m[warp] = m;
          sh.l[warp] = l;
        }
      }
      // The warps go on with one `ok`: barriers follow that only an item in order has. (The scores and the appended row are
      // there for the whole CTA, too.)
      ok = !consumers_any(!ok);
      const int d = threadIdx.x;
      float mm = -FLT_MAX, ll = 0.f;
#pragma unroll
      for (int w = 0; w < kWarps; ++w) mm = fmaxf(mm, sh.m[w]);
      float c[kWarps];
#pragma unroll
      for (int w = 0; w < kWarps; ++w) {
        c[w] = sh.m[w] > -FLT_MAX ? ex2(sh.m[w] - mm) : 0.f;
        ll += sh.l[w] * c[w];
      }
      if (d < D) {
        float aa = 0.f;
#pragma unroll
        for (int w = 0; w < kWarps; ++w) aa += sh.acc[w][d] * c[w];
        if (!CLUSTER) {
          if (s.good) p.out[bh * D + d] = Elem<bf16>::from_float(aa / ll);
        } else {
          // hand the share to the CTA that merges it, which is known to run once the cluster's first barrier is through
          cluster_wait();
          const uint32_t rec = cluster_address(&sh.record[rank][0], second ? 1 : 0);
          st_cluster(rec + d * 4, aa);
          if (d == 0) {
            st_cluster(rec + D * 4, mm);
            st_cluster(rec + D * 4 + 4, ll);
          }
          if (WEIGHTS && d < ranks) {
            const uint32_t to = cluster_address(&sh.state[rank], d);
            st_cluster(to, mm);
            st_cluster(to + 4, ll);
          }
        }
      }
      auto add_weights = [&](float m_all, float l_all) {
        const float inv = 1.f / l_all;
        float* weights = p.weights + bh * max_len;
        // Several rows of a thread on their way together. One after the other 4 x 24 heads of 128 (clusters), 4000 rows, took
        // 41.7 us, so 39; 64 x 12 heads of 64, 1000 rows, 47.5 / 45.0 (42.0 with the bf16 products; with 8 at a time 48.2: the
        // next item's vectors are spilt).
        constexpr int kAhead = CLUSTER ? 8 : 4;
        auto rows = [&](int from, int to) {
          for (int j = from + d; j < to; j += kAhead * kWarps * 32) {
            float sc[kAhead], w[kAhead];
#pragma unroll
            for (int u = 0; u < kAhead; ++u)
              if (j + u * kWarps * 32 < to) {
                sc[u] = scores[j + u * kWarps * 32];
                w[u] = weights[j + u * kWarps * 32];
              }
#pragma unroll
            for (int u = 0; u < kAhead; ++u)
              if (j + u * kWarps * 32 < to) weights[j + u * kWarps * 32] = w[u] + ex2(sc[u] - m_all) * inv;
          }
        };
        rows(min(s.t0, view.a) * V::kRows, min(min(s.t1, view.a) * V::kRows, view.sinks));
        rows(view.first + max(s.t0 - view.a, 0) * V::kRows,
             min(view.first + max(s.t1 - view.a, 0) * V::kRows, s.len));
        if (share == shares - 1 && d == 0) weights[s.len] = ex2(scores[s.len] - m_all) * inv;
      };
      if (WEIGHTS && !CLUSTER && s.good && ok) add_weights(mm, ll);
      if (WEIGHTS && CLUSTER) {
        // the others' (m, l): behind the cluster's second barrier, which the producer warp and the threads beyond D join below
        if (d >= D) cluster_wait();
        cluster_arrive();
        cluster_wait();
        if (s.good && ok) {
          float m_all = -FLT_MAX, l_all = 0.f;
          const int j0 = rank - share;
          for (int j = j0; j < j0 + shares; ++j) m_all = fmaxf(m_all, sh.state[j].x);
          for (int j = j0; j < j0 + shares; ++j) l_all += sh.state[j].y * ex2(sh.state[j].x - m_all);
          add_weights(m_all, l_all);
        }
      }
      // the token filled the tail: it becomes a block
      if (FP8 && s.good && ok && share == shares - 1 && s.len % kFp8Block == kFp8Block - 1) {
        constexpr int kPieces = kFp8Block * D / 8 / (kWarps * 32);   // 16-byte pieces of the tail per thread
        const size_t from = bh * kFp8Block * D, to = (bh * max_len + view.full) * D;
#pragma unroll
        for (int side = 0; side < 2; ++side) {
          const uint4* tail = reinterpret_cast<const uint4*>((side ? p.v_tail : p.k_tail) + from);
          uint4 raw[kPieces];
#pragma unroll
          for (int i = 0; i < kPieces; ++i) raw[i] = tail[i * kWarps * 32 + d];
          bool plain;
          float most = most_of_bf16(raw, plain);
#pragma unroll
          for (int o = 16; o > 0; o >>= 1) most = fmaxf(most, __shfl_xor_sync(0xffffffffu, most, o));
          consumers_sync();   // (sh.m is read: the output's sums, or the other side's block)
          if (lane == 0) sh.m[warp] = most;
          consumers_sync();
#pragma unroll
          for (int w = 0; w < kWarps; ++w) most = fmaxf(most, sh.m[w]);
          const int e = fp8_exponent(most);
          uint2* codes = reinterpret_cast<uint2*>(static_cast<uint8_t*>(side ? p.v : p.k) + to);
#pragma unroll
          for (int i = 0; i < kPieces; ++i) codes[i * kWarps * 32 + d] = fp8_of_bf16(raw[i], power_of_two(-e), plain);
          if (d == 0) (side ? p.v_scale : p.k_scale)[bh * p.blocks + s.len / kFp8Block] = power_of_two(e);
        }
      }
      if (!CLUSTER) {
        if (!s.good && s.h == 0 && threadIdx.x == 0) atomicExch(p.status, DADATTN_E_ARG);
        consumers_sync();   // sh.acc / sh.m are read: the next item may write them
        have = have && ok;
      }
    }
  }

  if (CLUSTER) {
    // Threads without a share to hand over join the first barrier here; after the second the shares are merged.
    const int d = threadIdx.x;
    if (!WEIGHTS || warp == kWarps) {
      if (d >= D) cluster_wait();
      cluster_arrive();
      cluster_wait();
    }
    if (merges >= 0) {
      if (merged.good) {
        if (d < D) {
          float mm = -FLT_MAX;
          for (int j = from; j < from + merged_shares; ++j) mm = fmaxf(mm, sh.record[j][D]);
          float ll = 0.f, aa = 0.f;
          for (int j = from; j < from + merged_shares; ++j) {
            const float c = ex2(sh.record[j][D] - mm);   // a share without rows has m = -FLT_MAX: 0
            ll += sh.record[j][D + 1] * c;
            aa += sh.record[j][d] * c;
          }
          p.out[(static_cast<size_t>(merged.b) * H + merged.h) * D + d] = Elem<bf16>::from_float(aa / ll);
        }
      } else if (merged.h == 0 && d == 0) {
        atomicExch(p.status, DADATTN_E_ARG);
      }
    }
  }

  if (!snapshot) {   // the lengths were read all along: tickets only now
    __shared__ int sh_advance;
    __syncthreads();
    if (threadIdx.x == 0) sh_advance = tickets.is_last(tickets.draw());
    __syncthreads();
    if (sh_advance)
      for (int i = threadIdx.x; i < B; i += kThreads) {
        const int len = p.lengths[i];
        if (len >= 0 && len < max_len) p.lengths[i] = len + 1;
      }
  }
  if (threadIdx.x == 0 && sh.abort_flag) report_timeout(p.status, sh.abort_flag);
}

constexpr size_t decode_smem(int stages) { return static_cast<size_t>(stages) * 2 * kTileBytes + sizeof(Shared); }
static_assert((decode_smem(kFewStages) + 1024) * kFewPerSm <= 228 * 1024 && kFewStages <= kMaxStages &&
              (decode_smem(kManyStages) + 1024) * kManyPerSm <= 228 * 1024 && kManyStages <= kMaxStages,
              "shared memory of an SM exceeded");

template <bool FP8, int D, bool WEIGHTS>
int launch(Params p, cudaStream_t st) {
  int dev = 0, sms = 0;
  DAD_CUDA(cudaGetDevice(&dev));
  DAD_CUDA(cudaDeviceGetAttribute(&sms, cudaDevAttrMultiProcessorCount, dev));
  const long long pairs = static_cast<long long>(p.B) * p.H;
  // CTAs per (sequence, head): one for each tile (16 KB of K and V) of the rows that a token can see at most, while all of the
  // call's CTAs still fit on the GPU at once; but no cluster for 64 KB, or 32 KB of 8-bit rows, and less, where meeting costs
  // more than it saves. us, 12 heads of 64 (a CTA for each 64 KB / for each 16 KB): one sequence of 650 rows of 1024 5.05 /
  // 4.70, 8 bits 6.10 / 4.70; 400 of 512 5.56 / 4.20, 8 bits 5.36 / 4.86; two sequences 5.77 / 4.88, 8 bits 6.71 / 5.12; 8 the
  // same. 200 of 256 3.99 with one CTA, 4.20 with four, 8 bits 4.87 with one, 5.55 with two.
  const long long rows = p.window > 0 ? std::min<long long>(p.max_len, static_cast<long long>(p.window) + p.sinks) : p.max_len;
  const long long bytes = rows * 2 * D * (FP8 ? 1 : 2);
  const int resident = kManyPerSm * sms;
  p.ranks = 1;
  if (bytes > (FP8 ? 32768 : 65536))
    while (p.ranks < kMaxCluster && p.ranks * 2LL * kTileBytes < bytes && pairs * p.ranks * 2 <= resident) p.ranks *= 2;
  long long grid = p.ranks > 1 ? pairs * p.ranks : std::min(pairs, static_cast<long long>(resident));
  // Clusters of four or eight for two sequences in place of two or four CTAs for each, where lengths may differ and some room
  // is left on the GPU; decode.cu has both sides of the limits. Here: 4 sequences x 24 heads x 128 in 8 bits, of 1000, 3000,
  // 5000 and 7000 rows: 33.0 us with four CTAs for each, 25.2 so, and 25.2 both ways where each has 4000 rows. Under a window
  // the sequences that are longer than it are alike. (The rule does not see a window that most are shorter than: the same
  // sequences with one as long as the cache take 34.1 us, 26.3 without.)
  const long long paired = static_cast<long long>((p.B + 1) / 2) * p.H * p.ranks * 2;
  p.paired = p.window == 0 && p.ranks > 1 && p.ranks < kMaxCluster && p.B >= 2 && p.B <= kMaxPaired &&
             paired * 100 <= resident * (p.ranks * 2 == kMaxCluster ? 84LL : 92LL);
  if (p.paired) p.ranks *= 2, grid = paired;
  p.stages = grid <= kFewPerSm * sms ? kFewStages : kManyStages;
  // Longest first pays once a CTA takes more than one item (not under a window, behind which sequences are alike; 64 x 12 heads
  // of 9 .. 1017 rows in 8 bits with a window that hides nothing 20.8 us, 18.9 ranked); the in-kernel ranking, 0.9 us, handles
  // 32..256 sequences.
  p.reorder = p.B >= 32 && p.B <= kMaxRanked && pairs > grid && p.window == 0;
  auto kern = p.ranks > 1 ? decode_window_kernel<FP8, D, true, WEIGHTS> : decode_window_kernel<FP8, D, false, WEIGHTS>;
  DAD_CUDA(cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, static_cast<int>(decode_smem(kMaxStages))));
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3(static_cast<unsigned>(grid));
  cfg.blockDim = dim3(kThreads);
  cfg.dynamicSmemBytes = decode_smem(p.stages);
  cfg.stream = st;
  cudaLaunchAttribute attrs[2];
  attrs[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attrs[0].val.programmaticStreamSerializationAllowed = 1;
  attrs[1].id = cudaLaunchAttributeClusterDimension;
  attrs[1].val.clusterDim = {static_cast<unsigned>(p.ranks), 1, 1};
  cfg.attrs = attrs;
  cfg.numAttrs = p.ranks > 1 ? 2 : 1;
  DAD_CUDA(cudaLaunchKernelEx(&cfg, kern, p));
  return DADATTN_OK;
}

// Sizes and the arguments that both entry points have.
int check(const char* name, std::initializer_list<const void*> wide, const void* lengths, int B, int H, int D, int max_len,
          float scale, int window, int sinks, const void* workspace, size_t given, bool weights) {
  for (const void* x : wide)
    if (!x) return fail(DADATTN_E_ARG, "%s: null pointer", name);
  if (!lengths) return fail(DADATTN_E_ARG, "%s: null pointer", name);
  if (B <= 0 || H <= 0 || max_len <= 0 || H > 65535 || static_cast<long long>(B) * H > 0x7fffffffLL / kMaxCluster)
    return fail(DADATTN_E_ARG, "%s: bad sizes B=%d H=%d max_len=%d", name, B, H, max_len);
  if (max_len > DADATTN_MAX_CACHE_LEN)
    return fail(DADATTN_E_UNSUPPORTED, "%s: max_len %d exceeds %d", name, max_len, DADATTN_MAX_CACHE_LEN);
  if (D != 64 && D != 128) return fail(DADATTN_E_UNSUPPORTED, "%s: unsupported D %d", name, D);
  if (window < 0 || sinks < 0) return fail(DADATTN_E_ARG, "%s: window %d and sinks %d must not be negative", name, window, sinks);
  if (!(scale > -INFINITY && scale < INFINITY)) return fail(DADATTN_E_ARG, "%s: scale must be finite", name);
  for (const void* x : wide)
    if (!aligned(x, 16)) return fail(DADATTN_E_ARG, "%s: pointers must be 16-byte aligned", name);
  if (!aligned(lengths, 4)) return fail(DADATTN_E_ARG, "%s: lengths must be 4-byte aligned", name);
  if (!workspace || !aligned(workspace, 16))
    return fail(DADATTN_E_ARG, "%s: workspace must be a 16-byte aligned device pointer", name);
  const size_t need = window_workspace_bytes(B, H, max_len, weights);
  if (given < need) return fail(DADATTN_E_WORKSPACE, "%s: workspace %zu < %zu bytes", name, given, need);
  return DADATTN_OK;
}

}  // namespace
}  // namespace dadattn

using namespace dadattn;

extern "C" size_t dadattn_decode_window_workspace_bytes(int B, int H, int D, int max_len, int with_weights) {
  if (B <= 0 || H <= 0 || D <= 0 || max_len <= 0) return 0;
  return window_workspace_bytes(B, H, max_len, with_weights != 0);
}

extern "C" int dadattn_decode_bf16_window(uint16_t* out, const uint16_t* q, const uint16_t* k_new, const uint16_t* v_new,
                                          uint16_t* k_cache, uint16_t* v_cache, int32_t* lengths, float* weights, int B,
                                          int H, int D, int max_len, float scale, int window, int sinks, void* workspace,
                                          size_t workspace_bytes, dadattn_stream_t stream) {
  if (int rc = check("windowed decode", {out, q, k_new, v_new, k_cache, v_cache}, lengths, B, H, D, max_len, scale, window,
                     sinks, workspace, workspace_bytes, weights != nullptr))
    return rc;
  if (weights && !aligned(weights, 4)) return fail(DADATTN_E_ARG, "windowed decode: weights must be 4-byte aligned");
  Params p = {};
  p.status = device_status_word();
  if (!p.status) return DADATTN_E_CUDA;
  p.out = reinterpret_cast<bf16*>(out);
  p.q = reinterpret_cast<const bf16*>(q);
  p.k_new = reinterpret_cast<const bf16*>(k_new);
  p.v_new = reinterpret_cast<const bf16*>(v_new);
  p.k = k_cache;
  p.v = v_cache;
  p.lengths = lengths;
  p.weights = weights;
  p.counters = static_cast<unsigned*>(workspace);
  p.scores = reinterpret_cast<float*>(static_cast<uint8_t*>(workspace) + counter_bytes(B, H));
  p.B = B, p.H = H, p.max_len = max_len, p.window = window, p.sinks = sinks, p.scale = scale;
  cudaStream_t st = static_cast<cudaStream_t>(stream);
  if (weights) return D == 64 ? launch<false, 64, true>(p, st) : launch<false, 128, true>(p, st);
  return D == 64 ? launch<false, 64, false>(p, st) : launch<false, 128, false>(p, st);
}

extern "C" int dadattn_decode_fp8(uint16_t* out, const uint16_t* q, const uint16_t* k_new, const uint16_t* v_new,
                                  uint8_t* k_cache, uint8_t* v_cache, float* k_scale, float* v_scale, uint16_t* k_tail,
                                  uint16_t* v_tail, int32_t* lengths, int B, int H, int D, int max_len, float scale,
                                  int window, int sinks, void* workspace, size_t workspace_bytes, dadattn_stream_t stream) {
  if (int rc = check("8-bit decode", {out, q, k_new, v_new, k_cache, v_cache, k_tail, v_tail}, lengths, B, H, D, max_len,
                     scale, window, sinks, workspace, workspace_bytes, false))
    return rc;
  if (!k_scale || !v_scale || !aligned(k_scale, 4) || !aligned(v_scale, 4))
    return fail(DADATTN_E_ARG, "8-bit decode: k_scale and v_scale must be 4-byte aligned device pointers");
  Params p = {};
  p.status = device_status_word();
  if (!p.status) return DADATTN_E_CUDA;
  p.out = reinterpret_cast<bf16*>(out);
  p.q = reinterpret_cast<const bf16*>(q);
  p.k_new = reinterpret_cast<const bf16*>(k_new);
  p.v_new = reinterpret_cast<const bf16*>(v_new);
  p.k = k_cache;
  p.v = v_cache;
  p.k_scale = k_scale;
  p.v_scale = v_scale;
  p.k_tail = reinterpret_cast<bf16*>(k_tail);
  p.v_tail = reinterpret_cast<bf16*>(v_tail);
  p.lengths = lengths;
  p.counters = static_cast<unsigned*>(workspace);
  p.B = B, p.H = H, p.max_len = max_len, p.window = window, p.sinks = sinks, p.scale = scale;
  p.blocks = fp8_scale_blocks(max_len);
  cudaStream_t st = static_cast<cudaStream_t>(stream);
  return D == 64 ? launch<true, 64, false>(p, st) : launch<true, 128, false>(p, st);
}
