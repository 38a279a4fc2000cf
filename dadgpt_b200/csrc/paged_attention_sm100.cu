// Causal attention of a packed, ragged batch's new tokens over the pages of their sequences, for sm_100a (tcgen05, TMEM, TMA).
//
//   out_i = sum_j p_ij v_j,  p_ij = exp(scale q_i.k_j - lse_i),  lse_i = ln sum_j exp(scale q_i.k_j)   over j <= lengths[b] + i
//
// for token i of the count[b] that sequence b brings, whose rows are in their pages already. The `group` query heads that share
// a key head are rows of one tile: a 128-row tile is 128 / group tokens of all of them, so K and V are read once for the group
// and a short piece of a prompt still fills tiles.
//
// A CTA has two softmax groups of 128 threads (a row each), two tensor-core issuers and one ring of 128-key K and V tiles. An
// item is
//   * a pair of adjacent query tiles, A and B, of a sequence and key head. Both use every K / V tile of the ring; while the
//     threads of one compute exponentials the tensor pipe runs the products of the other;
//   * or one tile, where a sequence has no second one: the groups share its keys, A takes the even steps (of 128 keys, or of 64
//     at head size 64), B the odd ones, and they join their maxima, sums and accumulators, which each finds in tensor memory, at
//     the end.
// CTAs are persistent and take items from the grid's own queue (clusterlaunchcontrol): keys of the next item are on their way
// while the current one ends. Where the tiles do not fill the GPU (CLUSTER > 1), every CTA of a cluster takes a run of one tile's
// keys, both groups as above, and the results are joined through distributed shared memory: no workspace.
// The two groups' exponentials take turns: left to themselves they fall into step, each at half the exp2 unit's rate, and the
// tensor pipe idles (a count in shared memory says how far the other is; it is waited for with a limit and nothing depends on it).
// Keys come through the page table: lane i of the producer warp fetches the i-th box of a tile (as high as a page, up to the
// tile), and looks its page up a tile ahead. Rows behind a sequence's last are not trusted: their scores are masked, and the
// softmax threads set their V to zero in shared memory before they hand over the probabilities of that tile.
//   warp 0       scheduler + K / V producer        warp 1     issuer of group A, tensor memory
//   warp 2       issuer of group B                 warp 3     Q
//   warps 4-7    softmax group A                   warps 8-11 softmax group B
// Bound by the steps of a group, which wait for each other: scores, maximum, exponentials, probabilities, product. At head size
// 128 one CTA has an SM, a step of both groups takes 3500 clk (2048 of the exp2 unit, 2048 of the tensor pipe, which is what is
// busy 60 % of the time); at head size 64 two CTAs do, and 64 keys of their four groups take 3300 to 3600 (2048 of the exp2 unit).
// Measured (us): 2048 tokens behind 14336 rows, 32 heads on 8 of 128 453 (1137 TFLOP/s; 516 at the power cap); 24 sequences with
// up to 3690 rows ahead and 1 to 512 new ones, the same heads, 112-130; 16 prompts of up to 1024 tokens, 12 heads of 64 36; 301
// tokens behind 700 rows, 12 heads of 64 12.5.
// At head size 128 an instance has all 168 registers of a thread and spills 40 (single CTAs) or 52 bytes.
// Not kept: exponentials as polynomials, in any share (slower at both head sizes: the threads, not the exp2 unit, are short of
// time); 64-key steps with two score buffers at head size 128 (514 for the first); probabilities handed over in quarters (481),
// the turn passed on earlier (482-501).
// Every wait is bounded (sm100_ptx.cuh).
#include <cuda_bf16.h>

#include <algorithm>
#include <climits>
#include <cmath>

#include "decode_common.cuh"
#include "paged.cuh"
#include "rotary.cuh"
#include "sm100_ptx.cuh"

namespace dadattn {
namespace {

using namespace ptx;
using bf16 = __nv_bfloat16;

constexpr int kT = 128;                 // tile edge: query rows of a group, keys of a K / V tile
constexpr int kPanel = 128 * 128;       // [128 rows][64 bf16]: 16 KB, 128-byte rows, swizzled
constexpr int kThreads = 12 * 32;
constexpr int kGroup = 128;             // threads of a softmax group
constexpr int kItems = 4;               // items a CTA knows of (a power of two)
constexpr int kSlots = 5;               // ring of K and V tiles, K0 V0 K1 V1 ...
constexpr int kMaxCluster = 8;
constexpr float kLog2e = 1.4426950408889634f;
constexpr float kLn2 = 0.6931471805599453f;
constexpr float kRescaleAt = 8.0f;      // log2 units: O is rescaled only when the maximum grew by 2^8

template <int D>
struct Plan {
  static constexpr int kPerSm = D == 128 ? 1 : 2;           // CTAs
  static constexpr int kN = D == 128 ? 128 : 64;            // keys of a step
  static constexpr int kSteps = kT / kN;                    // steps of a key tile
  static constexpr int kPanels = D / 64;
  static constexpr int kTileBytes = kPanels * kPanel;
  static constexpr int kQ = 0;                              // [A, B]
  static constexpr int kKV = kQ + 2 * kTileBytes;
  static constexpr int kBars = kKV + kSlots * kTileBytes;
  static constexpr int kBytes = kBars + 1024;
  static constexpr int kPitch = D + 4;                      // floats of a row of an accumulator that a cluster joins (banks)
  static constexpr int kStats = kKV + kT * kPitch * 4;      // and the rows' maxima and sums behind them, in the ring's place
  static constexpr uint32_t kTmemCols = 512 / kPerSm, kColS = 0, kColO = 2 * kN;
  // Registers per thread at launch, and once the warpgroups have rebalanced.
  static constexpr int kRegsLaunch = D == 128 ? 168 : 80, kRegsSoftmax = D == 128 ? 208 : 88, kRegsHelper = D == 128 ? 88 : 64;
  static_assert(kPerSm * (kBytes + 1024) <= 228 * 1024, "shared memory of an SM exceeded");
  static_assert(kStats + kT * 8 <= kBars, "the accumulator in the ring's place");
  static_assert(2 * (kN + D) <= kTmemCols, "tensor memory");
  static_assert(2 * kGroup * kRegsSoftmax + 128 * kRegsHelper <= kThreads * kRegsLaunch,
                "the warpgroups ask for more registers than the CTA owns");
  static_assert(kPerSm * kThreads * kRegsLaunch <= 65536 && kPerSm * kThreads * (kRegsLaunch + 8) > 65536,
                "kRegsLaunch is not what the compiler gives a CTA of this size");
};

struct Bars {
  __align__(16) uint4 stolen;             // answer to a request for another block
  uint64_t stolen_full;
  uint64_t item_ready[kItems], item_free[kItems];
  uint64_t q_full[2], q_empty[2], slot_full[kSlots], slot_empty[kSlots];
  uint64_t s_full[2], p_full[2][2], o_done[2], settled[2];   // [group]; p_full: [group][64 keys of a step]
  uint64_t joined, parted, freed;         // groups that share a tile: results are there; numbers, accumulators have been read
  uint32_t tmem_base;
  int abort_flag;
  int any_bad;                            // a page outside the pool, in any item
  int exps[2][4];                         // tiles whose exponentials a warp of a group is through with
  // sequence (-1: the end), first token, rows ahead, first packed row, tokens, key head, and whether a page is outside the pool:
  // of the key tiles that both groups see, of those that only a pair's second one sees
  int item[kItems][8];
};
static_assert(sizeof(Bars) <= 1024, "barrier block");

struct ChunkParams {
  int wide;     // rows of out begin at multiples of 32 bytes
  int sorted;   // items do not all start at once
  bf16* out;
  float* lse;
  int64_t out_token, out_head;
  PagedCache cache;
  int T, max_new, heads_q, group, tile_tokens;   // tokens of a tile: 128 / group
  int item_tokens, token_shift;                  // of an item, two tiles or one; their log2, -1: not a power of two
  int chunk;                                     // rows of a K / V box
  float scale;
  int* status;
};

__device__ __forceinline__ float4 ld_cluster4(uint32_t addr) {
  float4 v;
  asm volatile("ld.shared::cluster.v4.f32 {%0, %1, %2, %3}, [%4];"
               : "=f"(v.x), "=f"(v.y), "=f"(v.z), "=f"(v.w)
               : "r"(addr)
               : "memory");
  return v;
}
__device__ __forceinline__ float2 ld_cluster2(uint32_t addr) {
  float2 v;
  asm volatile("ld.shared::cluster.v2.f32 {%0, %1}, [%2];" : "=f"(v.x), "=f"(v.y) : "r"(addr) : "memory");
  return v;
}
// Two columns of a lane's
__device__ __forceinline__ void tmem_st2(uint32_t taddr, uint32_t a, uint32_t b) {
  asm volatile("tcgen05.st.sync.aligned.32x32b.x2.b32 [%0], {%1, %2};" ::"r"(taddr), "r"(a), "r"(b) : "memory");
}
__device__ __forceinline__ void tmem_ld2(uint32_t taddr, float& a, float& b) {
  asm volatile("tcgen05.ld.sync.aligned.32x32b.x2.b32 {%0, %1}, [%2];" : "=f"(a), "=f"(b) : "r"(taddr) : "memory");
}
__device__ __forceinline__ int ld_cluster_int(uint32_t addr) {
  int v;
  asm volatile("ld.shared::cluster.s32 %0, [%1];" : "=r"(v) : "r"(addr) : "memory");
  return v;
}

// 16 floats to bf16, 32 bytes of a row: a thread has a row to itself, and a store costs the lines it touches.
__device__ __forceinline__ void store_16(bf16* to, const float (&y)[16], bool wide) {
  uint32_t w[8];
#pragma unroll
  for (int i = 0; i < 8; ++i) w[i] = pack_bf16(y[2 * i], y[2 * i + 1]);
  if (wide) {
    asm volatile("st.global.v8.b32 [%0], {%1, %2, %3, %4, %5, %6, %7, %8};" ::"l"(to), "r"(w[0]), "r"(w[1]), "r"(w[2]), "r"(w[3]),
                 "r"(w[4]), "r"(w[5]), "r"(w[6]), "r"(w[7])
                 : "memory");
  } else {
    reinterpret_cast<uint4*>(to)[0] = make_uint4(w[0], w[1], w[2], w[3]);
    reinterpret_cast<uint4*>(to)[1] = make_uint4(w[4], w[5], w[6], w[7]);
  }
}

// A tile of a group, or what is left of one: its rows, and how many key tiles they see.
struct Tile {
  int token0, rows, n;
  bool half;   // of the last key tile only the first half is seen
};
struct Item {
  int b, token0, ahead, first, count, kv_head;
  __device__ __forceinline__ bool single(const ChunkParams& p) const {
    return p.item_tokens == p.tile_tokens || token0 + p.tile_tokens >= count;
  }
  __device__ __forceinline__ Tile tile(const ChunkParams& p, int at) const {   // at: 0, or 1 for the second of a pair
    Tile t;
    t.token0 = token0 + at * p.tile_tokens;
    const int tokens = min(count - t.token0, p.tile_tokens);
    t.rows = tokens * p.group;
    const int keys = ahead + t.token0 + tokens;
    t.n = (keys + kT - 1) / kT;
    t.half = keys % kT != 0 && keys % kT <= kT / 2;
    return t;
  }
};
// What a CTA does of an item: key tiles lo .. lo + n_kv - 1, of STEPS steps each. Of a pair group A sees the first n_first. Of a
// single tile the groups take the steps in turn, or, with CTAs of a cluster, the tiles: those have no second CTA on their SM, and
// groups that begin with the same keys hinder each other (301 tokens, 12 heads of 64 13.3 us instead of 12.6).
template <int STEPS, int CLUSTER>
struct Share {
  static constexpr int kTurn = CLUSTER > 1 ? STEPS : 1;   // steps of a turn
  bool single;
  int lo, n_kv, n_first;
  int half;   // of the last of these tiles (of group x: bit x) only the first half is seen
  // steps of group x: all but a last half that nothing is seen of
  __device__ __forceinline__ int steps(int x) const {
    const int tiles = single || x ? n_kv : n_first;
    const int all = STEPS * tiles - (STEPS == 2 && tiles > 0 && (half >> x & 1) ? 1 : 0);
    return single ? all / (2 * kTurn) * kTurn + min(max(all % (2 * kTurn) - x * kTurn, 0), kTurn) : all;
  }
  // the k-th of them, among the steps of the CTA's tiles
  __device__ __forceinline__ int at(int x, int k) const { return single ? k / kTurn * 2 * kTurn + x * kTurn + k % kTurn : k; }
  // whether it is the group's first of a tile; its last, but for the very last
  __device__ __forceinline__ bool first_of(int k) const { return (single && kTurn < STEPS) || k % STEPS == 0; }
  __device__ __forceinline__ bool last_of(int k) const { return (single && kTurn < STEPS) || k % STEPS == STEPS - 1; }
};
template <int STEPS, int CLUSTER>
__device__ __forceinline__ Share<STEPS, CLUSTER> share_of(const Item& it, const ChunkParams& p, int rank) {
  Share<STEPS, CLUSTER> s;
  s.single = CLUSTER > 1 || it.single(p);
  const Tile last = it.tile(p, s.single ? 0 : 1);
  const int n = last.n;
  s.lo = CLUSTER > 1 ? static_cast<int>(static_cast<int64_t>(n) * rank / CLUSTER) : 0;
  s.n_kv = (CLUSTER > 1 ? static_cast<int>(static_cast<int64_t>(n) * (rank + 1) / CLUSTER) : n) - s.lo;
  s.n_first = 0;
  s.half = last.half && s.lo + s.n_kv == n ? 3 : 0;
  if (!s.single) {
    const Tile first = it.tile(p, 0);
    s.n_first = first.n;
    s.half = (s.half & 2) | (first.half ? 1 : 0);
  }
  return s;
}

// Block `block` is key head block % heads of the item of place block / heads in the order; by one warp. b < 0: there
// is none. Sequences that are refused have no items. The order: of 32 sequences at a time the items with the most keys, so
// that what starts last is short (one sequence after the other, each key head by itself: 16 prompts of up to 1024 tokens 46 us
// instead of 36). An item's weight is twice its keys; one tile counts half, since both groups work on it. How many items of a
// sequence reach a weight is an expression, so that the 64th of the range of weights in which the x-th falls is found by
// halving, and the item in it by counting. (To the last bit of the weight the search took 1.6 us, 4-8 % of whole calls.) Where
// all items start at once (`sorted` false) the order does not matter.
// The 32 sequences stay with the warp (Found) for the next block, which is behind this one as a rule: of 1024 sequences the
// search from the first on took a third of the time, of 2048 two thirds.
struct Found {
  int base = -32, ahead = 0, first = 0, count = 0;   // this lane's of sequences base .. base + 31
  int64_t before = 0;                                // items of the sequences ahead of those
};
__device__ __forceinline__ Item find_item(const ChunkParams& p, unsigned block, bool sorted, Found& f) {
  const PagedCache& c = p.cache;
  const int lane = threadIdx.x % 32, tokens = p.item_tokens;
  const int place = block / c.heads;
  Item it = {-1, 0, 0, 0, 0, static_cast<int>(block - static_cast<unsigned>(place) * c.heads)};
  if (place < f.before) f = Found();
  int64_t x = place - f.before;
  for (;;) {
    const int ahead = f.ahead, first = f.first, count = f.count;
    const int mine = (count + tokens - 1) / tokens;   // items: the i-th of them from token i * tokens on
    const int all = __reduce_add_sync(0xffffffffu, mine);
    if (x >= all) {
      x -= all;
      f.before += all;
      f.ahead = f.first = f.count = 0;
      if (f.base >= c.B) return it;
      f.base += 32;
      if (f.base + lane < c.B &&
          (!sequence_rows(c, f.base + lane, p.T, f.ahead, f.first, f.count) || f.count > p.max_new)) {
        atomicExch(p.status, DADATTN_E_ARG);
        f.count = 0;
      }
      continue;
    }
    int at, index;
    if (!sorted) {
      int upto = mine;
#pragma unroll
      for (int o = 1; o < 32; o <<= 1) {
        const int other = __shfl_up_sync(0xffffffffu, upto, o);
        if (lane >= o) upto += other;
      }
      at = __ffs(__ballot_sync(0xffffffffu, upto > x)) - 1;
      index = __shfl_sync(0xffffffffu, upto, at) - 1 - static_cast<int>(x);
    } else {
      // (keys are 2^30 at most, DADATTN_MAX_CACHE_LEN: weights are unsigned)
      const bool one = count - (mine - 1) * tokens <= p.tile_tokens && tokens > p.tile_tokens;   // the last item is one tile
      const unsigned keys = ahead + count, most = __reduce_max_sync(0xffffffffu, mine ? 2 * keys : 0u);
      const int unit = max(1, 26 - __clz(most));   // most < 64 << unit
      const int whole = max(mine - 1, 0), last = mine > 0 ? static_cast<int>((one ? keys : 2 * keys) >> unit) : -1;
      // the first of the sequence's whole items that reaches so many units, behind which all do; the last one is its own
      auto from = [&](int units) -> int {
        const int need = static_cast<int>(static_cast<unsigned>(units) << (unit - 1)) - ahead + tokens - 1;   // keys, to be divided
        return min(max((p.token_shift >= 0 ? need >> p.token_shift : need / tokens) - 1, 0), whole);
      };
      auto reach = [&](int units) -> int { return whole - from(units) + (last >= units); };
      int low = 0;   // the most units that more than x items reach
#pragma unroll
      for (int step = 32; step; step >>= 1)
        if (__reduce_add_sync(0xffffffffu, reach(low + step)) > static_cast<int>(x)) low += step;
      const int here = from(low + 1), with = here - from(low) + (last == low);   // the sequence's items of so many units
      const int rest = static_cast<int>(x) - __reduce_add_sync(0xffffffffu, whole - here + (last > low));
      int upto = with;
#pragma unroll
      for (int o = 1; o < 32; o <<= 1) {
        const int other = __shfl_up_sync(0xffffffffu, upto, o);
        if (lane >= o) upto += other;
      }
      at = __ffs(__ballot_sync(0xffffffffu, upto > rest)) - 1;
      const int nth = rest - (upto - with);   // of them: the last one, then the others from behind
      index = __shfl_sync(0xffffffffu, last == low && nth == 0 ? mine - 1 : here - 1 - nth + (last == low), at);
    }
    it.b = f.base + at;
    it.token0 = index * tokens;
    it.ahead = __shfl_sync(0xffffffffu, ahead, at);
    it.first = __shfl_sync(0xffffffffu, first, at);
    it.count = __shfl_sync(0xffffffffu, count, at);
    return it;
  }
}

// ---- the grid's queue -------------------------------------------------------------------------------
// Asks for a block of this grid that has not started yet, in its place; the answer (16 bytes) completes on `bar`.
// Not asked again once the answer was that there is none.
__device__ __forceinline__ void request_block(uint4* answer, uint64_t* bar) {
  asm volatile("clusterlaunchcontrol.try_cancel.async.shared::cta.mbarrier::complete_tx::bytes.b128 [%0], [%1];"
               ::"r"(smem_u32(answer)), "r"(smem_u32(bar))
               : "memory");
}
__device__ __forceinline__ bool read_answer(const uint4* answer, unsigned& block) {
  uint32_t ok;
  asm volatile(
      "{\n\t.reg .b128 h;\n\t.reg .pred p;\n\t"
      "ld.shared.b128 h, [%2];\n\t"
      "clusterlaunchcontrol.query_cancel.is_canceled.pred.b128 p, h;\n\t"
      "selp.u32 %0, 1, 0, p;\n\t"
      "mov.u32 %1, 0;\n\t"
      "@p clusterlaunchcontrol.query_cancel.get_first_ctaid.v4.b32.b128 {%1, _, _, _}, h;\n\t}"
      : "=&r"(ok), "=&r"(block)
      : "r"(smem_u32(answer))
      : "memory");
  return ok != 0;
}

// Every role reads the CTA's items, in order, from the ring that the scheduler fills, and gives each back.
struct Feed {
  Bars* bars;
  volatile int* abort_flag;
  int n;
  __device__ __forceinline__ const volatile int* entry() const { return bars->item[n & (kItems - 1)]; }
  __device__ __forceinline__ bool next(Item& it) {
    if (!mbar_wait(&bars->item_ready[n & (kItems - 1)], (n / kItems) & 1, abort_flag)) return false;
    const volatile int* e = entry();
    it = Item{e[0], e[1], e[2], e[3], e[4], e[5]};
    return it.b >= 0;
  }
  __device__ __forceinline__ void give_back(bool arrives = true) {
    if (arrives) mbar_arrive(&bars->item_free[n & (kItems - 1)]);
    ++n;
  }
};

// Which slot of the ring a tile's K (m = 0) or V is in, and the parity of that use. tile: of all that the CTA has gone through.
template <int D>
struct Slot {
  int at;
  uint32_t parity;
  __device__ __forceinline__ Slot(int tile, int m) {
    const uint32_t i = 2u * tile + m;
    at = i % kSlots;
    parity = (i / kSlots) & 1;
  }
};

template <int D, int CLUSTER>
__global__ void __launch_bounds__(kThreads, Plan<D>::kPerSm)
paged_attention_kernel(const __grid_constant__ CUtensorMap map_q, const __grid_constant__ CUtensorMap map_k,
                       const __grid_constant__ CUtensorMap map_v, const ChunkParams p) {
  using L = Plan<D>;
  // Tensor memory: the scores of group X at kN X (its probabilities in the first half of these columns), O at kColO + D X.
  constexpr int kN = L::kN, kSteps = L::kSteps;
  constexpr uint32_t kTmemCols = L::kTmemCols, kColS = L::kColS, kColO = L::kColO;
  extern __shared__ __align__(1024) uint8_t smem[];
  Bars* bars = reinterpret_cast<Bars*>(smem + L::kBars);
  volatile int* abort_flag = &bars->abort_flag;
  const int warp = threadIdx.x / 32, lane = threadIdx.x % 32;
  const int rank = CLUSTER > 1 ? blockIdx.x % CLUSTER : 0;
  const PagedCache& c = p.cache;

  if ((smem_u32(smem) & 1023u) != 0) {  // the swizzled layouts need a 1024-byte aligned base
    if (threadIdx.x == 0) atomicExch(p.status, DADATTN_E_CUDA);
    return;
  }
  if (threadIdx.x == 0) {
    mbar_init(&bars->stolen_full, 1);
    for (int i = 0; i < kItems; ++i) {
      mbar_init(&bars->item_ready[i], 1);
      mbar_init(&bars->item_free[i], 8 + 3);            // softmax warps, issuers, Q
    }
    for (int i = 0; i < kSlots; ++i) {
      mbar_init(&bars->slot_full[i], 1);
      mbar_init(&bars->slot_empty[i], 2);               // one arrival per issuer
    }
    for (int x = 0; x < 2; ++x) {
      mbar_init(&bars->q_full[x], 1);
      mbar_init(&bars->q_empty[x], 1);
      mbar_init(&bars->s_full[x], 1);
      mbar_init(&bars->p_full[x][0], 4);                // one arrival per warp
      mbar_init(&bars->p_full[x][1], 4);
      mbar_init(&bars->o_done[x], 1);
      mbar_init(&bars->settled[x], 1);
      for (int w = 0; w < 4; ++w) bars->exps[x][w] = 0;
    }
    mbar_init(&bars->joined, 8);
    // (softmax warps and the issuers: one whose group has no keys of a tile would not be missed otherwise, and could find the
    // barrier two items on)
    mbar_init(&bars->parted, 8 + 2);
    mbar_init(&bars->freed, 8);
    bars->abort_flag = 0;
    bars->any_bad = 0;
    fence_mbar_init();
  }
  if (warp == 1) {
    tmem_alloc(&bars->tmem_base, kTmemCols);
    tmem_relinquish();
  }
  tc_fence_before_sync();
  __syncthreads();
  tc_fence_after_sync();
  const uint32_t tmem = bars->tmem_base;
  pdl_wait();
  pdl_launch_dependents();

  Feed feed{bars, abort_flag, 0};
  Item it;
  if (warp < 4) {
    setmaxnreg_dec<L::kRegsHelper>();
    if (warp == 0) {
      // ------------------------------ scheduler + K / V producer ------------------------------
      const bool sorted = CLUSTER == 1 && p.sorted;
      const int per_tile = kT / p.chunk;   // boxes
      const int box = lane % per_tile, panel = lane / per_tile;
      int n_pub = 0, n_asked = 0, n_loaded = 0, slot = 0;
      Found found;
      uint32_t parity = 0;
      bool ok = true;
      auto ask = [&]() {
        if (lane == 0) {
          fence_proxy_async_smem();   // (the last answer has been read)
          mbar_arrive_expect_tx(&bars->stolen_full, 16);
          request_block(&bars->stolen, &bars->stolen_full);
        }
        __syncwarp();
        ++n_asked;
      };
      // the next block's item; b < 0 and `more` false: nothing left
      auto answer = [&](Item& it, bool& more) {
        unsigned block;
        ok = warp_wait(&bars->stolen_full, (n_asked - 1) & 1, abort_flag);
        more = ok && read_answer(&bars->stolen, block);
        __syncwarp();
        if (more) it = find_item(p, block, sorted, found);
        else it.b = -1;
      };
      it = find_item(p, blockIdx.x / CLUSTER, sorted, found);
      bool more = CLUSTER == 1;
      while (ok) {
        while (ok && it.b < 0 && more) {
          ask();
          answer(it, more);
        }
        if (!ok) break;
        const int e = n_pub & (kItems - 1);
        if (n_pub >= kItems && !(ok = warp_wait(&bars->item_free[e], (n_pub / kItems - 1) & 1, abort_flag))) break;
        if (lane == 0) {
          volatile int* to = bars->item[e];
          to[0] = it.b, to[1] = it.token0, to[2] = it.ahead, to[3] = it.first, to[4] = it.count, to[5] = it.kv_head, to[6] = to[7] = 0;
          mbar_arrive(&bars->item_ready[e]);
        }
        __syncwarp();
        ++n_pub;
        if (it.b < 0) break;
        const auto s = share_of<kSteps, CLUSTER>(it, p, rank);
        const int total = it.ahead + it.count;   // rows of the sequence
        const int32_t* table = c.table + static_cast<int64_t>(it.b) * c.max_pages;
        // Whether a row of this lane's box of a tile is there, and its page (looked at only when the box is fetched).
        auto there = [&](int tile) { return panel < L::kPanels && tile * kT + box * p.chunk < total; };
        auto look_up = [&](int tile) -> int { return there(tile) ? table[(tile * kT + box * p.chunk) >> c.page_shift] : 0; };
        int page = s.n_kv > 0 ? look_up(s.lo) : 0;
        for (int j = 0; ok && j < s.n_kv; ++j) {
          const int tile = s.lo + j, mine = page;
          // The next block is asked for only now: what a CTA holds in advance no idle CTA can take.
          if (j + 1 < s.n_kv) page = look_up(tile + 1);
          else if (CLUSTER == 1) ask();
          const int boxes = min((total - tile * kT + p.chunk - 1) / p.chunk, per_tile);
          const int row = tile * kT + box * p.chunk;
          // (a row coordinate outside the pool reads zeros)
          const bool good = mine >= 0 && mine < c.pages, mine_there = there(tile);
          if (!good) bars->item[e][s.single || j < s.n_first ? 6 : 7] = bars->any_bad = 1;
          const int y = good ? ((mine * c.heads + it.kv_head) << c.page_shift) + (row & ((1 << c.page_shift) - 1)) : -kMaxPage;
#pragma unroll
          for (int m = 0; m < 2; ++m) {
            if (n_loaded >= kSlots && !(ok = warp_wait(&bars->slot_empty[slot], parity ^ 1u, abort_flag))) break;
            if (lane == 0) mbar_arrive_expect_tx(&bars->slot_full[slot], boxes * L::kPanels * p.chunk * 128);
            __syncwarp();
            if (mine_there)
              tma_load_3d(smem + L::kKV + slot * L::kTileBytes + panel * kPanel + box * p.chunk * 128, m ? &map_v : &map_k,
                          &bars->slot_full[slot], panel * 64, y, 0);
            __syncwarp();
            ++n_loaded;
            if (++slot == kSlots) slot = 0, parity ^= 1u;
          }
        }
        if (CLUSTER == 1 && ok) answer(it, more);
        else it.b = -1;
      }
      if (lane == 0) {
        if (n_asked > 0) settle(&bars->stolen_full, (n_asked - 1) & 1);
        settle_ring(bars->slot_full, kSlots, n_loaded);
      }
    } else if (warp == 3) {
      // ------------------------------ Q ------------------------------
      if (lane == 0) {
        prefetch_tensormap(&map_q);
        int n[2] = {0, 0};
        bool ok = true;
        while (ok && feed.next(it)) {
          const auto s = share_of<kSteps, CLUSTER>(it, p, rank);
#pragma unroll
          for (int x = 0; x < 2; ++x) {
            if (s.steps(x) == 0) continue;
            if (n[x] > 0 && !(ok = mbar_wait(&bars->q_empty[x], (n[x] - 1) & 1, abort_flag))) break;
            mbar_arrive_expect_tx(&bars->q_full[x], L::kPanels * p.tile_tokens * p.group * 128);
            for (int h = 0; h < L::kPanels; ++h)
              tma_load_3d(smem + L::kQ + x * L::kTileBytes + h * kPanel, &map_q, &bars->q_full[x], h * 64, it.kv_head * p.group,
                          it.first + it.tile(p, s.single ? 0 : x).token0);
            ++n[x];
          }
          feed.give_back();
        }
#pragma unroll
        for (int x = 0; x < 2; ++x)
          if (n[x] > 0) settle(&bars->q_full[x], (n[x] - 1) & 1);
      }
    } else {
      // ------------------------------ MMA issuers ------------------------------
      const int x = warp - 1;
      if (elect_one()) {
        constexpr uint32_t idesc_s = make_idesc_bf16(kT, kN, 0, 0);   // Q, K: K-major
        constexpr uint32_t idesc_o = make_idesc_bf16(kT, D, 0, 1);    // P K-major, V MN-major
        const SmemDescBase q_desc = make_desc_base_sw128(smem_u32(smem + L::kQ) + x * L::kTileBytes, 0);
        // (read MN-major, a V tile's two 64-column panels are kPanel apart; K-major operands ignore that offset)
        const SmemDescBase kv_desc0 = make_desc_base_sw128(smem_u32(smem + L::kKV), kPanel);
        const uint32_t tS = tmem + kColS + x * kN, tO = tmem + kColO + x * D;
        uint32_t g = 0, u = 0, joins = 0;   // steps, items and shared tiles of this group so far
        int gone = 0;                       // key tiles of the CTA so far
        bool ok = true;
        auto wait_slot = [&](const Slot<D>& s) -> bool { return mbar_wait(&bars->slot_full[s.at], s.parity, abort_flag); };
        // a tile that this group has nothing to do with: given back once it is there, as the others are
        auto skip = [&](int tile) -> bool {
#pragma unroll
          for (int m = 0; m < 2; ++m) {
            const Slot<D> s(tile, m);
            if (!wait_slot(s)) return false;
            mbar_arrive(&bars->slot_empty[s.at]);
          }
          return true;
        };
        while (ok && feed.next(it)) {
          const auto s = share_of<kSteps, CLUSTER>(it, p, rank);
          const int steps = s.steps(x);
          auto tile_of = [&](int k) -> int { return s.at(x, k) / kSteps; };
          // Scores of the k-th step
          auto issue_s = [&](int k) -> bool {
            const int at = tile_of(k), h = s.at(x, k) % kSteps;
            const Slot<D> slot(gone + at, 0);
            if (s.first_of(k) && !wait_slot(slot)) return false;
            tc_fence_after_sync();
            const SmemDescBase k_desc{kv_desc0.lo + slot.at * (L::kTileBytes >> 4) + h * (kN * 128 >> 4), kv_desc0.hi};
#pragma unroll
            for (int kk = 0; kk < D / 16; ++kk) {
              const uint32_t off = (kk / 4) * kPanel + (kk % 4) * 32;
              mma_ss(tS, desc_at(q_desc, off), desc_at(k_desc, off), idesc_s, kk > 0 ? 1u : 0u);
            }
            const bool last = k + 1 == steps;
            if (s.last_of(k) || last) mma_commit(&bars->slot_empty[slot.at]);
            if (last) mma_commit(&bars->q_empty[x]);
            mma_commit(&bars->s_full[x]);
            // (the other's next tile, ahead of the wait for these probabilities: its slots are not to wait for those)
            if (s.single && (s.last_of(k) || last) && at + 1 < (last ? s.n_kv : tile_of(k + 1))) return skip(gone + at + 1);
            return true;
          };
          if (s.single && (steps > 0 ? tile_of(0) : s.n_kv) > 0) ok = skip(gone);
          if (ok && steps > 0) ok = mbar_wait(&bars->q_full[x], u++ & 1, abort_flag) && issue_s(0);
          for (int k = 0; ok && k < steps; ++k, ++g) {
            const int h = s.at(x, k) % kSteps;
            const Slot<D> v(gone + tile_of(k), 1);
            if (s.first_of(k) && !(ok = wait_slot(v))) break;
            // O (+)= P V, 64 keys at a time. (A new item's first may overwrite O: its probabilities come after the last results
            // have been read.)
            const SmemDescBase v_desc{kv_desc0.lo + v.at * (L::kTileBytes >> 4) + h * (kN * 128 >> 4), kv_desc0.hi};
#pragma unroll
            for (int part = 0; part < kN / 64; ++part) {
              // (polled for a while before the wait that suspends: 1.5 % at head size 128. Polls by the softmax threads: -2 %.)
              if (!(ok = mbar_wait_at<24>(&bars->p_full[x][part], g & 1, abort_flag, __LINE__))) break;
              tc_fence_after_sync();
#pragma unroll
              for (int kk = 4 * part; kk < 4 * part + 4; ++kk)
                mma_ts(tO, tS + kk * 8, desc_at(v_desc, kk * 2048), idesc_o, (k > 0 || kk > 0) ? 1u : 0u);
            }
            if (!ok) break;
            const bool last = k + 1 == steps;
            if (s.last_of(k) || last) mma_commit(&bars->slot_empty[v.at]);
            if (last) mma_commit(&bars->o_done[x]);
            else ok = issue_s(k + 1);   // over the probabilities, whose product is ahead in the pipe
          }
          // tiles that only the pair's other group sees
          if (!s.single)
            for (int j = x ? s.n_kv : s.n_first; ok && j < s.n_kv; ++j) ok = skip(gone + j);
          // (the groups' maxima and sums change hands where the next item's scores go)
          if (s.single && CLUSTER == 1 && ok) {
            mbar_arrive(&bars->parted);
            ok = mbar_wait(&bars->parted, joins++ & 1, abort_flag);
          }
          gone += s.n_kv;
          feed.give_back();
        }
        settle_products(&bars->settled[x]);
      }
    }
  } else {
    // ------------------------------ softmax ------------------------------
    setmaxnreg_inc<L::kRegsSoftmax>();
    const int x = warp / 4 - 1;
    const int quad = warp % 4;            // TMEM lane quadrant of this warp
    const int row = quad * 32 + lane;     // row within the tile = TMEM lane
    const uint32_t tlane = tmem + (static_cast<uint32_t>(quad * 32) << 16);
    const uint32_t tS = tlane + kColS + x * kN, tO = tlane + kColO + x * D;
    const float scale_log2 = p.scale * kLog2e;
    uint32_t g = 0, u = 0, joins = 0;     // steps, items with any and shared tiles of this group so far
    int gone = 0, others = 0;             // key tiles of the CTA and steps of the other group so far
    bool ok = true, shared = false;       // shared: the item before was, and its accumulators may still be read
    while (ok && feed.next(it)) {
      // (its first probabilities let a product overwrite them, its numbers others)
      if (shared && !(ok = mbar_wait(&bars->freed, (joins - 1) & 1, abort_flag))) break;
      shared = false;
      const auto s = share_of<kSteps, CLUSTER>(it, p, rank);
      const Tile t = it.tile(p, s.single ? 0 : x);
      const int steps = s.steps(x), total = it.ahead + it.count;
      const bool active = quad * 32 < t.rows;          // whether the warp has a row
      const int token = t.token0 + min(row, t.rows - 1) / p.group;   // (rows that are not there: the last one's mask)
      const int limit = it.ahead + token;
      float m = -INFINITY, l = 0.f;   // running max (log2 units, scaled) and sum
      for (int k = 0; k < steps; ++k, ++g) {
        if (!(ok = mbar_wait(&bars->s_full[x], g & 1, abort_flag))) break;
        tc_fence_after_sync();
        const int tile = s.at(x, k) / kSteps, h = s.at(x, k) % kSteps, key0 = (s.lo + tile) * kT;
        const int seen = limit - key0 - h * kN;   // the last column that the row sees
        const bool masked = __any_sync(0xffffffffu, seen < kN - 1);
        // 32 of the thread's scores
        auto load = [&](uint32_t (&sc)[32], int q) { tmem_ld32(tS + q * 32, sc); };
        auto mask = [&](uint32_t (&sc)[32], int q) {
          if (!masked) return;
#pragma unroll
          for (int e = 0; e < 32; ++e)
            if (q * 32 + e > seen) sc[e] = 0xff800000u;  // -inf
        };
        // max of the raw scores (scale > 0 commutes with max)
        float mx4[4] = {-INFINITY, -INFINITY, -INFINITY, -INFINITY};
        auto max_of = [&](const uint32_t (&sc)[32]) {
#pragma unroll
          for (int e = 0; e < 32; e += 2)
            mx4[(e >> 1) & 3] = fmax3(mx4[(e >> 1) & 3], __uint_as_float(sc[e]), __uint_as_float(sc[e + 1]));
        };
        // The step's maximum, and the accumulator to it where it has grown; false: a wait ran out.
        auto new_max = [&] {
          const float mx = __fmul_rn(fmaxf(fmax3(mx4[0], mx4[1], mx4[2]), mx4[3]), scale_log2);
          if (k == 0) {
            m = mx;  // O is first written by a product that does not accumulate: nothing to rescale
          } else if (__any_sync(0xffffffffu, row < t.rows && mx > m + kRescaleAt)) {   // (nobody else's rows decide)
            // (P V of the step before is through: these scores were issued behind it)
            const float m_new = fmaxf(m, mx);
            // m = -inf: nothing but zeros has been accumulated so far
            const float corr = (m == -INFINITY) ? 0.f : ex2(m - m_new);
#pragma unroll 1
            for (int q = 0; q < D / 16; ++q) {
              uint32_t o[16];
              tmem_ld16(tO + q * 16, o);
              tmem_wait_ld();
#pragma unroll
              for (int e = 0; e < 16; ++e) o[e] = __float_as_uint(__uint_as_float(o[e]) * corr);
              tmem_st16(tO + q * 16, o);
            }
            tmem_wait_st();
            l = __fmul_rn(l, corr);
            m = m_new;
          }
        };
        // p = exp2(s scale log2e - m). A row whose scores are all -inf so far must give p = 0, not exp2(NaN).
        float2 sum2[2] = {make_float2(0.f, 0.f), make_float2(0.f, 0.f)};
        auto weights = [&](const uint32_t (&sc)[32], uint32_t (&pk)[16]) {   // bf16 pairs (k, k + 1) per column
          const float2 sl = make_float2(scale_log2, scale_log2);
          const float neg_m = (m == -INFINITY) ? 0.f : -m;
          const float2 nm = make_float2(neg_m, neg_m);
#pragma unroll
          for (int e = 0; e < 32; e += 2) {
            const float2 y = ffma2(make_float2(__uint_as_float(sc[e]), __uint_as_float(sc[e + 1])), sl, nm);
            const float2 w = make_float2(ex2(y.x), ex2(y.y));
            sum2[(e >> 1) & 1] = fadd2(sum2[(e >> 1) & 1], w);
            pk[e / 2] = pack_bf16(w.x, w.y);
          }
        };
        auto hand_over = [&](int part) {
          if (active) tmem_wait_st();
          tc_fence_before_sync();
          __syncwarp();
          if (lane == 0) mbar_arrive(&bars->p_full[x][part]);
        };
        if (s.first_of(k) && total - key0 < kT) {
          // The sequence ends in this tile: V of the rows behind it, as far as the group goes.
          const Slot<D> v(gone + tile, 1);
          const int there = max(total - key0, h * kN), end = s.last_of(k) ? (h + 1) * kN : kT;
          if (!(ok = mbar_wait(&bars->slot_full[v.at], v.parity, abort_flag))) break;
          uint8_t* rows = smem + L::kKV + v.at * L::kTileBytes;
          for (int e = threadIdx.x % kGroup; e < (end - there) * (D / 8); e += kGroup) {
            const int r = there + e / (D / 8), ch = e % (D / 8);
            *reinterpret_cast<uint4*>(rows + (ch / 8) * kPanel + r * 128 + (ch & 7) * 16) = make_uint4(0, 0, 0, 0);
          }
          fence_proxy_async_smem();
        }
        if (D == 128) {
          uint32_t sc[4][32];
          if (active) {
#pragma unroll
            for (int q = 0; q < 4; ++q) load(sc[q], q);
            tmem_wait_ld();
#pragma unroll
            for (int q = 0; q < 4; ++q) mask(sc[q], q);
#pragma unroll
            for (int q = 0; q < 4; ++q) max_of(sc[q]);
            new_max();
          }
          // A's turn is behind B's step before, B's behind A's of the same place.
          {
            const int due = x == 0 ? min(k, s.steps(1)) : min(k + 1, s.steps(0));
            const volatile int* done = &bars->exps[1 - x][quad];
            for (int i = 0; i < 256 && *done < others + due; ++i) {}
          }
#pragma unroll
          for (int q = 0; q < 4; ++q) {
            uint32_t pk[16];
            if (active) weights(sc[q], pk);
            // (the first half's stores are through by now; waited for where they are issued they cost 4 %)
            if (q == 2) hand_over(0);
            if (active) tmem_st16(tS + q * 16, pk);
          }
          if (lane == 0) *const_cast<volatile int*>(&bars->exps[x][quad]) = static_cast<int>(g) + 1;
          hand_over(1);
        } else {
          if (active) {
            // (the probabilities go over the scores; 88 registers hold half of these, so the first half is read twice. All at once,
            // with 96 and the other warps at 48: 38 us for 16 prompts' 36.)
            uint32_t sc[32], first[16], second[16];
            load(sc, 0);
            tmem_wait_ld();
            mask(sc, 0);
            max_of(sc);
            load(sc, 1);
            tmem_wait_ld();
            mask(sc, 1);
            max_of(sc);
            new_max();
            weights(sc, second);
            load(sc, 0);
            tmem_wait_ld();
            mask(sc, 0);
            tmem_st16(tS + 16, second);
            weights(sc, first);
            tmem_st16(tS, first);
          }
          hand_over(0);
        }
        l += (sum2[0].x + sum2[1].x) + (sum2[0].y + sum2[1].y);
      }
      if (ok && steps > 0) ok = mbar_wait(&bars->o_done[x], u++ & 1, abort_flag);
      if (!ok) break;
      tc_fence_after_sync();
      const int64_t to_token = it.first + token;
      const int to_head = it.kv_head * p.group + min(row, t.rows - 1) % p.group;
      bf16* to = p.out + to_token * p.out_token + to_head * p.out_head;
      // Whether the row is written: not where a key tile that its query tile sees has a page outside the pool. Asked behind the
      // last product on these tiles, of a tile that the groups share behind the other's too: a group may have no steps of it, and
      // would find the flag as it was before the pages were looked at.
      auto write = [&] { return row < t.rows && !feed.entry()[6] && !(x == 1 && feed.entry()[7]); };
      l *= ex2(m == -INFINITY ? 0.f : m - m);   // (NaN where the max is not finite)
      if (!s.single) {
        // out = O / l, lse in natural-log units of the scaled scores
        const float f = 1.0f / l;
        const bool mine = write();
        if (active) {
#pragma unroll
          for (int q = 0; q < D / 32; ++q) {
            uint32_t o[32];
            tmem_ld32(tO + q * 32, o);
            tmem_wait_ld();
            if (mine) {
#pragma unroll
              for (int e = 0; e < 32; e += 16) {
                float y[16];
#pragma unroll
                for (int i = 0; i < 16; ++i) y[i] = __uint_as_float(o[e + i]) * f;
                store_16(to + q * 32 + e, y, p.wide);
              }
            }
          }
        }
        if (mine && p.lse) p.lse[to_token * p.heads_q + to_head] = (m + log2f(l)) * kLn2;
      } else {
        // The other group has the rest of the row's keys: each group joins one half of the columns. The rows' maxima and sums
        // change hands in the first columns of the scores.
        tmem_st2(tS, __float_as_uint(m), __float_as_uint(l));
        tmem_wait_st();
        tc_fence_before_sync();
        __syncwarp();
        if (lane == 0) mbar_arrive(&bars->joined);
        if (!(ok = mbar_wait(&bars->joined, joins & 1, abort_flag))) break;
        tc_fence_after_sync();
        const bool mine = write();
        float m1, l1;
        tmem_ld2(tlane + kColS + (1 - x) * kN, m1, l1);
        tmem_wait_ld();
        if (CLUSTER == 1) {   // (the next item's scores may go there)
          tc_fence_before_sync();
          __syncwarp();
          if (lane == 0) mbar_arrive(&bars->parted);
        }
        const float m_all = fmaxf(m, m1);
        // (a part that has seen nothing has nothing but garbage)
        const float f0 = m == -INFINITY ? 0.f : ex2(m - m_all), f1 = m1 == -INFINITY ? 0.f : ex2(m1 - m_all);
        const float l_all = l * f0 + l1 * f1;
        const float norm = CLUSTER == 1 ? 1.0f / l_all : 1.0f;
        float* acc = reinterpret_cast<float*>(smem + L::kKV) + row * L::kPitch;
        if (active) {
#pragma unroll
          for (int q = x * (D / 32); q < (x + 1) * (D / 32); ++q) {
            uint32_t o[16], o1[16];
            tmem_ld16(tO + q * 16, o);
            tmem_ld16(tlane + kColO + (1 - x) * D + q * 16, o1);
            tmem_wait_ld();
            float y[16];
#pragma unroll
            for (int i = 0; i < 16; ++i) {
              const float a = f0 == 0.f ? 0.f : __uint_as_float(o[i]) * f0;
              y[i] = (f1 == 0.f ? a : fmaf(__uint_as_float(o1[i]), f1, a)) * norm;
            }
            if (CLUSTER > 1) {
#pragma unroll
              for (int i = 0; i < 16; i += 4)
                *reinterpret_cast<float4*>(acc + q * 16 + i) = make_float4(y[i], y[i + 1], y[i + 2], y[i + 3]);
            } else if (mine) {
              store_16(to + q * 16, y, p.wide);
            }
          }
        }
        if (CLUSTER == 1 && x == 0 && mine && p.lse) p.lse[to_token * p.heads_q + to_head] = (m_all + log2f(l_all)) * kLn2;
        if (CLUSTER > 1 && x == 0) reinterpret_cast<float2*>(smem + L::kStats)[row] = make_float2(m_all, l_all);
        if (CLUSTER == 1) {
          tc_fence_before_sync();
          __syncwarp();
          if (lane == 0) mbar_arrive(&bars->freed);
          ++joins;
          shared = true;
        }
      }
      gone += s.n_kv;
      others += s.steps(1 - x);
      __syncwarp();
      feed.give_back(lane == 0);
    }
  }

  // ------------------------------ common exit ------------------------------
  tc_fence_before_sync();
  __syncthreads();
  if (warp == 1) {
    __syncwarp();
    tc_fence_after_sync();
    tmem_dealloc(tmem, kTmemCols);
  }
  if (CLUSTER > 1) {
    const volatile int* e = bars->item[0];
    it = Item{e[0], e[1], e[2], e[3], e[4], e[5]};
    cluster_arrive();
    cluster_wait();
    int bad = it.b < 0;   // (there is no item, or nobody published one)
#pragma unroll 1
    for (int r = 0; r < CLUSTER; ++r)
      bad |= ld_cluster_int(cluster_address(&bars->any_bad, r)) | ld_cluster_int(cluster_address(&bars->abort_flag, r));
    // This CTA's share of the rows, eight columns a thread.
    constexpr int kPieces = D / 8;
    const Tile t = it.tile(p, 0);
    const int share = (t.rows + CLUSTER - 1) / CLUSTER, row0 = rank * share, row1 = min(t.rows, row0 + share);
    for (int i = threadIdx.x; !bad && i < (row1 - row0) * kPieces; i += kThreads) {
      const int row = row0 + i / kPieces, col = i % kPieces * 8;
      float2 ml[CLUSTER];
      float m_all = -INFINITY, l_all = 0.f, y[8] = {};
#pragma unroll
      for (int r = 0; r < CLUSTER; ++r) ml[r] = ld_cluster2(cluster_address(smem + L::kStats + row * 8, r));
#pragma unroll
      for (int r = 0; r < CLUSTER; ++r) m_all = fmaxf(m_all, ml[r].x);
#pragma unroll
      for (int r = 0; r < CLUSTER; ++r) {
        const float f = ml[r].x == -INFINITY ? 0.f : ex2(ml[r].x - m_all);
        l_all = fmaf(ml[r].y, f, l_all);
        const uint32_t at = cluster_address(smem + L::kKV + (row * L::kPitch + col) * 4, r);
        const float4 a = ld_cluster4(at), b4 = ld_cluster4(at + 16);
        const float v[8] = {a.x, a.y, a.z, a.w, b4.x, b4.y, b4.z, b4.w};
#pragma unroll
        for (int k = 0; k < 8; ++k) y[k] = f == 0.f ? y[k] : fmaf(v[k], f, y[k]);
      }
      const float f = 1.0f / l_all;
#pragma unroll
      for (int k = 0; k < 8; ++k) y[k] *= f;
      const int64_t token = it.first + t.token0 + row / p.group;
      const int head = it.kv_head * p.group + row % p.group;
      *reinterpret_cast<uint4*>(p.out + token * p.out_token + head * p.out_head + col) =
          make_uint4(pack_bf16(y[0], y[1]), pack_bf16(y[2], y[3]), pack_bf16(y[4], y[5]), pack_bf16(y[6], y[7]));
      if (p.lse && col == 0) p.lse[token * p.heads_q + head] = (m_all + log2f(l_all)) * kLn2;
    }
    cluster_arrive();
    cluster_wait();   // (the others' shared memory stays until it has been read)
  }
  if (threadIdx.x == 0) {
    if (bars->abort_flag) report_timeout(p.status, bars->abort_flag);
    else if (bars->any_bad) atomicExch(p.status, DADATTN_E_ARG);
  }
}

struct Maps {
  CUtensorMap q, k, v;
};

template <int D, int CLUSTER>
int launch_chunk(const Maps& maps, ChunkParams p, long long items, cudaStream_t st) {
  using L = Plan<D>;
  p.sorted = items * p.cache.heads > static_cast<long long>(current_sm_count()) * L::kPerSm;
  auto kern = paged_attention_kernel<D, CLUSTER>;
  DAD_CUDA(cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, L::kBytes));
  static std::atomic<int> regs_seen;
  if (int rc = check_launch_registers(reinterpret_cast<const void*>(kern), L::kRegsLaunch, regs_seen)) return rc;
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3(static_cast<unsigned>(items * p.cache.heads * CLUSTER));
  cfg.blockDim = dim3(kThreads);
  cfg.dynamicSmemBytes = L::kBytes;
  cfg.stream = st;
  cudaLaunchAttribute attr[2];
  attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[0].val.programmaticStreamSerializationAllowed = 1;
  attr[1].id = cudaLaunchAttributeClusterDimension;
  attr[1].val.clusterDim.x = CLUSTER;
  attr[1].val.clusterDim.y = attr[1].val.clusterDim.z = 1;
  cfg.attrs = attr;
  cfg.numAttrs = CLUSTER > 1 ? 2 : 1;
  DAD_CUDA(cudaLaunchKernelEx(&cfg, kern, maps.q, maps.k, maps.v, p));
  return DADATTN_OK;
}

// How a call's tiles (of every key head) are shared out: pairs of them to a CTA, or each to a CTA or to a cluster of 2, 4 or 8.
// Pairs read a key tile once for two, and win where there are many (us, pairs / single tiles): 512 tiles of 2048 tokens behind
// 14336 of head size 128 466 / 539, 1024 tiles of 4096 128 / 147; at head size 64, where two CTAs are on an SM, 1536 of 16 x
// 1024 57 / 64, 1152 of 12 x 1024 45 / 50, 768 of 8 x 1024 36 / 36, of 16 x 512 22 / 26, of 8192 222 / 158. Of fewer tiles the
// cheapest in key tiles, 2 us each, that a group goes through: its items' own, and something for joining, by how often an SM is
// filled. One tile a CTA / 2 / 4 / 8:
//   head size 128   16 tiles, 8033 rows 70 / 40 / 27 / 38    64, 8256 72 / 43 / 57 / 109     128, 16512 142 / 147 / 175 / 274
//                   8, 60001 485 / 245 / 128 / 70            64, 256 8.8 / 11 / 25 / 71      160, 4001 87 / 83 / 90 / 150
//   head size 64    12, 1024 13.6 / 10.2 / 8.6 / 9.0         36, 1001 17 / 13 / 14 / 24      192, 4096 65 / 61 / 72 / 115
//                   15, 6322 76 / 37 / 23 / 19               128, 1512 24 / 20 / 32 / 64     32, 30128 341 / 162 / 88 / 67
// The sequences' counts and lengths are on the device, so tiles and rows are the most that there may be: rows those that the table
// has room for. Behind a wider table few tiles go to larger clusters than their rows are worth (us, tight / 8192 rows and more: 301
// tokens behind 700 rows, 12 heads of 64 12.5 / 24; one prompt of 2000, 12 of 128 26.6 / 47).
struct Sharing {
  bool pairs;
  int cluster;
};
Sharing share_out(long long tiles, long long pairs, long long most_rows, bool alike, int per_sm, int sms) {
  if (2 * tiles >= (per_sm == 1 ? 4 : 15) * sms) return {true, 1};
  const long long n = (most_rows + kT - 1) / kT;
  // how often `ctas` fill the GPU, or the part of it that clusters of their size can have (of 4 and 8: 33 and 15 on 148 SMs)
  auto fills = [&](double ctas, double slots) {
    const double x = ctas / slots;
    if (x <= 1.0) return 1.0;
    if (per_sm == 2) return std::max(1.3, 0.75 * x - 0.2);   // (two CTAs on an SM take a third as long again as one)
    return alike ? std::ceil(x) : x + 0.5;
  };
  Sharing best = {true, 1};
  // (two pairs on an SM take half as long again as one)
  double least = n * (per_sm == 2 && pairs > sms ? std::max(1.5, 0.75 * pairs / sms + 0.35) : fills(pairs, sms));
  const struct { int cluster; double slots, join; } ways[] = {{1, 1.0, 0.5}, {2, 1.0, 1.5}, {4, 0.892, 1.75}, {8, 0.811, 2.5}};
  for (const auto& w : ways) {
    const double each = static_cast<double>((n + 2 * w.cluster - 1) / (2 * w.cluster)) + w.join;
    const double cost = fills(static_cast<double>(tiles * w.cluster), w.slots * sms) * each;
    if (cost < least) least = cost, best = {false, w.cluster};
  }
  return best;
}

template <int D>
int launch_chunk_d(const Maps& maps, ChunkParams p, int max_new, long long most_rows, cudaStream_t st) {
  // Items of a key head: no more than these.
  const int tt = p.tile_tokens, B = p.cache.B;
  auto most_items = [&](int tokens) -> long long {
    const long long each = (max_new + tokens - 1) / tokens;   // of one sequence
    return std::min<long long>(each * B, p.T / tokens + B);
  };
  // (items are as long as each other, about, where one sequence has most of its rows ahead of the call)
  const Sharing how = share_out(most_items(tt) * p.cache.heads, most_items(2 * tt) * p.cache.heads, most_rows,
                                B == 1 && 2ll * max_new <= most_rows, Plan<D>::kPerSm, current_sm_count());
  p.item_tokens = how.pairs ? 2 * tt : tt;
  p.token_shift = (tt & (tt - 1)) ? -1 : log2_of(p.item_tokens);
  const long long items = most_items(p.item_tokens);
  switch (how.cluster) {
    case 1: return launch_chunk<D, 1>(maps, p, items, st);
    case 2: return launch_chunk<D, 2>(maps, p, items, st);
    case 4: return launch_chunk<D, 4>(maps, p, items, st);
    default: return launch_chunk<D, 8>(maps, p, items, st);
  }
}

}  // namespace
}  // namespace dadattn

using namespace dadattn;

extern "C" int dadattn_paged_attention_bf16(uint16_t* out, float* lse, const uint16_t* q, const int64_t* out_strides,
                                            const int64_t* q_strides, const uint16_t* k_pages, const uint16_t* v_pages,
                                            const int32_t* page_table, const int32_t* lengths, const int32_t* starts, int B,
                                            int T, int max_new, int Hq, int Hkv, int D, int pages, int page_size,
                                            int max_pages, float scale, dadattn_stream_t stream) {
  const char* name = "paged attention";
  if (int rc = check_paged(name, k_pages, v_pages, page_table, lengths, starts, B, Hkv, D, pages, page_size, max_pages)) return rc;
  if (T <= 0 || max_new <= 0) return fail(DADATTN_E_ARG, "%s: bad sizes T=%d max_new=%d", name, T, max_new);
  if (!starts && T != B) return fail(DADATTN_E_ARG, "%s: without starts T=%d is B=%d", name, T, B);
  if (Hq <= 0 || Hq % Hkv) return fail(DADATTN_E_ARG, "%s: Hq=%d must be a multiple of Hkv=%d", name, Hq, Hkv);
  if (Hq / Hkv > kT) return fail(DADATTN_E_UNSUPPORTED, "%s: %d query heads share a key head, more than %d", name, Hq / Hkv, kT);
  if (!(scale > 0.0f && scale < INFINITY)) return fail(DADATTN_E_ARG, "%s: scale must be positive and finite", name);
  if (int rc = check_packed(name, out, out_strides, 8, true, T, Hq)) return rc;
  if (int rc = check_packed(name, q, q_strides, 8, false, T, Hq)) return rc;
  if ((T > 1 && q_strides[0] == 0) || (Hq > 1 && q_strides[1] == 0))
    return fail(DADATTN_E_ARG, "%s: the queries' rows must not lie over each other", name);
  if (!aligned(lse, 4)) return fail(DADATTN_E_ARG, "%s: lse must be 4-byte aligned", name);
  ChunkParams p = {};
  p.out = reinterpret_cast<bf16*>(out), p.lse = lse;
  p.out_token = out_strides[0], p.out_head = out_strides[1];
  p.cache = PagedCache{page_table, lengths, starts, B, pages, log2_of(page_size), max_pages, Hkv};
  p.wide = aligned(out, 32) && out_strides[0] % 16 == 0 && out_strides[1] % 16 == 0;
  p.T = T, p.max_new = max_new, p.heads_q = Hq, p.group = Hq / Hkv, p.tile_tokens = kT / p.group;
  p.chunk = page_size < kT ? page_size : kT;
  p.scale = scale;
  if (max_new > T) max_new = T;   // (bounds the items)
  if ((static_cast<long long>(T) / p.tile_tokens + B) * kMaxCluster > 0x7fffffffll / Hkv)
    return fail(DADATTN_E_UNSUPPORTED, "%s: T=%d, B=%d and Hkv=%d are too many", name, T, B, Hkv);
  p.status = device_status_word();
  if (!p.status) return DADATTN_E_CUDA;
  const int rows = pages * Hkv * page_size;
  Maps maps;
  if (int rc = make_tensor_map_bf16_tokens(&maps.q, q, T, Hq, D, q_strides[0], q_strides[1], p.group, p.tile_tokens)) return rc;
  if (int rc = make_tensor_map_bf16(&maps.k, k_pages, 1, rows, D, p.chunk)) return rc;
  if (int rc = make_tensor_map_bf16(&maps.v, v_pages, 1, rows, D, p.chunk)) return rc;
  const long long most_rows = static_cast<long long>(max_pages) * page_size;
  cudaStream_t st = static_cast<cudaStream_t>(stream);
  return D == 64 ? launch_chunk_d<64>(maps, p, max_new, most_rows, st) : launch_chunk_d<128>(maps, p, max_new, most_rows, st);
}
