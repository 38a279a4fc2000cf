// Causal attention of a packed, ragged batch's new tokens over the pages of their sequences, for sm_100a (tcgen05, TMEM, TMA).
//
//   out_i = sum_j p_ij v_j,  p_ij = exp(scale q_i.k_j - lse_i),  lse_i = ln sum_j exp(scale q_i.k_j)   over j <= lengths[b] + i
//
// for token i of the count[b] that sequence b brings, whose rows are in their pages already. The `group` query heads that share
// a key head are rows of one tile: a 128-row tile is 128 / group tokens of all of them, so K and V are read once for the group
// and a short piece of a prompt still fills tiles.
//
// A CTA has two softmax groups of 128 threads (a row each), two tensor-core issuers and one ring of 128-key K and V tiles:
//   * pairs (CLUSTER = 1): two adjacent query tiles, A and B, of a sequence and key head. Both use every K / V tile of the
//     ring; while the threads of one compute exponentials the tensor pipe runs the products of the other;
//   * one tile: where a sequence has no second one, the two groups share its keys, A the even tiles of the ring, B the odd
//     ones, and join their maxima, sums and accumulators at the end;
//   * clusters: where the tiles do not fill the GPU every CTA of a cluster takes a run of one tile's keys, both groups as above,
//     and the results are joined through distributed shared memory: no workspace.
// Keys come through the page table: lane i of the producer warp fetches the i-th box of a tile (as high as a page, up to the
// tile), and looks its page up a tile ahead. Rows behind a sequence's last are not trusted: their scores are masked, and the
// softmax threads set their V to zero in shared memory before they hand over the probabilities of that tile.
//   warp 0       K / V producer                    warp 1     issuer of group A, tensor memory
//   warp 2       issuer of group B                 warp 3     Q
//   warps 4-7    softmax group A                   warps 8-11 softmax group B
// Every wait is bounded (sm100_ptx.cuh).
#include <cuda_bf16.h>

#include <algorithm>

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
constexpr int kMaxCluster = 8;
constexpr float kLog2e = 1.4426950408889634f;
constexpr float kLn2 = 0.6931471805599453f;
constexpr float kRescaleAt = 8.0f;      // log2 units: O is rescaled only when the maximum grew by 2^8
// Registers per thread once the warpgroups have rebalanced (a softmax thread holds 128 scores).
constexpr int kRegsLaunch = 168, kRegsSoftmax = 208, kRegsHelper = 88;
static_assert(2 * kGroup * kRegsSoftmax + 128 * kRegsHelper <= kThreads * kRegsLaunch,
              "the warpgroups ask for more registers than the CTA owns");
static_assert(kThreads * kRegsLaunch <= 65536 && (kRegsLaunch + 8) * kThreads > 65536,
              "kRegsLaunch is not what the compiler gives a CTA of this size");

template <int D>
struct Plan {
  static constexpr int kPanels = D / 64;
  static constexpr int kTileBytes = kPanels * kPanel;
  static constexpr int kSlots = D == 128 ? 5 : 10;          // ring of K and V tiles, K0 V0 K1 V1 ...
  static constexpr int kQ = 0;                              // [A, B]
  static constexpr int kKV = kQ + 2 * kTileBytes;           // (from Q's second tile on where there is one)
  static constexpr int kHalf = D == 128 ? 3 : 5;            // slots of a group's own ring, where there is one tile
  static constexpr int kBars = kKV + kSlots * kTileBytes;
  static constexpr int kBytes = kBars + 1024 + 2 * 2 * 128 * 4;
  static constexpr int kPitch = D + 4;                      // floats of a row of the accumulators that are joined (banks)
  static constexpr int kAcc = kT * kPitch * 4;              // in the ring's place
  static_assert(kBytes <= 232448, "shared memory budget of one CTA exceeded");
  static_assert(2 * kAcc <= kSlots * kTileBytes, "accumulators in the ring's place");
  static_assert(2 * kHalf <= kSlots + 1, "the groups' rings");
};

constexpr int kMaxSlots = 10;   // of either way of using the ring
static_assert(Plan<64>::kSlots <= kMaxSlots && Plan<128>::kSlots <= kMaxSlots && 2 * Plan<64>::kHalf <= kMaxSlots &&
              2 * Plan<128>::kHalf <= kMaxSlots, "barriers of the slots");
struct Bars {
  uint64_t q_full[2], slot_full[kMaxSlots], slot_empty[kMaxSlots];
  uint64_t s_full[2], p_full[2][2], o_done[2], settled[2];   // [group]; p_full: [group][half of the keys]
  uint32_t tmem_base;
  int abort_flag, bad;
  int item[5];   // sequence, first token of the item in it, rows ahead, first row in the packed tensors, tokens of the sequence
};
static_assert(sizeof(Bars) <= 1024, "barrier block");

struct ChunkParams {
  bf16* out;
  float* lse;
  int64_t out_token, out_head;
  PagedCache cache;
  int T, max_new, heads_q, group, tile_tokens;   // tokens of a tile: 128 / group
  int chunk;                            // rows of a K / V box
  float scale;
  int* status;
};

// A tile of a group: its rows, and how many key tiles it needs.
struct Tile {
  int token0, rows, n;
};

// K and V tiles in shared memory, K0 V0 K1 V1 ... The two tiles of a pair use one ring, each tile of which both issuers give
// back. Groups that share the keys of one tile have a ring each: an issuer that passed over the other's tiles without
// holding them could not tell their uses apart by the barriers' parity.
struct Ring {
  uint64_t *full, *empty;
  uint32_t at;   // shared-memory address of the first slot
  int len;
  __device__ __forceinline__ int slot(int i) const { return i % len; }
  __device__ __forceinline__ uint32_t use(int i) const { return (i / len) & 1; }
};

__device__ __forceinline__ float4 ld_cluster4(uint32_t addr) {
  float4 v;
  asm volatile("ld.shared::cluster.v4.f32 {%0, %1, %2, %3}, [%4];" : "=f"(v.x), "=f"(v.y), "=f"(v.z), "=f"(v.w) : "r"(addr) : "memory");
  return v;
}
__device__ __forceinline__ float ld_cluster(uint32_t addr) {
  float v;
  asm volatile("ld.shared::cluster.f32 %0, [%1];" : "=f"(v) : "r"(addr) : "memory");
  return v;
}
__device__ __forceinline__ int ld_cluster_int(uint32_t addr) {
  int v;
  asm volatile("ld.shared::cluster.s32 %0, [%1];" : "=r"(v) : "r"(addr) : "memory");
  return v;
}

// The lowest-numbered sequence whose items, `tokens` tokens each, reach index x; by one warp. item[0] < 0: there is none.
// Sequences that are refused have no items.
__device__ __forceinline__ void find_item(const ChunkParams& p, int x, int tokens, int (&item)[5]) {
  const PagedCache& c = p.cache;
  const int lane = threadIdx.x % 32;
  item[0] = -1;
  int64_t before = 0;   // items of the sequences so far
  for (int base = 0; base < c.B; base += 32) {
    int ahead = 0, first = 0, count = 0;
    if (base + lane < c.B && (!sequence_rows(c, base + lane, p.T, ahead, first, count) || count > p.max_new)) {
      atomicExch(p.status, DADATTN_E_ARG);
      count = 0;
    }
    const int mine = (count + tokens - 1) / tokens;
    int upto = mine;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const int other = __shfl_up_sync(0xffffffffu, upto, o);
      if (lane >= o) upto += other;
    }
    const unsigned reached = __ballot_sync(0xffffffffu, before + upto > x);
    if (reached) {
      const int at = __ffs(reached) - 1;
      // the last tokens first: their rows see the most keys
      const int index = mine - 1 - static_cast<int>(x - before - (upto - mine));
      item[0] = base + at;
      item[1] = __shfl_sync(0xffffffffu, index, at) * tokens;
      item[2] = __shfl_sync(0xffffffffu, ahead, at);
      item[3] = __shfl_sync(0xffffffffu, first, at);
      item[4] = __shfl_sync(0xffffffffu, count, at);
      return;
    }
    before += __shfl_sync(0xffffffffu, upto, 31);
  }
}

template <int D, int CLUSTER>
__global__ void __launch_bounds__(kThreads, 1)
paged_attention_kernel(const __grid_constant__ CUtensorMap map_q, const __grid_constant__ CUtensorMap map_k,
                       const __grid_constant__ CUtensorMap map_v, const ChunkParams p) {
  using L = Plan<D>;
  constexpr int kSlots = L::kSlots;
  // Tensor memory: the scores of group X at 128 X (its probabilities in the first 64 columns of them), O at 256 + D X.
  constexpr uint32_t kTmemCols = 512, kColS = 0, kColO = 256;
  extern __shared__ __align__(1024) uint8_t smem[];
  Bars* bars = reinterpret_cast<Bars*>(smem + L::kBars);
  float* stats = reinterpret_cast<float*>(smem + L::kBars + 1024);   // [group][m, l][128]
  volatile int* abort_flag = &bars->abort_flag;
  const int warp = threadIdx.x / 32, lane = threadIdx.x % 32;
  const int rank = CLUSTER > 1 ? blockIdx.x % CLUSTER : 0, kv_head = blockIdx.y;
  const PagedCache& c = p.cache;

  if ((smem_u32(smem) & 1023u) != 0) {  // the swizzled layouts need a 1024-byte aligned base
    if (threadIdx.x == 0) atomicExch(p.status, DADATTN_E_CUDA);
    return;
  }
  const int item_tokens = (CLUSTER > 1 ? 1 : 2) * p.tile_tokens;
  if (warp == 0) {
    pdl_wait();
    int item[5];
    find_item(p, blockIdx.x / CLUSTER, item_tokens, item);
    if (lane == 0) {
#pragma unroll
      for (int i = 0; i < 5; ++i) bars->item[i] = item[i];
    }
  }
  __syncthreads();
  const int b = bars->item[0];
  if (b < 0) return;   // (the same for a whole cluster)
  const int token0 = bars->item[1], ahead = bars->item[2], first = bars->item[3], count = bars->item[4];
  // One tile, whose keys the groups share, or two.
  const bool single = CLUSTER > 1 || token0 + p.tile_tokens >= count;
  auto tile_of = [&](int x) {
    Tile t;
    t.token0 = token0 + (single ? 0 : x * p.tile_tokens);
    const int tokens = min(count - t.token0, p.tile_tokens);
    t.rows = tokens * p.group;
    t.n = (ahead + t.token0 + tokens + kT - 1) / kT;
    return t;
  };
  // K / V tiles of this CTA: lo .. lo + n_kv - 1
  const int n_last = tile_of(1).n;
  const int lo = CLUSTER > 1 ? static_cast<int>(static_cast<int64_t>(n_last) * rank / CLUSTER) : 0;
  const int n_kv = (CLUSTER > 1 ? static_cast<int>(static_cast<int64_t>(n_last) * (rank + 1) / CLUSTER) : n_last) - lo;
  // Those of group x: every `stride`-th from `from`, `n` of them.
  const int stride = single ? 2 : 1;
  auto from_of = [&](int x) { return single ? x : 0; };
  auto tiles_of = [&](int x) { return single ? (n_kv - x + 1) / 2 : tile_of(x).n; };
  auto ring_of = [&](int x) {
    const int s = single ? x * L::kHalf : 0;
    return Ring{bars->slot_full + s, bars->slot_empty + s,
                smem_u32(smem) + L::kQ + (single ? 1 : 2) * L::kTileBytes + s * L::kTileBytes, single ? L::kHalf : kSlots};
  };

  if (threadIdx.x == 0) {
    for (int i = 0; i < kMaxSlots; ++i) {
      mbar_init(&bars->slot_full[i], 1);
      mbar_init(&bars->slot_empty[i], single ? 1 : 2);   // one arrival per issuer of the ring
    }
    for (int x = 0; x < 2; ++x) {
      mbar_init(&bars->q_full[x], 1);
      mbar_init(&bars->s_full[x], 1);
      mbar_init(&bars->p_full[x][0], kGroup);
      mbar_init(&bars->p_full[x][1], kGroup);
      mbar_init(&bars->o_done[x], 1);
      mbar_init(&bars->settled[x], 1);
    }
    bars->abort_flag = 0;
    bars->bad = 0;
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

  const int total = ahead + count;   // rows of the sequence
  if (warp < 4) {
    setmaxnreg_dec<kRegsHelper>();
    if (warp == 0) {
      // ------------------------------ K / V producer ------------------------------
      const int32_t* table = c.table + static_cast<int64_t>(b) * c.max_pages;
      const int per_tile = kT / p.chunk;
      const int box = lane % per_tile, panel = lane / per_tile;
      // the page of this lane's box; -1: no row of it is there
      auto look_up = [&](int tile) -> int {
        const int row = tile * kT + box * p.chunk;
        if (panel >= L::kPanels || row >= total) return -1;
        const int page = table[row >> c.page_shift];
        if (page >= 0 && page < c.pages) return page;
        bars->bad = 1;
        return -2;
      };
      int page = n_kv > 0 ? look_up(lo) : -1, issued0 = 0, issued1 = 0;   // tiles, by ring
      bool ok = true;
      for (int j = 0; ok && j < n_kv; ++j) {
        const int tile = lo + j, mine = page;
        if (j + 1 < n_kv) page = look_up(tile + 1);
        const int boxes = min((total - tile * kT + p.chunk - 1) / p.chunk, per_tile);
        const int row = tile * kT + box * p.chunk;
        // (a row coordinate outside the pool reads zeros)
        const int y = mine >= 0 ? ((mine * c.heads + kv_head) << c.page_shift) + (row & ((1 << c.page_shift) - 1)) : -kMaxPage;
        const int x = single ? j & 1 : 0;
        const Ring r = ring_of(x);
        int& issued = x ? issued1 : issued0;
#pragma unroll
        for (int m = 0; m < 2; ++m) {
          const int i = issued, slot = r.slot(i);
          if (i >= r.len && !(ok = warp_wait(&r.empty[slot], r.use(i) ^ 1u, abort_flag))) break;
          if (lane == 0) mbar_arrive_expect_tx(&r.full[slot], boxes * L::kPanels * p.chunk * 128);
          __syncwarp();
          if (mine != -1)
            tma_load_3d(r.at + slot * L::kTileBytes + panel * kPanel + box * p.chunk * 128, m ? &map_v : &map_k, &r.full[slot],
                        panel * 64, y, 0);
          __syncwarp();
          ++issued;
        }
      }
      if (lane == 0) {
        settle_ring(ring_of(0).full, ring_of(0).len, issued0);
        if (single) settle_ring(ring_of(1).full, ring_of(1).len, issued1);
      }
    } else if (warp == 3) {
      // ------------------------------ Q ------------------------------
      if (lane == 0) {
        const int copies = single ? 1 : 2;
        for (int x = 0; x < copies; ++x) {
          mbar_arrive_expect_tx(&bars->q_full[x], L::kPanels * p.tile_tokens * p.group * 128);
          for (int h = 0; h < L::kPanels; ++h)
            tma_load_3d(smem + L::kQ + x * L::kTileBytes + h * kPanel, &map_q, &bars->q_full[x], h * 64, kv_head * p.group,
                        first + tile_of(x).token0);
        }
        for (int x = 0; x < copies; ++x) settle(&bars->q_full[x], 0);
      }
    } else {
      // ------------------------------ MMA issuers ------------------------------
      const int x = warp - 1;
      if (elect_one()) {
        constexpr uint32_t idesc_s = make_idesc_bf16(kT, kT, 0, 0);   // Q, K: K-major
        constexpr uint32_t idesc_o = make_idesc_bf16(kT, D, 0, 1);    // P K-major, V MN-major
        const int q_at = single ? 0 : x;
        const SmemDescBase q_desc = make_desc_base_sw128(smem_u32(smem + L::kQ) + q_at * L::kTileBytes, 0);
        // (read MN-major, a V tile's two 64-column panels are kPanel apart; K-major operands ignore that offset)
        const Ring ring = ring_of(x);
        const SmemDescBase kv_desc0 = make_desc_base_sw128(ring.at, kPanel);
        const uint32_t tS = tmem + kColS + x * 128, tO = tmem + kColO + x * D;
        const int n = tiles_of(x);
        bool ok = true;
        auto wait_slot = [&](int i) -> bool { return mbar_wait(&ring.full[ring.slot(i)], ring.use(i), abort_flag); };
        auto issue_s = [&](int i) -> bool {
          if (!wait_slot(2 * i)) return false;
          const int slot = ring.slot(2 * i);
          tc_fence_after_sync();
          const SmemDescBase k_desc{kv_desc0.lo + slot * (L::kTileBytes >> 4), kv_desc0.hi};
#pragma unroll
          for (int kk = 0; kk < D / 16; ++kk) {
            const uint32_t off = (kk / 4) * kPanel + (kk % 4) * 32;
            mma_ss(tS, desc_at(q_desc, off), desc_at(k_desc, off), idesc_s, kk > 0 ? 1u : 0u);
          }
          mma_commit(&ring.empty[slot]);
          mma_commit(&bars->s_full[x]);
          return true;
        };
        ok = n == 0 || (mbar_wait(&bars->q_full[q_at], 0, abort_flag) && issue_s(0));
        for (int i = 0; ok && i < n; ++i) {
          if (!(ok = wait_slot(2 * i + 1))) break;
          const int slot = ring.slot(2 * i + 1);
          const SmemDescBase v_desc{kv_desc0.lo + slot * (L::kTileBytes >> 4), kv_desc0.hi};
#pragma unroll
          for (int h = 0; h < 2; ++h) {   // O (+)= P[:, 64 h .. 64 h + 63] V[64 h .. 64 h + 63, :]
            if (!(ok = mbar_wait(&bars->p_full[x][h], i & 1, abort_flag))) break;
            tc_fence_after_sync();
#pragma unroll
            for (int kk = 4 * h; kk < 4 * h + 4; ++kk)
              mma_ts(tO, tS + kk * 8, desc_at(v_desc, kk * 2048), idesc_o, (i > 0 || kk > 0) ? 1u : 0u);
          }
          if (!ok) break;
          mma_commit(&ring.empty[slot]);
          if (i + 1 < n) ok = issue_s(i + 1);   // over the probabilities, whose product is ahead in the pipe
          else mma_commit(&bars->o_done[x]);
        }
        // tiles of the pair's other group: given back once they are there
        if (!single)
          for (int i = 2 * n; ok && i < 2 * n_kv; ++i)
            if ((ok = wait_slot(i))) mbar_arrive(&ring.empty[ring.slot(i)]);
        settle_products(&bars->settled[x]);
      }
    }
  } else {
    // ------------------------------ softmax ------------------------------
    setmaxnreg_inc<kRegsSoftmax>();
    const int x = warp / 4 - 1;
    const int quad = warp % 4;            // TMEM lane quadrant of this warp
    const int row = quad * 32 + lane;     // row within the tile = TMEM lane
    const uint32_t tlane = tmem + (static_cast<uint32_t>(quad * 32) << 16);
    const uint32_t tS = tlane + kColS + x * 128, tO = tlane + kColO + x * D;
    const float scale_log2 = p.scale * kLog2e;
    const Tile t = tile_of(x);
    const int n = tiles_of(x);
    const bool active = quad * 32 < t.rows;          // whether the warp has a row
    const int mine = min(row, t.rows - 1);           // (rows that are not there take the last one's mask)
    const int token = t.token0 + mine / p.group, limit = ahead + token;
    float m = -INFINITY, l = 0.f;   // running max (log2 units, scaled) and sum
    bool ok = true;
    int j = from_of(x);
    for (int i = 0; i < n; ++i, j += stride) {
      if (!(ok = mbar_wait(&bars->s_full[x], i & 1, abort_flag))) break;
      tc_fence_after_sync();
      const int key0 = (lo + j) * kT;
      uint32_t s[4][32];
      if (active) {
#pragma unroll
        for (int q = 0; q < 4; ++q) tmem_ld32(tS + q * 32, s[q]);
        tmem_wait_ld();
        const int seen = limit - key0;   // the last column that the row sees
        if (__any_sync(0xffffffffu, seen < kT - 1)) {
#pragma unroll
          for (int q = 0; q < 4; ++q)
#pragma unroll
            for (int e = 0; e < 32; ++e)
              if (q * 32 + e > seen) s[q][e] = 0xff800000u;  // -inf
        }
        // max of the raw scores (scale > 0 commutes with max)
        float mx4[4] = {-INFINITY, -INFINITY, -INFINITY, -INFINITY};
#pragma unroll
        for (int q = 0; q < 4; q += 2)
#pragma unroll
          for (int e = 0; e < 32; ++e)
            mx4[e & 3] = fmax3(mx4[e & 3], __uint_as_float(s[q][e]), __uint_as_float(s[q + 1][e]));
        const float mx = __fmul_rn(fmaxf(fmax3(mx4[0], mx4[1], mx4[2]), mx4[3]), scale_log2);
        if (i == 0) {
          m = mx;  // O is first written by a product that does not accumulate: nothing to rescale
        } else if (__any_sync(0xffffffffu, row < t.rows && mx > m + kRescaleAt)) {   // (nobody else's rows decide)
          // (P V of the tile before is through: these scores were issued behind it)
          const float m_new = fmaxf(m, mx);
          // m = -inf: nothing but zeros has been accumulated so far
          const float corr = (m == -INFINITY) ? 0.f : ex2(m - m_new);
#pragma unroll 1
          for (int q = 0; q < D / 32; ++q) {
            uint32_t o[32];
            tmem_ld32(tO + q * 32, o);
            tmem_wait_ld();
#pragma unroll
            for (int e = 0; e < 32; ++e) o[e] = __float_as_uint(__uint_as_float(o[e]) * corr);
            tmem_st32(tO + q * 32, o);
          }
          tmem_wait_st();
          l = __fmul_rn(l, corr);
          m = m_new;
        }
      }
      if (total - key0 < kT) {
        // The sequence ends in this tile: V of the rows behind it.
        const Ring ring = ring_of(x);
        const int slot = ring.slot(2 * i + 1), there = total - key0;
        if (!(ok = mbar_wait(&ring.full[slot], ring.use(2 * i + 1), abort_flag))) break;
        const uint32_t v = ring.at + slot * L::kTileBytes;
        for (int e = threadIdx.x % kGroup; e < (kT - there) * (D / 8); e += kGroup) {
          const int r = there + e / (D / 8), ch = e % (D / 8);
          asm volatile("st.shared.v4.b32 [%0], {%1, %1, %1, %1};" ::"r"(v + (ch / 8) * kPanel + r * 128 + (ch & 7) * 16), "r"(0)
                       : "memory");
        }
        fence_proxy_async_smem();
      }
      // p = exp2(s scale log2e - m). A row whose scores are all -inf so far must give p = 0, not exp2(NaN).
      float2 sum2[2] = {make_float2(0.f, 0.f), make_float2(0.f, 0.f)};
      const float2 sl = make_float2(scale_log2, scale_log2);
      const float neg_m = (m == -INFINITY) ? 0.f : -m;
      const float2 nm = make_float2(neg_m, neg_m);
#pragma unroll
      for (int q = 0; q < 4; ++q) {
        if (active) {
          uint32_t pk[16];   // bf16 pairs (k, k + 1) per column
#pragma unroll
          for (int e = 0; e < 32; e += 2) {
            const float2 y = ffma2(make_float2(__uint_as_float(s[q][e]), __uint_as_float(s[q][e + 1])), sl, nm);
            const float2 w = make_float2(ex2(y.x), ex2(y.y));
            sum2[(e >> 1) & 1] = fadd2(sum2[(e >> 1) & 1], w);
            pk[e / 2] = pack_bf16(w.x, w.y);
          }
          tmem_st16(tS + q * 16, pk);
        }
        if (q & 1) {
          if (active) tmem_wait_st();
          tc_fence_before_sync();
          mbar_arrive(&bars->p_full[x][q / 2]);
        }
      }
      l += (sum2[0].x + sum2[1].x) + (sum2[0].y + sum2[1].y);
    }
    if (ok && n > 0) ok = mbar_wait(&bars->o_done[x], 0, abort_flag);
    tc_fence_after_sync();
    const int q_head = kv_head * p.group + mine % p.group;
    if (!single) {
      // Results: out = O / l, lse in natural-log units of the scaled scores. They leave through the group's Q tile, which
      // nobody reads any more: every Q K^T has completed before the last s_full was observed.
      if (ok && active && !bars->bad) {
        const float l_tot = l * ex2(m - m);   // (NaN where the max is not finite)
        const float f = 1.0f / l_tot;
        uint8_t* stage = smem + L::kQ + x * L::kTileBytes + quad * 32 * 128;   // this warp's rows
#pragma unroll
        for (int q = 0; q < D / 32; ++q) {
          uint32_t o[32];
          tmem_ld32(tO + q * 32, o);
          tmem_wait_ld();
          uint8_t* dst = stage + (q / 2) * kPanel + lane * 128;
#pragma unroll
          for (int i = 0; i < 4; ++i) {
            float y[8];
#pragma unroll
            for (int e = 0; e < 8; ++e) y[e] = __uint_as_float(o[8 * i + e]) * f;
            *reinterpret_cast<uint4*>(dst + ((((q & 1) * 4 + i) ^ (lane & 7)) << 4)) =
                make_uint4(pack_bf16(y[0], y[1]), pack_bf16(y[2], y[3]), pack_bf16(y[4], y[5]), pack_bf16(y[6], y[7]));
          }
        }
        if (p.lse && row < t.rows) p.lse[static_cast<int64_t>(first + token) * p.heads_q + q_head] = (m + log2f(l_tot)) * kLn2;
        __syncwarp();
        constexpr int kPieces = D / 8;   // 16-byte pieces of a row
#pragma unroll 4
        for (int i = lane; i < 32 * kPieces; i += 32) {
          const int r = i / kPieces, ch = i % kPieces, at = quad * 32 + r;
          if (at >= t.rows) break;
          const uint4 v = *reinterpret_cast<const uint4*>(stage + (ch / 8) * kPanel + r * 128 + (((ch & 7) ^ (r & 7)) << 4));
          bf16* dst = p.out + static_cast<int64_t>(first + t.token0 + at / p.group) * p.out_token +
                      static_cast<int64_t>(kv_head * p.group + at % p.group) * p.out_head + ch * 8;
          *reinterpret_cast<uint4*>(dst) = v;
        }
      }
    } else {
      // Both groups are through with the ring: accumulators, maxima and sums go there.
      asm volatile("bar.sync 1, %0;" ::"n"(2 * kGroup) : "memory");
      stats[x * 256 + row] = ok && n > 0 ? m : -INFINITY;
      stats[x * 256 + 128 + row] = l * ex2(m == -INFINITY ? 0.f : m - m);
      if (ok && n > 0 && active) {
        float* acc = reinterpret_cast<float*>(smem + L::kKV + x * L::kAcc) + row * L::kPitch;
#pragma unroll
        for (int q = 0; q < D / 32; ++q) {
          uint32_t o[32];
          tmem_ld32(tO + q * 32, o);
          tmem_wait_ld();
#pragma unroll
          for (int e = 0; e < 32; e += 4)
            *reinterpret_cast<uint4*>(acc + q * 32 + e) = make_uint4(o[e], o[e + 1], o[e + 2], o[e + 3]);
        }
      }
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
  if (single) {
    int bad = bars->bad | bars->abort_flag;
    if (CLUSTER > 1) {
      cluster_arrive();
      cluster_wait();
      bad = 0;
#pragma unroll 1
      for (int r = 0; r < CLUSTER; ++r)
        bad |= ld_cluster_int(cluster_address(&bars->bad, r)) | ld_cluster_int(cluster_address(&bars->abort_flag, r));
    }
    // This CTA's share of the rows, eight columns a thread.
    constexpr int kPieces = D / 8;
    const Tile t = tile_of(0);
    const int share = (t.rows + CLUSTER - 1) / CLUSTER, row0 = rank * share, row1 = min(t.rows, row0 + share);
    for (int i = threadIdx.x; !bad && i < (row1 - row0) * kPieces; i += kThreads) {
      const int row = row0 + i / kPieces, col = i % kPieces * 8;
      float m_tot = -INFINITY, l_tot = 0.f, y[8] = {};
#pragma unroll 1
      for (int r = 0; r < 2 * CLUSTER; ++r) m_tot = fmaxf(m_tot, ld_cluster(cluster_address(&stats[(r & 1) * 256 + row], r / 2)));
#pragma unroll 2
      for (int r = 0; r < 2 * CLUSTER; ++r) {
        const float mr = ld_cluster(cluster_address(&stats[(r & 1) * 256 + row], r / 2));
        const float lr = ld_cluster(cluster_address(&stats[(r & 1) * 256 + 128 + row], r / 2));
        if (mr == -INFINITY) continue;   // (nothing was accumulated)
        const float f = ex2(mr - m_tot);
        l_tot = fmaf(lr, f, l_tot);
        const uint32_t at = cluster_address(smem + L::kKV + (r & 1) * L::kAcc + (row * L::kPitch + col) * 4, r / 2);
        const float4 a = ld_cluster4(at), b4 = ld_cluster4(at + 16);
        const float v[8] = {a.x, a.y, a.z, a.w, b4.x, b4.y, b4.z, b4.w};
#pragma unroll
        for (int e = 0; e < 8; ++e) y[e] = fmaf(v[e], f, y[e]);
      }
      const float f = 1.0f / l_tot;
#pragma unroll
      for (int e = 0; e < 8; ++e) y[e] *= f;
      const int64_t token = first + t.token0 + row / p.group;
      const int head = kv_head * p.group + row % p.group;
      *reinterpret_cast<uint4*>(p.out + token * p.out_token + head * p.out_head + col) =
          make_uint4(pack_bf16(y[0], y[1]), pack_bf16(y[2], y[3]), pack_bf16(y[4], y[5]), pack_bf16(y[6], y[7]));
      if (p.lse && col == 0) p.lse[token * p.heads_q + head] = (m_tot + log2f(l_tot)) * kLn2;
    }
    if (CLUSTER > 1) {
      cluster_arrive();
      cluster_wait();   // (the others' shared memory stays until it has been read)
    }
  }
  if (threadIdx.x == 0) {
    if (bars->abort_flag) report_timeout(p.status, bars->abort_flag);
    else if (bars->bad) atomicExch(p.status, DADATTN_E_ARG);
  }
}

struct Maps {
  CUtensorMap q, k, v;
};

template <int D, int CLUSTER>
int launch_chunk(const Maps& maps, const ChunkParams& p, long long items, cudaStream_t st) {
  using L = Plan<D>;
  auto kern = paged_attention_kernel<D, CLUSTER>;
  DAD_CUDA(cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, L::kBytes));
  static std::atomic<int> regs_seen;
  if (int rc = check_launch_registers(reinterpret_cast<const void*>(kern), kRegsLaunch, regs_seen)) return rc;
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3(static_cast<unsigned>(items * CLUSTER), static_cast<unsigned>(p.cache.heads));
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

template <int D>
int launch_chunk_d(const Maps& maps, const ChunkParams& p, int max_new, long long most_rows, cudaStream_t st) {
  // Items of every key head: no more than these (the sequences' counts are on the device).
  const int tt = p.tile_tokens, B = p.cache.B;
  auto most_items = [&](int tokens) -> long long {
    const long long each = (max_new + tokens - 1) / tokens;   // of one sequence
    return std::min<long long>(each * B, p.T / tokens + B);
  };
  const long long tiles = most_items(tt), sms = current_sm_count();
  int cluster = 1;
  while (cluster < kMaxCluster && tiles * p.cache.heads * cluster * 2 <= sms && cluster * 4ll * kT <= most_rows) cluster *= 2;
  switch (cluster) {
    case 1: return launch_chunk<D, 1>(maps, p, most_items(2 * tt), st);
    case 2: return launch_chunk<D, 2>(maps, p, tiles, st);
    case 4: return launch_chunk<D, 4>(maps, p, tiles, st);
    default: return launch_chunk<D, 8>(maps, p, tiles, st);
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
  if (Hkv > 65535) return fail(DADATTN_E_UNSUPPORTED, "%s: Hkv=%d exceeds 65535", name, Hkv);
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
  p.T = T, p.max_new = max_new, p.heads_q = Hq, p.group = Hq / Hkv, p.tile_tokens = kT / p.group;
  p.chunk = page_size < kT ? page_size : kT;
  p.scale = scale;
  if (max_new > T) max_new = T;   // (bounds the items)
  if ((static_cast<long long>(T) / p.tile_tokens + B) * kMaxCluster > 0x7fffffffll)
    return fail(DADATTN_E_UNSUPPORTED, "%s: T=%d and B=%d are too many", name, T, B);
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
