// One decode step over a paged KV cache: the token of every sequence is turned by its position, appended to its page and
// attended for, in one launch.
//
//   out_r = sum_j p_rj v_j,  p_rj = exp(scale q_r.k_j - m_r) / l_r   over rows j = 0 .. lengths[b]
//
// for the `group` query heads r that share a key head: they are the 8 columns (up to 16: two times 8) of the second operand of
// the warp-wide matrix instruction (m16n8k16, bf16 in, fp32 sums), so that K and V are read once for all of them. The products are
// transposed, S^T = K Q^T and O^T = V^T P^T: 16 rows of the cache, not 16 of 1 to 8 query rows, fill the instruction's 16 (3 %
// faster than the other way round, and 32 registers fewer). Bound by HBM: 4 D bytes a cached row and key head, 2 to 16 FLOPs a
// byte; what counts is that enough of them are on their way, and that a call is over soon after its longest sequence. tcgen05
// would need its scores back from tensor memory, and 128 rows for each product.
//   * a CTA (a cluster, where few items share the GPU) per sequence, key head and 16 query heads. Of a cluster each CTA takes
//     a run of the tiles (64 or 128 rows), and they join their maxima, sums and accumulators through distributed shared memory: no
//     workspace, and nothing that two calls could share.
//   * one producer warp: lane i fetches the i-th box of a tile (TMA, 128-byte swizzle, boxes as high as a page, up to the
//     tile; 16 rows in a sequence's last tile, of which only those with a row are fetched), and looks its page up a tile ahead.
//   * four consumer warps, or eight where a CTA has its SM to itself, 16 rows of a tile each, with a running maximum and sum of
//     their own. Scores and probabilities stay in registers: as a result they lie transposed to the next product's operand, which
//     movmatrix puts right. Accumulators are rescaled only when the maximum has grown by 2^8.
//   * turned queries are not rounded to bf16: what rounding leaves is a second operand, whose products are as good as free here
//     (rounded, the result's error against 64 bits was 2.7e-3 and more of its norm; 2.1e-3 without, as without a rotation).
//   * the new token needs no row of the cache: its scores, with k as rounded for the cache, are where one warp's running
//     maximum begins, and v its accumulator.
// Measured (us, rotating caches): 64 sequences of 3 .. 1023 rows, 12 heads of 64 21 (4.9 TB/s), all of 1000 38-39 (5.1); 8 of
// 999 .. 15999, 8 key heads of 128 for 32 46 (5.6; 47 turned), one of 60000 59 (4.2); 12 heads of 64, 699 rows 5.2 (6.0 turned).
// Two warps a CTA, seven CTAs an SM: 31 for the first; eight warps, two CTAs: 23, and 53 for 128 sequences of up to 999 (45);
// persistent CTAs that take a long and a short item each 24. More figures at share_out.
// Rows behind the last one are not trusted: their scores are masked and their V set to zero in shared memory.
// Every wait is bounded (sm100_ptx.cuh).
#include <cuda_bf16.h>

#include <algorithm>
#include <climits>

#include "decode_common.cuh"
#include "paged.cuh"
#include "rotary.cuh"

namespace dadattn {
namespace {

using namespace ptx;
using bf16 = __nv_bfloat16;

constexpr int kWarpRows = 16;                 // cache rows of a consumer warp in a stage
constexpr int kRows = 16;                     // query rows of an item, at most
constexpr int kMaxCluster = 16;
// Sequences of a lane that are ranked: 128 of a call. (More come in the caller's order. us, mixed / longest first: 256 of up to 1000
// rows, 12 heads of 64 66 / 71; 256 of up to 2000, 8 of 128 156 / 153; 130 of up to 4000 163 / 151.)
constexpr int kRanked = 4;
constexpr float kLog2e = 1.4426950408889634f, kLn2 = 0.6931471805599453f;
constexpr float kRescaleAt = 8.0f;

// WARPS: consumer warps, 4, or 8 where a CTA has its SM to itself.
template <int D, int NT, int WARPS>
struct Plan {
  static constexpr int kThreads = (WARPS + 1) * 32;          // and one producer warp
  static constexpr int kTile = WARPS * kWarpRows;
  static constexpr int kPerSm = WARPS == 8 ? 1 : D == 64 ? 4 : 3;
  static constexpr int kStages = 192 * 1024 / (kPerSm * kTile * D * 4);   // 192 KB on their way into an SM
  static constexpr int kPanels = D / 64;
  static constexpr int kPanelBytes = kTile * 128;            // [kTile rows][64 bf16], swizzled
  static constexpr int kSide = kPanels * kPanelBytes;        // K or V of a tile
  static constexpr int kStageBytes = 2 * kSide;
  // Behind the ring, or in its place once it has been read: accumulators of the warps and the CTA's.
  static constexpr int kPitch = D + 4;                       // floats of a row (banks)
  static constexpr int kWarpAcc = 8 * NT * kPitch;
  static constexpr int kAccBytes = (WARPS + 1) * kWarpAcc * 4;
  static constexpr int kBytes = kStages * kStageBytes > kAccBytes ? kStages * kStageBytes : kAccBytes;
};

template <int D, int NT, int WARPS>
struct DecodeShared {
  uint64_t full[Plan<D, NT, WARPS>::kStages], empty[Plan<D, NT, WARPS>::kStages];
  int abort_flag, bad;
  float m[WARPS][kRows], l[WARPS][kRows];
  float m_all[kRows], l_all[kRows];           // of the CTA, read by the cluster's others
  __align__(16) float2 table[kMaxRotaryHead / 4];   // (cos, sin): D / 2 at most
  __align__(16) bf16 q[2][8 * NT][D + 8];           // turned queries in two parts, the second what rounding left of the first
  __align__(16) bf16 k_new[D], v_new[D];
};

struct DecodeParams {
  bf16* out;
  float* lse;
  const bf16 *q, *k_new, *v_new;
  bf16 *k_pages, *v_pages;
  int64_t out_token, out_head, q_token, q_head, k_token, k_head, v_token, v_head;
  PagedCache cache;
  int heads_q, group, parts;   // query heads of a key head, in `parts` items of up to 16
  int chunk;                   // rows of a box: those of a page, up to a tile
  float scale;
  RotaryParams r;
  int* status;
  int ranked;   // items do not all start at once: they are taken by length
};

__device__ __forceinline__ void ldmatrix4(uint32_t addr, uint32_t (&r)[4]) {
  asm volatile("ldmatrix.sync.aligned.m8n8.x4.shared.b16 {%0, %1, %2, %3}, [%4];"
               : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3])
               : "r"(addr)
               : "memory");
}
__device__ __forceinline__ void ldmatrix4_trans(uint32_t addr, uint32_t (&r)[4]) {
  asm volatile("ldmatrix.sync.aligned.m8n8.x4.trans.shared.b16 {%0, %1, %2, %3}, [%4];"
               : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3])
               : "r"(addr)
               : "memory");
}
// c (16 x 8) += a (16 x 16) b (16 x 8)
__device__ __forceinline__ void mma_16816(float (&c)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
  asm volatile(
      "mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%0, %1, %2, %3};"
      : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
      : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}
// An 8 x 8 block of 16-bit elements in the operands' layout (row lane / 4, columns 2 (lane % 4) and the next), transposed.
__device__ __forceinline__ uint32_t transpose_8x8(uint32_t x) {
  uint32_t y;
  asm volatile("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(y) : "r"(x));
  return y;
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

// The sequence of this place in an order by length, in 64ths of the longest's (so that what starts last is short), and its
// length; by every warp for itself.
__device__ __forceinline__ void by_length(const PagedCache& c, int place, int& b, int& ahead) {
  const int lane = threadIdx.x % 32;
  int lens[kRanked], units[kRanked], most = 0;
#pragma unroll
  for (int i = 0; i < kRanked; ++i) {
    lens[i] = lane + 32 * i < c.B ? c.lengths[lane + 32 * i] : INT_MIN;
    most = max(most, lens[i]);
  }
  most = __reduce_max_sync(0xffffffffu, most);
  const int unit = max(0, 26 - __clz(most));   // most < 64 << unit
#pragma unroll
  for (int i = 0; i < kRanked; ++i) units[i] = lane + 32 * i < c.B ? max(lens[i], 0) >> unit : -1;
  auto reach = [&](int least) -> int {
    int n = 0;
#pragma unroll
    for (int i = 0; i < kRanked; ++i) n += units[i] >= least;
    return __reduce_add_sync(0xffffffffu, n);
  };
  int low = 0;   // the most units that more than `place` sequences reach
#pragma unroll 1
  for (int step = 32; step; step >>= 1)
    if (reach(low + step) > place) low += step;
  int rest = place - reach(low + 1);
#pragma unroll
  for (int i = 0; i < kRanked; ++i) {
    const unsigned have = __ballot_sync(0xffffffffu, units[i] == low);
    const int many = __popc(have);
    if (rest >= 0 && rest < many) {
      const int at = __fns(have, 0, rest + 1);
      b = at + 32 * i;
      ahead = __shfl_sync(0xffffffffu, lens[i], at);
    }
    rest -= many;
  }
}

template <int D, int NT, int CLUSTER, int WARPS>
__global__ void __launch_bounds__(Plan<D, NT, WARPS>::kThreads, Plan<D, NT, WARPS>::kPerSm)
paged_decode_kernel(const __grid_constant__ CUtensorMap map_k, const __grid_constant__ CUtensorMap map_v,
                    const __grid_constant__ CUtensorMap map_k16, const __grid_constant__ CUtensorMap map_v16,
                    const DecodeParams p) {
  using L = Plan<D, NT, WARPS>;
  constexpr int kStages = L::kStages, kSteps = D / 16, kTile = L::kTile, kThreads = L::kThreads;
  extern __shared__ __align__(1024) uint8_t smem[];
  __shared__ DecodeShared<D, NT, WARPS> sh;
  volatile int* abort_flag = &sh.abort_flag;
  const PagedCache& c = p.cache;
  const int warp = threadIdx.x / 32, lane = threadIdx.x % 32;
  const int rank = CLUSTER > 1 ? blockIdx.x % CLUSTER : 0;
  const int item = blockIdx.x / CLUSTER;
  const int per_seq = c.heads * p.parts;
  const int place = item / per_seq, kv_head = (item - place * per_seq) / p.parts, part = item % p.parts;
  const int head0 = kv_head * p.group + part * kRows, rows = min(p.group - part * kRows, kRows);

  if ((smem_u32(smem) & 1023u) != 0) {
    if (threadIdx.x == 0) atomicExch(p.status, DADATTN_E_CUDA);
    return;
  }
  if (threadIdx.x == 0) {
    for (int s = 0; s < kStages; ++s) {
      mbar_init(&sh.full[s], 1);
      mbar_init(&sh.empty[s], WARPS);
    }
    sh.abort_flag = 0;
    sh.bad = 0;
    fence_mbar_init();
  }
  __syncthreads();
  pdl_wait();
  pdl_launch_dependents();

  int b = place, ahead;
  if (p.ranked) by_length(c, place, b, ahead);
  else ahead = c.lengths[b];
  // (the same for every CTA of a cluster: nobody waits for one that has left)
  if (ahead < 0 || ahead >= c.max_pages << c.page_shift) {
    if (threadIdx.x == 0) atomicExch(p.status, DADATTN_E_ARG);
    return;
  }
  const int n_tiles = (ahead + kTile - 1) / kTile;
  const int first_tile = static_cast<int>(static_cast<int64_t>(n_tiles) * rank / CLUSTER);
  const int end_tile = static_cast<int>(static_cast<int64_t>(n_tiles) * (rank + 1) / CLUSTER);
  const int n = end_tile - first_tile;
  const bool last_rank = rank == CLUSTER - 1;   // has the new token

  // Transposed: O^T is 16 columns of O and 8 query rows at a time. A lane has query rows 2 (lane % 4) and the one behind it,
  // of elements (o[..][0], o[..][1]) lane / 4 and (o[..][2], o[..][3]) 8 behind that.
  float o[kSteps][NT][4], m[NT][2], l[NT][2];
#pragma unroll
  for (int t = 0; t < NT; ++t) m[t][0] = m[t][1] = -INFINITY, l[t][0] = l[t][1] = 0.f;
  if (warp == WARPS) {
    // ------------------------------ producer ------------------------------
    const int32_t* table = c.table + static_cast<int64_t>(b) * c.max_pages;
    int issued = 0;
    auto plan = [&](int tile, int& box_rows, int& boxes) {   // boxes of one side and panel
      const int there = min(ahead - tile * kTile, kTile);
      box_rows = there < kTile ? 16 : p.chunk;
      boxes = (there + box_rows - 1) / box_rows;
    };
    // the page of this lane's box of a tile
    auto look_up = [&](int tile) -> int {
      int box_rows, boxes;
      plan(tile, box_rows, boxes);
      const int i = lane % boxes;
      return lane < boxes * L::kPanels * 2 ? table[(tile * kTile + i * box_rows) >> c.page_shift] : 0;
    };
    int page = n > 0 ? look_up(first_tile) : 0;
    for (int j = 0; j < n; ++j) {
      const int s = j % kStages, tile = first_tile + j;
      int box_rows, boxes;
      plan(tile, box_rows, boxes);
      const int count = boxes * L::kPanels * 2, mine = page;
      if (j + 1 < n) page = look_up(tile + 1);
      if (j >= kStages && !warp_wait(&sh.empty[s], (j / kStages - 1) & 1, abort_flag)) break;
      if (lane == 0) mbar_arrive_expect_tx(&sh.full[s], count * box_rows * 128);
      __syncwarp();
      if (lane < count) {
        const int i = lane % boxes, panel = lane / boxes % L::kPanels, side = lane / (boxes * L::kPanels);
        const int row = tile * kTile + i * box_rows;
        const bool good = mine >= 0 && mine < c.pages;
        if (!good) sh.bad = 1;
        // (a row coordinate outside the pool reads zeros)
        const int y = good ? ((mine * c.heads + kv_head) << c.page_shift) + (row & ((1 << c.page_shift) - 1)) : -kMaxPage;
        const CUtensorMap* map = side ? (box_rows == 16 ? &map_v16 : &map_v) : (box_rows == 16 ? &map_k16 : &map_k);
        tma_load_3d(smem + s * L::kStageBytes + side * L::kSide + panel * L::kPanelBytes + i * box_rows * 128, map, &sh.full[s],
                    panel * 64, y, 0);
      }
      __syncwarp();
      ++issued;
    }
    if (lane == 0) settle_ring(sh.full, kStages, issued);
  } else {
    // ------------------------------ set-up of the consumers ------------------------------
    const int t = threadIdx.x;
    constexpr int kConsumers = WARPS * 32, kUnits = D / kTurnUnit;
    const int half = p.r.rot / 2;
    // pieces of 16 elements: of the query rows, then of k and v
    const int pieces = (8 * NT + 2) * kUnits;
    for (int e = t; e < half; e += kConsumers) sh.table[e] = cos_sin<false>(ahead, p.r.turns[e], p.r.factor);
    // (not the producer, who is at work)
    auto consumers_meet = [] { asm volatile("bar.sync 1, %0;" ::"n"(kConsumers) : "memory"); };
    consumers_meet();
    const int new_page = last_rank ? c.table[static_cast<int64_t>(b) * c.max_pages + (ahead >> c.page_shift)] : 0;
    const bool can_append = new_page >= 0 && new_page < c.pages;
    if (!can_append) sh.bad = 1;
    const int64_t new_row = (((static_cast<int64_t>(new_page) * c.heads + kv_head) << c.page_shift) +
                             (ahead & ((1 << c.page_shift) - 1))) * D;
    const bool turned = p.r.rot > 0;
    for (int i = t; i < pieces; i += kConsumers) {
      const int row = i / kUnits, u = i % kUnits;
      const bool is_v = row == (8 * NT) + 1;
      const int first = is_v ? u * kTurnUnit : unit_first(u, p.r), second = is_v ? 8 : unit_second(u, p.r);
      if (row >= (8 * NT) && !last_rank) continue;
      Sixteen<bf16> x, rest;
      rest.a = rest.b = make_uint4(0, 0, 0, 0);
      if (row < (8 * NT)) {
        if (row < rows) x.load(p.q, b * p.q_token + (head0 + row) * p.q_head + first, second);
        else x.a = x.b = make_uint4(0, 0, 0, 0);
      } else if (is_v) {
        x.load(p.v_new, b * p.v_token + kv_head * p.v_head + first, second);
      } else {
        x.load(p.k_new, b * p.k_token + kv_head * p.k_head + first, second);
      }
      if (!is_v && u * kTurnUnit < p.r.rot) {
        float f[16];
        x.to_floats(f);
        float2 cs[8];
#pragma unroll
        for (int k = 0; k < 8; ++k) cs[k] = sh.table[u * 8 + k];
        turn_unit(f, cs, p.r.interleaved);
        x.from_floats(f);
        float g[16];
        x.to_floats(g);
#pragma unroll
        for (int k = 0; k < 16; ++k) f[k] -= g[k];
        rest.from_floats(f);
      }
      if (turned && row < (8 * NT)) rest.store(sh.q[1][row], first, second);
      x.store(row < (8 * NT) ? sh.q[0][row] : is_v ? sh.v_new : sh.k_new, first, second);
      if (row >= (8 * NT) && part == 0 && can_append) x.store(is_v ? p.v_pages : p.k_pages, new_row + first, second);
    }
    consumers_meet();

    uint32_t qf[kSteps][NT][2];
#pragma unroll
    for (int s = 0; s < kSteps; ++s)
#pragma unroll
      for (int t = 0; t < NT; ++t)
#pragma unroll
        for (int h = 0; h < 2; ++h)
          qf[s][t][h] = *reinterpret_cast<const uint32_t*>(&sh.q[0][8 * t + lane / 4][s * 16 + (lane % 4) * 2 + 8 * h]);
    auto rest_of = [&](int s, int t, int h) {
      return *reinterpret_cast<const uint32_t*>(&sh.q[1][8 * t + lane / 4][s * 16 + (lane % 4) * 2 + 8 * h]);
    };
    const float scale_log2 = p.scale * kLog2e;
#pragma unroll
    for (int i = 0; i < kSteps; ++i)
#pragma unroll
      for (int t = 0; t < NT; ++t) o[i][t][0] = o[i][t][1] = o[i][t][2] = o[i][t][3] = 0.f;
    if (last_rank && warp == 0) {
#pragma unroll
      for (int t = 0; t < NT; ++t) {
        float2 dot = make_float2(0.f, 0.f);   // of query row lane / 4, by the quad
#pragma unroll
        for (int s = 0; s < kSteps; ++s)
#pragma unroll
          for (int h = 0; h < 2; ++h) {
            const uint32_t k = *reinterpret_cast<const uint32_t*>(&sh.k_new[s * 16 + (lane % 4) * 2 + 8 * h]);
            fma_bf16(dot, qf[s][t][h], k);
            if (turned) fma_bf16(dot, rest_of(s, t, h), k);
          }
        float d = dot.x + dot.y;
        d += __shfl_xor_sync(0xffffffffu, d, 1);
        d += __shfl_xor_sync(0xffffffffu, d, 2);
        d = __fmul_rn(d, scale_log2);
#pragma unroll
        for (int x = 0; x < 2; ++x) {
          m[t][x] = __shfl_sync(0xffffffffu, d, 4 * (2 * (lane % 4) + x));
          // (1; NaN where the score is infinite or NaN, 0 for minus infinity. The lanes' parts are added up.)
          l[t][x] = lane / 4 == 0 && m[t][x] != -INFINITY ? ex2(m[t][x] - m[t][x]) : 0.f;
        }
      }
#pragma unroll
      for (int i = 0; i < kSteps; ++i)
#pragma unroll
        for (int t = 0; t < NT; ++t)
#pragma unroll
          for (int e = 0; e < 4; ++e)
            o[i][t][e] = m[t][e & 1] == -INFINITY ? 0.f : __bfloat162float(sh.v_new[i * 16 + lane / 4 + 8 * (e >> 1)]);
    }

    // ------------------------------ the tiles ------------------------------
    const uint32_t ring = smem_u32(smem);
    for (int j = 0; j < n; ++j) {
      const int s = j % kStages, tile = first_tile + j;
      const int there = min(ahead - tile * kTile - warp * kWarpRows, kWarpRows);   // rows of this warp's 16
      if (!warp_wait(&sh.full[s], (j / kStages) & 1, abort_flag)) break;
      if (there > 0) {
        const uint32_t k_tile = ring + s * L::kStageBytes + warp * kWarpRows * 128, v_tile = k_tile + L::kSide;
        // scores, transposed: S^T (16 rows of the cache x 8 query rows) = K Q^T
        float sc[NT][4] = {};
#pragma unroll
        for (int step = 0; step < kSteps; ++step) {
          uint32_t kf[4];
          const int key = lane & 15, ch = step * 2 + (lane >> 4);
          ldmatrix4(k_tile + (ch / 8) * L::kPanelBytes + key * 128 + (((ch & 7) ^ (key & 7)) << 4), kf);
#pragma unroll
          for (int t = 0; t < NT; ++t) mma_16816(sc[t], kf, qf[step][t][0], qf[step][t][1]);
          if (turned) {
#pragma unroll
            for (int t = 0; t < NT; ++t) mma_16816(sc[t], kf, rest_of(step, t, 0), rest_of(step, t, 1));
          }
        }
        if (there < kWarpRows) {
          // Rows that are not there: no score, and a V of zeros (what the page holds there could be anything).
#pragma unroll
          for (int t = 0; t < NT; ++t)
#pragma unroll
            for (int e = 0; e < 4; ++e)
              if (lane / 4 + 8 * (e >> 1) >= there) sc[t][e] = -INFINITY;
          for (int i = lane; i < (kWarpRows - there) * D / 8; i += 32) {
            const int row = there + i / (D / 8), ch = i % (D / 8);
            const uint32_t at = v_tile + (ch / 8) * L::kPanelBytes + row * 128 + ((ch & 7) << 4);
            asm volatile("st.shared.v4.b32 [%0], {%1, %1, %1, %1};" ::"r"(at), "r"(0) : "memory");
          }
          fence_proxy_async_smem();
          __syncwarp();
        }
        bool grown = false;
        float mx[NT][2];
#pragma unroll
        for (int t = 0; t < NT; ++t)
#pragma unroll
          for (int x = 0; x < 2; ++x) {
            mx[t][x] = __fmul_rn(fmaxf(sc[t][x], sc[t][2 + x]), scale_log2);
            grown |= mx[t][x] > m[t][x] + kRescaleAt || m[t][x] == -INFINITY;
          }
        if (__any_sync(0xffffffffu, grown)) {
#pragma unroll
          for (int t = 0; t < NT; ++t)
#pragma unroll
            for (int x = 0; x < 2; ++x) {
#pragma unroll
              for (int d = 4; d < 32; d <<= 1) mx[t][x] = fmaxf(mx[t][x], __shfl_xor_sync(0xffffffffu, mx[t][x], d));
              const float m_new = fmaxf(m[t][x], mx[t][x]);
              const float corr = m[t][x] == -INFINITY ? 0.f : ex2(m[t][x] - m_new);
              m[t][x] = m_new;
              l[t][x] = __fmul_rn(l[t][x], corr);
#pragma unroll
              for (int i = 0; i < kSteps; ++i) o[i][t][x] *= corr, o[i][t][2 + x] *= corr;
            }
        }
        uint32_t pf[NT][2];   // P^T as the second operand: the 8 x 8 blocks of the scores' layout, transposed
#pragma unroll
        for (int t = 0; t < NT; ++t) {
          float e[4];
#pragma unroll
          for (int i = 0; i < 4; ++i) e[i] = ex2(fmaf(sc[t][i], scale_log2, m[t][i & 1] == -INFINITY ? 0.f : -m[t][i & 1]));
          l[t][0] += e[0] + e[2];
          l[t][1] += e[1] + e[3];
          pf[t][0] = transpose_8x8(pack_bf16(e[0], e[1]));
          pf[t][1] = transpose_8x8(pack_bf16(e[2], e[3]));
        }
        // O^T += V^T P^T, 16 columns of V at a time
#pragma unroll
        for (int i = 0; i < kSteps; ++i) {
          uint32_t vf[4];
          const int key = (lane & 7) + (lane >> 4) * 8, ch = i * 2 + ((lane >> 3) & 1);
          ldmatrix4_trans(v_tile + (ch / 8) * L::kPanelBytes + key * 128 + (((ch & 7) ^ (key & 7)) << 4), vf);
#pragma unroll
          for (int t = 0; t < NT; ++t) mma_16816(o[i][t], vf, pf[t][0], pf[t][1]);
        }
      }
      __syncwarp();
      if (lane == 0) mbar_arrive(&sh.empty[s]);
    }
#pragma unroll
    for (int t = 0; t < NT; ++t)
#pragma unroll
      for (int x = 0; x < 2; ++x)
#pragma unroll
        for (int d = 4; d < 32; d <<= 1) l[t][x] += __shfl_xor_sync(0xffffffffu, l[t][x], d);
  }

  // ------------------------------ the warps', then the CTAs' results together ------------------------------
  __syncthreads();   // (nobody reads the ring any more; the producer has seen its copies land)
  float* acc = reinterpret_cast<float*>(smem);               // [warps][rows][kPitch]
  float* sum = acc + WARPS * L::kWarpAcc;                   // [rows][kPitch]
  if (warp < WARPS) {
#pragma unroll
    for (int t = 0; t < NT; ++t)
#pragma unroll
      for (int x = 0; x < 2; ++x) {
        const int row = 8 * t + 2 * (lane % 4) + x;
        if (row < rows) {
#pragma unroll
          for (int i = 0; i < kSteps; ++i)
#pragma unroll
            for (int h = 0; h < 2; ++h) acc[warp * L::kWarpAcc + row * L::kPitch + i * 16 + lane / 4 + 8 * h] = o[i][t][2 * h + x];
          if (lane < 4) sh.m[warp][row] = m[t][x], sh.l[warp][row] = l[t][x];
        }
      }
  }
  __syncthreads();
  auto write_out = [&](int row, int col, float a, float b2, float l_tot) {
    const float f = 1.0f / l_tot;
    *reinterpret_cast<uint32_t*>(p.out + b * p.out_token + (head0 + row) * p.out_head + col) = pack_bf16(a * f, b2 * f);
  };
  for (int i = threadIdx.x; i < rows * (D / 2); i += kThreads) {
    const int row = i / (D / 2), col = i % (D / 2) * 2;
    float m_tot = sh.m[0][row];
#pragma unroll
    for (int w = 1; w < WARPS; ++w) m_tot = fmaxf(m_tot, sh.m[w][row]);
    float l_tot = 0.f, a = 0.f, b2 = 0.f;
#pragma unroll
    for (int w = 0; w < WARPS; ++w) {
      const float mw = sh.m[w][row], f = mw == -INFINITY ? 0.f : ex2(mw - m_tot);
      const float2 v = *reinterpret_cast<const float2*>(acc + w * L::kWarpAcc + row * L::kPitch + col);
      l_tot = fmaf(sh.l[w][row], f, l_tot);
      a = fmaf(v.x, f, a);
      b2 = fmaf(v.y, f, b2);
    }
    if (CLUSTER == 1) {
      if (!sh.bad && !sh.abort_flag) {
        write_out(row, col, a, b2, l_tot);
        if (p.lse && col == 0) p.lse[static_cast<int64_t>(b) * p.heads_q + head0 + row] = (m_tot + log2f(l_tot)) * kLn2;
      }
    } else {
      *reinterpret_cast<float2*>(sum + row * L::kPitch + col) = make_float2(a, b2);
      if (col == 0) sh.m_all[row] = m_tot, sh.l_all[row] = l_tot;
    }
  }
  if (CLUSTER > 1) {
    cluster_arrive();
    cluster_wait();
    int bad = 0;
#pragma unroll 1
    for (int r = 0; r < CLUSTER; ++r)
      bad |= ld_cluster_int(cluster_address(&sh.bad, r)) | ld_cluster_int(cluster_address(&sh.abort_flag, r));
    // this CTA's share of the results
    const int all = rows * (D / 2), share = (all + CLUSTER - 1) / CLUSTER;
    for (int i = rank * share + threadIdx.x; i < min(all, (rank + 1) * share); i += kThreads) {
      const int row = i / (D / 2), col = i % (D / 2) * 2;
      float mr[CLUSTER], m_tot = -INFINITY;
#pragma unroll
      for (int r = 0; r < CLUSTER; ++r) mr[r] = ld_cluster(cluster_address(&sh.m_all[row], r));
#pragma unroll
      for (int r = 0; r < CLUSTER; ++r) m_tot = fmaxf(m_tot, mr[r]);
      float l_tot = 0.f, a = 0.f, b2 = 0.f;
#pragma unroll
      for (int r = 0; r < CLUSTER; ++r) {
        const float f = mr[r] == -INFINITY ? 0.f : ex2(mr[r] - m_tot);
        const uint32_t at = cluster_address(sum + row * L::kPitch + col, r);
        l_tot = fmaf(ld_cluster(cluster_address(&sh.l_all[row], r)), f, l_tot);
        a = fmaf(ld_cluster(at), f, a);
        b2 = fmaf(ld_cluster(at + 4), f, b2);
      }
      if (!bad) {
        write_out(row, col, a, b2, l_tot);
        if (p.lse && col == 0) p.lse[static_cast<int64_t>(b) * p.heads_q + head0 + row] = (m_tot + log2f(l_tot)) * kLn2;
      }
    }
    cluster_arrive();
    cluster_wait();   // (the others' shared memory stays until it has been read)
  }
  if (threadIdx.x == 0) {
    if (sh.abort_flag) report_timeout(p.status, sh.abort_flag);
    else if (sh.bad) atomicExch(p.status, DADATTN_E_ARG);
  }
}

struct Maps {
  CUtensorMap k, v, k16, v16;
};

template <int D, int NT, int CLUSTER, int WARPS>
struct Launch {
  using L = Plan<D, NT, WARPS>;
  static int prepare() {
    auto kern = paged_decode_kernel<D, NT, CLUSTER, WARPS>;
    DAD_CUDA(cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, L::kBytes));
    if (CLUSTER > 8) DAD_CUDA(cudaFuncSetAttribute(kern, cudaFuncAttributeNonPortableClusterSizeAllowed, 1));
    return DADATTN_OK;
  }
  static void configure(cudaLaunchConfig_t& cfg, cudaLaunchAttribute (&attr)[2], int items, cudaStream_t st) {
    cfg.gridDim = dim3(static_cast<unsigned>(items) * CLUSTER);
    cfg.blockDim = dim3(L::kThreads);
    cfg.dynamicSmemBytes = L::kBytes;
    cfg.stream = st;
    attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr[0].val.programmaticStreamSerializationAllowed = 1;
    attr[1].id = cudaLaunchAttributeClusterDimension;
    attr[1].val.clusterDim.x = CLUSTER;
    attr[1].val.clusterDim.y = attr[1].val.clusterDim.z = 1;
    cfg.attrs = attr;
    cfg.numAttrs = CLUSTER > 1 ? 2 : 1;
  }
  // Items that the GPU works on at once. (Clusters stay within a part of the GPU, and not all of these are of one size.)
  static int places(int dev) {
    if (CLUSTER == 1) return current_sm_count() * L::kPerSm;
    static std::atomic<int> seen[64];   // by device; 1 more, 0: not asked yet
    if (dev < 0 || dev >= 64) return 0;
    int n = seen[dev].load(std::memory_order_relaxed) - 1;
    if (n >= 0) return n;
    cudaLaunchConfig_t cfg = {};
    cudaLaunchAttribute attr[2];
    configure(cfg, attr, 1, nullptr);
    cfg.attrs = attr + 1, cfg.numAttrs = 1;
    if (prepare() != DADATTN_OK ||
        cudaOccupancyMaxActiveClusters(&n, paged_decode_kernel<D, NT, CLUSTER, WARPS>, &cfg) != cudaSuccess) {
      cudaGetLastError();
      return 0;   // (no cluster of this size: not taken)
    }
    seen[dev].store(n + 1, std::memory_order_relaxed);
    return n;
  }
  static int run(const Maps& maps, DecodeParams p, int items, cudaStream_t st) {
    p.ranked = p.cache.B > 1 && p.cache.B <= 32 * kRanked &&
               static_cast<long long>(items) * CLUSTER > static_cast<long long>(current_sm_count()) * L::kPerSm;
    if (int rc = prepare()) return rc;
    cudaLaunchConfig_t cfg = {};
    cudaLaunchAttribute attr[2];
    configure(cfg, attr, items, st);
    DAD_CUDA(cudaLaunchKernelEx(&cfg, paged_decode_kernel<D, NT, CLUSTER, WARPS>, maps.k, maps.v, maps.k16, maps.v16, p));
    return DADATTN_OK;
  }
};

// The instance for `cluster` CTAs of an item: f(Launch<...>()).
template <int D, int NT, int WARPS, typename F>
int with_cluster(int cluster, F f) {
  switch (cluster) {
    case 1: return f(Launch<D, NT, 1, WARPS>());
    case 2: return f(Launch<D, NT, 2, WARPS>());
    case 4: return f(Launch<D, NT, 4, WARPS>());
    case 8: return f(Launch<D, NT, 8, WARPS>());
    default: return f(Launch<D, NT, 16, WARPS>());
  }
}

// How items are shared out: to clusters of so many CTAs, each by itself on its SM with eight consumer warps (`alone`), or with
// others and four. A CTA is bound by its warps' waits for their own steps: 16 rows of a tile take a warp 1450 clk at head size 64,
// whatever the ring holds (three times as deep a ring: nothing), so that eight warps are as good as twice the cluster, which has
// more to join. us, clusters of 1 / 2 / 4 / 8 / 16 with four warps, and with eight (-: they do not all fit):
//   1 x 12 heads of 64, 699 rows    9.4 / 7.2 / 5.6 / 5.7 / 6.9      - / - / 5.2 / 5.6 / -
//   1 x 13 of 64, 2000              23 / 14 / 8.7 / 6.9 / 7.7        14 / 9.4 / 6.7 / 6.2 / -
//   1 x 7 of 128, 16000             190 / 98 / 52 / 30 / 20          115 / 61 / 33 / 20 / 16
//   1 x 18 of 128, 16000            191 / 98 / 53 / 33 / 28          116 / 61 / 34 / - / -
//   1 x 24 of 128, 16000            191 / 98 / 53 / 35 / -           116 / 61 / 34 / - / -
//   8 x 4 of 128, up to 3750        47 / 27 / 17 / 13 / -            30 / 18 / 12 / - / -
//   64 x 2 of 128, up to 694        11.3 / 9.1 / - / - / -           8.2 / - / - / - / -
//   64 x 12 of 64, up to 1023       21 / 30 / 48 / 88 / 230          -
//   8 x 8 of 128, up to 15999       187 / 98 / 60 / 46 / 67          -
//   32 x 8 of 128, up to 3999       58 / 48 / 53 / 79 / 140          -
// Eight key heads are where the two ways meet, clusters of 16 with four warps and of 8 with eight, and the tie goes to the second,
// which is faster up to some 30000 rows and slower behind that:
//   1 x 8 of 128: 4000 rows 9.6 and 8.4, 8000 13.8 and 12.8, 16000 20.9 and 20.0, 30000 32.3 and 32.5, 60000 56.5 and 58.8,
//   120000 104.6 and 111.0; 1 x 12 of 64: 16000 17.6 and 17.0, 60000 46.9 and 48.7; 1 x 10 of 128: 60000 59.6 and 59.0
// More than 8 query heads to a key head (NT = 2; five of its instances at head size 128 spill 8 to 16 bytes):
//   1 x 8 x 16 of 64, 4000 rows     45 / 26 / 15 / 10.9 / 10.1       28 / 16 / 10.6 / 8.2 / 16
//   1 x 1 x 12 of 128, 16000        256 / 130 / 69 / 38 / 24         120 / 63 / 35 / 21 / 14.7
//   16 x 1 x 16 of 64, up to 3875   43 / 25 / 15 / 10.8 / 10.5       27 / 16 / 10.5 / 14 / 26
//   16 x 8 x 12 of 128, up to 3875  68 / 44 / 31.6 / 47 / -          35 / 32 / 49 / 94 / -
//   64 x 1 x 12 of 128, up to 992   20 / 14.5 / 11.7 / 19 / 42       11.5 / 9.4 / 16 / 41 / 94
//   64 x 8 x 16 of 64, up to 992    18 / 24 / - / - / -              29 / 53 / - / - / -
//   16 x 8 x 32 of 128, up to 3875  74 / 47 / 54 / - / -             37.8 / 56 / 90 / - / -   (the rule: 47)
// So as many CTAs to an item as all items have room for at once (half as many items again where there are several sequences, of
// different lengths, and long ones), and no more than have two and a half tiles each of the longest sequence that there may be (of
// eight warps' tiles, which are 128 rows, one and a quarter, but in clusters of 16). The longest sequence that there may be is what
// the table has room for: behind a wider one clusters are larger than the rows are worth. (us, tight / 8192 rows and more: 8
// sequences of 300 rows, 8 key heads of 128 6.0 / 15.1, of 1000 9.3 / 18.8; 16 of 300, 12 of 64 6.3 / 12.5; one of 100, 12 of 64
// 3.6 / 6.0, of 700 5.5 / 5.9.)
struct Sharing {
  int cluster;
  bool alone;
};
template <int D, int NT>
Sharing share_out(int items, int sequences, long long most_rows) {
  int dev = 0;
  if (cudaGetDevice(&dev) != cudaSuccess) return {1, false};
  auto places = [&](int cluster, bool alone) {
    auto ask = [&](auto launch) { return decltype(launch)::places(dev); };
    return alone ? with_cluster<D, NT, 8>(cluster, ask) : with_cluster<D, NT, 4>(cluster, ask);
  };
  auto holds = [&](int cluster) {
    const long long n = places(cluster, false);
    return items <= n || (sequences > 1 && 2ll * items <= 3 * n && most_rows >= 512ll * cluster);
  };
  int c = 1, a = 0;
  while (c < kMaxCluster && most_rows >= 320ll * c && holds(2 * c)) c *= 2;
  for (int k = 1; k <= kMaxCluster && most_rows >= (k == 1 ? 0 : k == kMaxCluster ? 320ll * k : 160ll * k); k *= 2)
    if (items <= places(k, true)) a = k;
  return 2 * a >= c ? Sharing{a, true} : Sharing{c, false};
}

template <int D, int NT>
int launch_decode(DecodeParams& p, int items, int page_size, cudaStream_t st) {
  const PagedCache& c = p.cache;
  const Sharing how = share_out<D, NT>(items, c.B, static_cast<long long>(c.max_pages) * page_size);
  const int tile = how.alone ? Plan<D, NT, 8>::kTile : Plan<D, NT, 4>::kTile, rows = c.pages * c.heads * page_size;
  p.chunk = std::min(page_size, tile);
  Maps maps;
  if (int rc = make_tensor_map_bf16(&maps.k, p.k_pages, 1, rows, D, p.chunk)) return rc;
  if (int rc = make_tensor_map_bf16(&maps.v, p.v_pages, 1, rows, D, p.chunk)) return rc;
  if (int rc = make_tensor_map_bf16(&maps.k16, p.k_pages, 1, rows, D, 16)) return rc;
  if (int rc = make_tensor_map_bf16(&maps.v16, p.v_pages, 1, rows, D, 16)) return rc;
  auto run = [&](auto launch) { return decltype(launch)::run(maps, p, items, st); };
  return how.alone ? with_cluster<D, NT, 8>(how.cluster, run) : with_cluster<D, NT, 4>(how.cluster, run);
}

}  // namespace
}  // namespace dadattn

using namespace dadattn;

extern "C" int dadattn_decode_paged_bf16(uint16_t* out, float* lse, const uint16_t* q, const uint16_t* k_new,
                                         const uint16_t* v_new, const int64_t* out_strides, const int64_t* q_strides,
                                         const int64_t* k_strides, const int64_t* v_strides, uint16_t* k_pages,
                                         uint16_t* v_pages, const int32_t* page_table, const int32_t* lengths, int B, int Hq,
                                         int Hkv, int D, int pages, int page_size, int max_pages, float scale,
                                         const uint64_t* turns, float factor, int rot_dim, int interleaved,
                                         dadattn_stream_t stream) {
  const char* name = "paged decode";
  if (int rc = check_paged(name, k_pages, v_pages, page_table, lengths, nullptr, B, Hkv, D, pages, page_size, max_pages)) return rc;
  if (Hq <= 0 || Hq % Hkv) return fail(DADATTN_E_ARG, "%s: Hq=%d must be a multiple of Hkv=%d", name, Hq, Hkv);
  if (!(scale > 0.0f && scale < INFINITY)) return fail(DADATTN_E_ARG, "%s: scale must be positive and finite", name);
  if (int rc = check_rotary(name, turns, factor, rot_dim, D)) return rc;
  if (int rc = check_packed(name, out, out_strides, 8, true, B, Hq)) return rc;
  if (int rc = check_packed(name, q, q_strides, 8, false, B, Hq)) return rc;
  if (int rc = check_packed(name, k_new, k_strides, 8, false, B, Hkv)) return rc;
  if (int rc = check_packed(name, v_new, v_strides, 8, false, B, Hkv)) return rc;
  if (!aligned(lse, 4)) return fail(DADATTN_E_ARG, "%s: lse must be 4-byte aligned", name);
  const int group = Hq / Hkv, parts = (group + kRows - 1) / kRows;
  const long long items = static_cast<long long>(B) * Hkv * parts;
  if (items * kMaxCluster > 0x7fffffffll) return fail(DADATTN_E_UNSUPPORTED, "%s: B=%d and Hkv=%d are too many", name, B, Hkv);
  DecodeParams p = {};
  p.out = reinterpret_cast<bf16*>(out), p.lse = lse;
  p.q = reinterpret_cast<const bf16*>(q);
  p.k_new = reinterpret_cast<const bf16*>(k_new), p.v_new = reinterpret_cast<const bf16*>(v_new);
  p.k_pages = reinterpret_cast<bf16*>(k_pages), p.v_pages = reinterpret_cast<bf16*>(v_pages);
  p.out_token = out_strides[0], p.out_head = out_strides[1], p.q_token = q_strides[0], p.q_head = q_strides[1];
  p.k_token = k_strides[0], p.k_head = k_strides[1], p.v_token = v_strides[0], p.v_head = v_strides[1];
  p.cache = PagedCache{page_table, lengths, nullptr, B, pages, log2_of(page_size), max_pages, Hkv};
  p.heads_q = Hq, p.group = group, p.parts = parts;
  p.scale = scale;
  p.r = RotaryParams{turns, factor, rot_dim, interleaved != 0, 0};
  p.status = device_status_word();
  if (!p.status) return DADATTN_E_CUDA;
  cudaStream_t st = static_cast<cudaStream_t>(stream);
  const bool few = group <= 8;   // rows of an item
  const int n = static_cast<int>(items);
  if (D == 64) return few ? launch_decode<64, 1>(p, n, page_size, st) : launch_decode<64, 2>(p, n, page_size, st);
  return few ? launch_decode<128, 1>(p, n, page_size, st) : launch_decode<128, 2>(p, n, page_size, st);
}
