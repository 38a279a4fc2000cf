// Eviction from a bf16 KV cache by accumulated attention weight (decode_window.cu adds the weights up).
//
// Per (sequence, head): of n rows the last `recent` stay and, of the others, the budget - recent with the largest weights
// (equal ones: the lower index; NaN counts as the least). The rows that stay are moved together, in order, with their
// weights, into another cache or within their own.
//
// A CTA has a (sequence, head), or the CTAs of a cluster share it where there are few:
//   * each turns the weights of its part of the rows into integers of the same order in shared memory; the smallest kept one is
//     found byte by byte from the top, by histograms of those that agree in the bytes before, which the cluster adds up. Four
//     passes at most: the search ends where all that agree so far stay. After the second the rows that stay for certain are
//     asked for in L2.
//   * each counts and numbers the rows of its part that are larger than the smallest kept, and the first ones that are equal
//     to it, and writes them into the list of the CTA that will copy them;
//   * the rows of the list are copied in 16-byte pieces: into another cache by shares of the list, within one cache by columns
//     (there every CTA of the cluster has the whole list).
// Bound by HBM where there are enough (sequence, head) pairs: the weights once, each kept row in and out. Where all heads are as
// long as they can be, the selections of all CTAs come first and the copies after them: 64 x 12 heads of 64, 1024 rows to 512,
// take 45.6 us, 9 of them selection, and 38.5 where nothing is to be selected (203 MB: 5.3 TB/s). 4 x 24 heads of 128, 8000 rows to 2048:
// 52.4 us, 38.8 with nothing to select. (There each CTA selecting for itself, and copying as it went through the rows 1024 at a
// time, took 87; all four passes 61.7; every list written by all CTAs 57; two waves of clusters of two for 64 x 12 heads 55.
// Adding up equal bytes of a warp by votes before the shared atomics cost 1 to 3 us.)
//
// Within one cache it is about as fast where CTAs have a (sequence, head) each, 64 x 12 heads of 64, 1024 rows to 512: 48.0 us,
// of 9 .. 1017 rows 26.7 (33.6 into another: short sequences stay as they are), and slower for clusters, whose CTAs copy a few
// pieces of every row each, batch by batch: 4 x 24 heads of 128, 8000 rows to 2048 63.4, 2056 to 2048 66.7 (into another 52.9
// and 47.9). The second launch, for the lengths, is in these.
//
// Within one cache: a row's place is never behind the row, so rows that are loaded in order may be stored as soon as every
// thread has loaded its pieces of the same batch; what is stored lies ahead of all that is loaded later. The columns of a
// cluster's CTAs are their own, and the weights, which one of them moves, were read by all behind a cluster barrier.
#include <cuda_bf16.h>

#include <algorithm>

#include "common.cuh"
#include "decode_common.cuh"
#include "sm100_ptx.cuh"

namespace dadattn {
namespace {

constexpr int kEvictThreads = 256;
// 16-byte pieces that a thread has in registers, and CTAs that an SM holds. Clusters: six on an SM (40 registers, 64 bytes
// spilt), so that their waits for each other are covered. One CTA for each pair: 64 x 12 heads of 1 .. 1024 rows to 512 take 32.4 us with four
// that have 8 pieces in flight (all of 1024 rows: 45.6), 35.2 with six of 4 (45.6), 34.7 with five of 4 (57.1: a second wave).
constexpr int kClusterBatch = 4, kClusterPerSm = 6;
constexpr int kSingleBatch = 8, kSinglePerSm = 4;
constexpr int kMaxParts = 8;                // CTAs of a cluster
constexpr int kMaxStaged = 24576;           // rows whose weights a CTA has in shared memory (96 KB),
constexpr int kMaxListed = 24576;           // and kept rows that it has at a time

struct EvictParams {
  uint16_t *k_dst, *v_dst;
  float* weights_dst;
  int32_t* lengths_dst;
  const uint16_t *k_src, *v_src;
  const float* weights_src;
  const int32_t* lengths_src;
  int* status;
  int H, D, max_len_dst, max_len_src, budget, recent, parts, listed;
  bool in_place;
};

struct EvictShared {
  int histogram[2][256];   // of this CTA's rows; passes take turns
  int counts[kMaxParts];   // of every CTA: rows larger than the smallest kept, and equal to it
  int equals[kMaxParts];
  int warp_total[kEvictThreads / 32];
  int chosen, above, of_chosen;   // a pass's byte, how many keys are larger, and how many have it
};

__device__ __forceinline__ void st_cluster_int(uint32_t addr, int v) {
  asm volatile("st.shared::cluster.s32 [%0], %1;" ::"r"(addr), "r"(v) : "memory");
}
__device__ __forceinline__ int ld_cluster_int(uint32_t addr) {
  int v;
  asm volatile("ld.shared::cluster.s32 %0, [%1];" : "=r"(v) : "r"(addr) : "memory");
  return v;
}
// All CTAs of the cluster
__device__ __forceinline__ void meet(int parts) {
  if (parts == 1) {
    __syncthreads();
  } else {
    cluster_arrive();
    cluster_wait();
  }
}

// An integer of the same order; zeros of either sign are equal, NaN is the least.
__device__ __forceinline__ uint32_t key_of(float w) {
  if (!(w == w)) return 0u;
  const uint32_t u = __float_as_uint(w + 0.f);   // -0 + 0 = 0
  return (u & 0x80000000u) ? ~u : u | 0x80000000u;
}

// Sums of the threads before this one, and the total, by the whole CTA (two barriers).
__device__ __forceinline__ int prefix_sum(EvictShared& sh, int mine, int& total) {
  const int lane = threadIdx.x % 32, warp = threadIdx.x / 32;
  int sum = mine;
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const int below = __shfl_up_sync(0xffffffffu, sum, o);
    if (lane >= o) sum += below;
  }
  if (lane == 31) sh.warp_total[warp] = sum;
  __syncthreads();
  int before = 0;
  total = 0;
#pragma unroll
  for (int w = 0; w < kEvictThreads / 32; ++w) {
    const int t = sh.warp_total[w];
    if (w < warp) before += t;
    total += t;
  }
  __syncthreads();
  return before + sum - mine;
}

template <bool CLUSTER>
__global__ void __launch_bounds__(kEvictThreads, CLUSTER ? kClusterPerSm : kSinglePerSm) kv_cache_evict_kernel(const __grid_constant__ EvictParams p) {
  extern __shared__ __align__(16) int dynamic[];   // the list, then the keys of this CTA's rows
  int* list = dynamic;
  uint32_t* keys = reinterpret_cast<uint32_t*>(dynamic + p.listed);
  __shared__ EvictShared sh;
  constexpr int kBatch = CLUSTER ? kClusterBatch : kSingleBatch;
  const int parts = CLUSTER ? p.parts : 1, part = static_cast<int>(blockIdx.x) % parts, bh = static_cast<int>(blockIdx.x) / parts, b = bh / p.H;
  const int t = threadIdx.x, D = p.D;
  sh.histogram[0][t] = 0;
  sh.histogram[1][t] = 0;
  pdl_wait();
  pdl_launch_dependents();
  const int n = p.lengths_src[b];
  // (the same for all CTAs of a cluster, who leave together)
  if (n < 0 || n > p.max_len_src) {
    if (bh % p.H == 0 && part == 0 && t == 0) atomicExch(p.status, DADATTN_E_ARG);
    return;
  }
  const int kept = min(n, p.budget);
  if (!p.in_place && bh % p.H == 0 && part == 0 && t == 0) p.lengths_dst[b] = kept;
  if (n == 0 || (p.in_place && n <= p.budget)) return;
  const float* weights = p.weights_src + static_cast<size_t>(bh) * p.max_len_src;
  const bool all = n <= p.budget;
  const int candidates = all ? 0 : n - p.recent;   // rows that are chosen from; those behind stay
  const int wanted = all ? 0 : p.budget - p.recent;
  // this CTA's rows, and those of them that are chosen from
  const int share = (n + parts - 1) / parts, row0 = min(part * share, n), row1 = min(row0 + share, n), end = min(row1, candidates);
#pragma unroll 4
  for (int row = row0 + t; row < end; row += kEvictThreads) keys[row - row0] = key_of(weights[row]);

  // The smallest kept key, and how many of the rows that have it stay (the first ones).
  uint32_t least = 0xffffffffu;
  int equal_wanted = 0;
  if (wanted > 0) {
    uint32_t prefix = 0;
    int left = wanted;
    for (int shift = 24, turn = 0; shift >= 0; shift -= 8, turn ^= 1) {
      __syncthreads();   // (the keys, and the cleared histogram)
      int* histogram = sh.histogram[turn];
#pragma unroll 4
      for (int row = t; row < end - row0; row += kEvictThreads) {
        const uint32_t k = keys[row];
        // (shift + 8 = 32 in the first pass: every key counts)
        if (shift == 24 || (k >> (shift + 8)) == prefix) atomicAdd(&histogram[(k >> shift) & 255u], 1);
      }
      meet(parts);
      // thread t has byte 255 - t of all CTAs: the sums before it are of the larger bytes
      int mine = 0;
      if (parts == 1) {
        mine = histogram[255 - t];
      } else {
        int of[kMaxParts];   // (all on their way together)
#pragma unroll
        for (int i = 0; i < kMaxParts; ++i)
          if (i < parts) of[i] = ld_cluster_int(cluster_address(&histogram[255 - t], i));
#pragma unroll
        for (int i = 0; i < kMaxParts; ++i)
          if (i < parts) mine += of[i];
      }
      sh.histogram[turn ^ 1][t] = 0;   // (everybody is past the pass before)
      int total;
      const int above = prefix_sum(sh, mine, total);
      if (above < left && left <= above + mine) {
        sh.chosen = 255 - t;
        sh.above = above;
        sh.of_chosen = mine;
      }
      __syncthreads();
      prefix = prefix << 8 | static_cast<uint32_t>(sh.chosen);
      left -= sh.above;
      least = prefix;
      if (sh.of_chosen == left && prefix > 0) {   // all that agree stay
        least = (prefix << shift) - 1;
        left = 0;
        break;
      }
      if (shift == 16) {   // rows that stay for certain: on their way while the rest is found
        for (int row = t; row < end - row0; row += kEvictThreads)
          if ((keys[row] >> 16) > prefix) {
            const size_t at = (static_cast<size_t>(bh) * p.max_len_src + row0 + row) * D;
            for (int i = 0; i < D; i += 64) {   // 128 bytes
              asm volatile("prefetch.global.L2 [%0];" ::"l"(p.k_src + at + i));
              asm volatile("prefetch.global.L2 [%0];" ::"l"(p.v_src + at + i));
            }
          }
      }
    }
    equal_wanted = left;
  }
  auto is_larger = [&](int row) { return row >= candidates || (wanted > 0 && keys[row - row0] > least); };
  auto is_equal = [&](int row) { return row < candidates && wanted > 0 && keys[row - row0] == least; };

  // How many rows of the CTAs before this one stay
  int larger = 0, equal = 0;
  if (CLUSTER && !all) {   // (a part has no more than kMaxStaged < 2^16 rows)
    int counted = 0, total;
    for (int row = row0 + t; row < row1; row += kEvictThreads) {
      if (is_larger(row)) ++counted;
      else if (is_equal(row)) counted += 1 << 16;
    }
    prefix_sum(sh, counted, total);
    if (wanted == 0) meet(parts);   // (no pass has met yet: a CTA has to run before another one stores to it)
    if (t < parts) {
      st_cluster_int(cluster_address(&sh.counts[part], t), total & 0xffff);
      st_cluster_int(cluster_address(&sh.equals[part], t), total >> 16);
    }
    meet(parts);   // (and every CTA has read its weights: one of them may move them now)
    for (int i = 0; i < part; ++i) larger += sh.counts[i], equal += sh.equals[i];
  }

  const int row_pieces = D / 8;   // 16-byte pieces of a row
  const size_t src0 = static_cast<size_t>(bh) * p.max_len_src, dst0 = static_cast<size_t>(bh) * p.max_len_dst;
  const bool by_rows = !p.in_place, with_list = !all && !CLUSTER;   // weights that move as their rows are listed
  for (int begin = 0; begin < kept; begin += p.listed) {   // (one turn, unless the budget is larger than the list)
    const int count = min(kept - begin, p.listed), chunk = (count + parts - 1) / parts;
    // another cache: a share of the rows; the same: a share of the columns, of K or of V where the cluster is large enough
    const int first = by_rows ? min(part * chunk, count) : 0, last = by_rows ? min(first + chunk, count) : count;
    if (all) {
      for (int i = first + t; i < last; i += kEvictThreads) list[i] = begin + i;
      __syncthreads();
    }
    // Numbers of this CTA's kept rows: a thread has four rows in turn of 1024
    int before_gt = larger, before_eq = equal;
    for (int r0 = row0; !all && r0 < row1; r0 += 4 * kEvictThreads) {
      int gt = 0, eq = 0;
      float w[4];
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const int row = r0 + 4 * t + i;
        if (row < row1) {
          if (with_list) w[i] = weights[row];
          if (is_larger(row)) gt |= 1 << i;
          else if (is_equal(row)) eq |= 1 << i;
        }
      }
      int total;
      const int before = prefix_sum(sh, __popc(gt) | __popc(eq) << 16, total);
      int g = before_gt + (before & 0xffff), e = before_eq + (before >> 16);
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const bool is_gt = gt >> i & 1, is_eq = eq >> i & 1;
        const int place = g + min(e, equal_wanted) - begin;
        if ((is_gt || (is_eq && e < equal_wanted)) && place >= 0 && place < count) {
          if (with_list) p.weights_dst[dst0 + begin + place] = w[i];
          if (!CLUSTER) {
            list[place] = r0 + 4 * t + i;
          } else {
            const int owner = by_rows ? place / chunk : 0;
            for (int j = owner; j < (by_rows ? owner + 1 : parts); ++j) st_cluster_int(cluster_address(&list[place], j), r0 + 4 * t + i);
          }
        }
        g += is_gt;
        e += is_eq;
      }
      before_gt += total & 0xffff;
      before_eq += total >> 16;
    }
    if (!all) meet(parts);   // the list is there

    const int sides = by_rows || parts == 1 ? 2 : 1, slices = by_rows || parts == 1 ? 1 : parts / 2;
    const int pieces = row_pieces / slices, shift = 31 - __clz(pieces);
    const int column = by_rows || parts == 1 ? 0 : part / 2 * pieces;
    const int work = (last - first) << shift;
    for (int i = 0; i < sides; ++i) {
      const bool is_v = sides == 2 ? i : part % 2;
      const uint4* src = reinterpret_cast<const uint4*>(is_v ? p.v_src : p.k_src) + src0 * row_pieces + column;
      uint4* dst = reinterpret_cast<uint4*>(is_v ? p.v_dst : p.k_dst) + (dst0 + begin + first) * row_pieces + column;
      for (int i0 = 0; i0 < work; i0 += kBatch * kEvictThreads) {
        uint4 x[kBatch];
#pragma unroll
        for (int j = 0; j < kBatch; ++j) {
          const int at = i0 + j * kEvictThreads + t;
          if (at < work) x[j] = src[static_cast<size_t>(list[first + (at >> shift)]) * row_pieces + (at & (pieces - 1))];
        }
        if (p.in_place) __syncthreads();
#pragma unroll
        for (int j = 0; j < kBatch; ++j) {
          const int at = i0 + j * kEvictThreads + t;
          if (at < work) dst[static_cast<size_t>(at >> shift) * row_pieces + (at & (pieces - 1))] = x[j];
        }
      }
    }
    if (!with_list && (by_rows || part == 0)) {
      for (int i0 = first; i0 < last; i0 += kBatch * kEvictThreads) {
        float x[kBatch];
#pragma unroll
        for (int j = 0; j < kBatch; ++j) {
          const int at = i0 + j * kEvictThreads + t;
          if (at < last) x[j] = weights[list[at]];
        }
        if (p.in_place) __syncthreads();
#pragma unroll
        for (int j = 0; j < kBatch; ++j) {
          const int at = i0 + j * kEvictThreads + t;
          if (at < last) p.weights_dst[dst0 + begin + at] = x[j];
        }
      }
    }
    if (begin + p.listed < kept) meet(parts);   // the list is read
  }
}

// Within one cache the lengths change once nobody reads them any more.
__global__ void evict_lengths_kernel(int32_t* lengths, int B, int max_len, int budget) {
  pdl_wait();
  pdl_launch_dependents();
  const int b = blockIdx.x * blockDim.x + threadIdx.x;
  if (b < B && lengths[b] > budget && lengths[b] <= max_len) lengths[b] = budget;
}

// Whether two arrays share memory without being the same.
bool overlap(const void* a, size_t a_bytes, const void* b, size_t b_bytes) {
  const uintptr_t x = reinterpret_cast<uintptr_t>(a), y = reinterpret_cast<uintptr_t>(b);
  return x < y + b_bytes && y < x + a_bytes;
}

}  // namespace
}  // namespace dadattn

using namespace dadattn;

extern "C" int dadattn_kv_cache_evict_bf16(uint16_t* k_dst, uint16_t* v_dst, float* weights_dst, int32_t* lengths_dst,
                                           const uint16_t* k_src, const uint16_t* v_src, const float* weights_src,
                                           const int32_t* lengths_src, int B, int H, int D, int max_len_dst, int max_len_src,
                                           int budget, int recent, dadattn_stream_t stream) {
  const void* const dst[4] = {k_dst, v_dst, weights_dst, lengths_dst};
  const void* const src[4] = {k_src, v_src, weights_src, lengths_src};
  for (int i = 0; i < 4; ++i)
    if (!dst[i] || !src[i]) return fail(DADATTN_E_ARG, "cache eviction: null pointer");
  if (B <= 0 || H <= 0 || max_len_dst <= 0 || max_len_src <= 0 || static_cast<long long>(B) * H > 0x7fffffffLL / 8)
    return fail(DADATTN_E_ARG, "cache eviction: bad sizes B=%d H=%d max_len %d and %d", B, H, max_len_dst, max_len_src);
  if (max_len_dst > DADATTN_MAX_CACHE_LEN || max_len_src > kMaxParts * kMaxStaged)
    return fail(DADATTN_E_UNSUPPORTED, "cache eviction: max_len of the source may not exceed %d", kMaxParts * kMaxStaged);
  if (D != 64 && D != 128) return fail(DADATTN_E_UNSUPPORTED, "cache eviction: unsupported D %d", D);
  if (budget < 1 || budget > max_len_dst || recent < 0 || recent > budget)
    return fail(DADATTN_E_ARG, "cache eviction: budget %d must be in [1, %d], recent %d in [0, budget]", budget, max_len_dst, recent);
  for (int i = 0; i < 4; ++i)
    if (!aligned(dst[i], i < 2 ? 16 : 4) || !aligned(src[i], i < 2 ? 16 : 4))
      return fail(DADATTN_E_ARG, "cache eviction: caches must be 16-byte aligned, weights and lengths 4-byte");
  // one cache for all four arrays, or another place for each
  const size_t pairs = static_cast<size_t>(B) * H;
  const size_t dst_bytes[4] = {pairs * max_len_dst * D * 2, pairs * max_len_dst * D * 2, pairs * max_len_dst * 4, static_cast<size_t>(B) * 4};
  const size_t src_bytes[4] = {pairs * max_len_src * D * 2, pairs * max_len_src * D * 2, pairs * max_len_src * 4, static_cast<size_t>(B) * 4};
  const bool in_place = k_dst == k_src;
  for (int i = 0; i < 4; ++i) {
    if (in_place && (dst[i] != src[i] || max_len_dst != max_len_src))
      return fail(DADATTN_E_ARG, "cache eviction: within one cache all arrays and max_len are the same");
    for (int j = 0; j < 4; ++j) {
      if (!(in_place && i == j) && overlap(dst[i], dst_bytes[i], src[j], src_bytes[j]))
        return fail(DADATTN_E_ARG, "cache eviction: arrays overlap");
      if (i != j && overlap(dst[i], dst_bytes[i], dst[j], dst_bytes[j]))
        return fail(DADATTN_E_ARG, "cache eviction: arrays overlap");
    }
  }
  int dev = 0, sms = 0;
  DAD_CUDA(cudaGetDevice(&dev));
  DAD_CUDA(cudaDeviceGetAttribute(&sms, cudaDevAttrMultiProcessorCount, dev));
  EvictParams p = {k_dst, v_dst, weights_dst, lengths_dst, k_src, v_src, weights_src, lengths_src, device_status_word(),
                   H, D, max_len_dst, max_len_src, budget, recent, 1, std::min(std::min(budget, max_len_src), kMaxListed), in_place};
  if (!p.status) return DADATTN_E_CUDA;
  // CTAs for each pair: as many as fit the GPU at once, and as the weights need room
  while (p.parts < kMaxParts && (static_cast<long long>(pairs) * p.parts * 2 <= static_cast<long long>(kClusterPerSm) * sms || max_len_src > p.parts * kMaxStaged)) p.parts *= 2;
  cudaStream_t st = static_cast<cudaStream_t>(stream);
  const size_t smem = sizeof(int) * (p.listed + static_cast<size_t>(max_len_src + p.parts - 1) / p.parts);
  auto kern = p.parts > 1 ? kv_cache_evict_kernel<true> : kv_cache_evict_kernel<false>;
  DAD_CUDA(cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, (kMaxListed + kMaxStaged) * 4));
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3(static_cast<unsigned>(pairs * p.parts));
  cfg.blockDim = dim3(kEvictThreads);
  cfg.dynamicSmemBytes = smem;
  cfg.stream = st;
  cudaLaunchAttribute attrs[2];
  attrs[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attrs[0].val.programmaticStreamSerializationAllowed = 1;
  attrs[1].id = cudaLaunchAttributeClusterDimension;
  attrs[1].val.clusterDim = {static_cast<unsigned>(p.parts), 1, 1};
  cfg.attrs = attrs;
  cfg.numAttrs = p.parts > 1 ? 2 : 1;
  DAD_CUDA(cudaLaunchKernelEx(&cfg, kern, p));
  if (in_place)
    DAD_CUDA(launch_pdl(evict_lengths_kernel, dim3((B + 255) / 256), dim3(256), 0, st, lengths_dst, B, max_len_src, budget));
  return DADATTN_OK;
}
