// Eviction from a bf16 KV cache by accumulated attention weight (decode_window.cu adds the weights up).
//
// Per (sequence, head): of n rows the last `recent` stay and, of the others, the budget - recent with the largest weights
// (equal ones: the lower index; NaN counts as the least). The rows that stay are moved together, in order, with their
// weights, into another cache or within their own.
//
// The CTAs of a cluster share a (sequence, head): K or V, and columns of the rows. Each finds the selection for itself:
//   * the weights become integers of the same order in shared memory, and the smallest kept one is found byte by byte from
//     the top, by histograms of those that agree in the bytes before (four passes, whatever the values);
//   * the rows are gone through 1024 at a time: a prefix sum over "larger than the smallest kept" and "equal to it" gives
//     each kept row its place, and 16-byte pieces of the kept rows are copied.
// Bound by HBM where there are enough (sequence, head) pairs: the weights once, each kept row in and out.
//
// Within one cache: a row's place is never behind the row, so rows that are loaded in order may be stored as soon as every
// thread has loaded its pieces of the same batch; what is stored lies ahead of all that is loaded later. The columns of a
// cluster's CTAs are their own. Weights are read by every CTA of the cluster and moved by one: behind a cluster barrier.
#include <cuda_bf16.h>

#include <algorithm>

#include "common.cuh"
#include "decode_common.cuh"
#include "sm100_ptx.cuh"

namespace dadattn {
namespace {

constexpr int kEvictThreads = 256;
constexpr int kChunk = 4 * kEvictThreads;   // rows of a step
constexpr int kBatch = 4;                   // 16-byte pieces that a thread has in registers
constexpr int kMaxStaged = 49152;           // rows whose weights fit shared memory (192 KB)

struct EvictParams {
  uint16_t *k_dst, *v_dst;
  float* weights_dst;
  int32_t* lengths_dst;
  const uint16_t *k_src, *v_src;
  const float* weights_src;
  const int32_t* lengths_src;
  int* status;
  int H, D, max_len_dst, max_len_src, budget, recent, parts, staged;
  bool in_place;
};

struct EvictShared {
  int histogram[256];
  int warp_total[kEvictThreads / 32];
  int chosen, above;    // a pass's byte, and how many keys are larger
  int list[kChunk];     // rows of the step that stay
};

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

__global__ void __launch_bounds__(kEvictThreads) kv_cache_evict_kernel(const EvictParams p) {
  extern __shared__ __align__(16) uint32_t keys[];   // the weights of a staged call, then nothing
  __shared__ EvictShared sh;
  pdl_wait();
  pdl_launch_dependents();
  const int part = static_cast<int>(blockIdx.x) % p.parts, bh = static_cast<int>(blockIdx.x) / p.parts, b = bh / p.H;
  const int t = threadIdx.x;
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
  auto key = [&](int row) { return p.staged ? keys[row] : key_of(weights[row]); };
  if (p.staged) {
#pragma unroll 4
    for (int row = t; row < candidates; row += kEvictThreads) keys[row] = key_of(weights[row]);
  }

  // The smallest kept key, and how many of the rows that have it stay (the first ones).
  uint32_t least = 0xffffffffu;
  int equal_wanted = 0;
  if (wanted > 0) {
    uint32_t prefix = 0;
    int left = wanted;
    for (int shift = 24; shift >= 0; shift -= 8) {
      sh.histogram[t] = 0;
      __syncthreads();
#pragma unroll 4
      for (int row = t; row < candidates; row += kEvictThreads) {
        const uint32_t k = key(row);
        // (shift + 8 = 32 in the first pass: every key counts)
        if (shift == 24 || (k >> (shift + 8)) == prefix) atomicAdd(&sh.histogram[(k >> shift) & 255u], 1);
      }
      __syncthreads();
      // thread t has byte 255 - t: the sums before it are of the larger bytes
      const int mine = sh.histogram[255 - t];
      int total;
      const int above = prefix_sum(sh, mine, total);
      if (above < left && left <= above + mine) {
        sh.chosen = 255 - t;
        sh.above = above;
      }
      __syncthreads();
      prefix = prefix << 8 | static_cast<uint32_t>(sh.chosen);
      left -= sh.above;
    }
    least = prefix;
    equal_wanted = left;
  }
  if (p.parts > 1 && p.in_place) {   // (only staged calls come here: every CTA has its copy of the weights)
    __syncthreads();
    cluster_arrive();
    cluster_wait();
  }

  const bool both = p.parts == 1;
  const int slices = both ? 1 : p.parts / 2, pieces = p.D / 8 / slices;   // 16-byte pieces of a row that are this CTA's
  const int shift = 31 - __clz(pieces), column = (both ? 0 : part / 2) * pieces;
  const int row_pieces = p.D / 8;
  int larger = 0, equal = 0;   // rows before the step that are larger than the least, and that are equal to it
  int done = 0;                // rows kept before the step
  for (int row0 = 0; row0 < n; row0 += kChunk) {
    // a thread's four rows: bit i of `gt`, `eq`
    int gt = 0, eq = 0;
    float w[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const int row = row0 + 4 * t + i;
      w[i] = 0.f;
      if (row < n) {
        if (part == 0) w[i] = weights[row];
        if (row >= candidates) {
          gt |= 1 << i;
        } else if (wanted > 0) {
          const uint32_t k = key(row);
          if (k > least) gt |= 1 << i;
          else if (k == least) eq |= 1 << i;
        }
      }
    }
    int total;
    const int before = prefix_sum(sh, __popc(gt) | __popc(eq) << 16, total);
    int g = larger + (before & 0xffff), e = equal + (before >> 16);
    const int first = done;
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const bool is_gt = gt >> i & 1, is_eq = eq >> i & 1;
      const int place = g + min(e, equal_wanted);
      if (is_gt || (is_eq && e < equal_wanted)) {
        sh.list[place - first] = row0 + 4 * t + i;
        // (every thread has read its weights of this step, and what is stored lies ahead of the steps to come)
        if (part == 0) p.weights_dst[static_cast<size_t>(bh) * p.max_len_dst + place] = w[i];
      }
      g += is_gt;
      e += is_eq;
    }
    larger += total & 0xffff;
    equal += total >> 16;
    done = larger + min(equal, equal_wanted);
    __syncthreads();
    const int count = (done - first) << shift;
    for (int side = both ? 0 : part % 2; side < (both ? 2 : part % 2 + 1); ++side) {
      const uint4* src = reinterpret_cast<const uint4*>(side ? p.v_src : p.k_src) + static_cast<size_t>(bh) * p.max_len_src * row_pieces + column;
      uint4* dst = reinterpret_cast<uint4*>(side ? p.v_dst : p.k_dst) + (static_cast<size_t>(bh) * p.max_len_dst + first) * row_pieces + column;
      for (int i0 = 0; i0 < count; i0 += kBatch * kEvictThreads) {
        uint4 x[kBatch];
#pragma unroll
        for (int i = 0; i < kBatch; ++i) {
          const int at = i0 + i * kEvictThreads + t;
          if (at < count) x[i] = src[static_cast<size_t>(sh.list[at >> shift]) * row_pieces + (at & (pieces - 1))];
        }
        if (p.in_place) __syncthreads();
#pragma unroll
        for (int i = 0; i < kBatch; ++i) {
          const int at = i0 + i * kEvictThreads + t;
          if (at < count) dst[static_cast<size_t>(at >> shift) * row_pieces + (at & (pieces - 1))] = x[i];
        }
      }
    }
    __syncthreads();   // the list is read
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
  if (max_len_dst > DADATTN_MAX_CACHE_LEN || max_len_src > DADATTN_MAX_CACHE_LEN)
    return fail(DADATTN_E_UNSUPPORTED, "cache eviction: max_len may not exceed %d", DADATTN_MAX_CACHE_LEN);
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
                   H, D, max_len_dst, max_len_src, budget, recent, 1, max_len_src <= kMaxStaged, in_place};
  if (!p.status) return DADATTN_E_CUDA;
  while (p.parts < 8 && static_cast<long long>(pairs) * p.parts * 2 <= 8LL * sms) p.parts *= 2;
  if (in_place && !p.staged) p.parts = 1;   // the weights are read all along, by the CTA that moves them
  cudaStream_t st = static_cast<cudaStream_t>(stream);
  const size_t smem = p.staged ? static_cast<size_t>(max_len_src) * 4 : 0;
  DAD_CUDA(cudaFuncSetAttribute(kv_cache_evict_kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, kMaxStaged * 4));
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
  DAD_CUDA(cudaLaunchKernelEx(&cfg, kv_cache_evict_kernel, p));
  if (in_place)
    DAD_CUDA(launch_pdl(evict_lengths_kernel, dim3((B + 255) / 256), dim3(256), 0, st, lengths_dst, B, max_len_src, budget));
  return DADATTN_OK;
}
