// What the decode kernels (decode.cu, decode_window.cu) share: elements, bulk copies, cluster stores, the order in
// which sequences are taken up, and the tickets that say when every CTA has read the lengths.
#pragma once

#include <cuda_bf16.h>

#include <climits>

#include "common.cuh"
#include "sm100_ptx.cuh"

namespace dadattn {
namespace {

constexpr unsigned kTicketGroups = 32;  // first-level counters of the "all lengths read" tickets
constexpr int kMaxRanked = 256;     // sequences whose lengths a CTA copies and can rank

// A 16-byte piece of a row as float pairs, and the softmax's exponential. Scores are kept in units
// that exp_of() takes: natural units and expf for fp32 caches, log2 units and ex2 for bf16 ones
// (whose 2^-9 rounding of the inputs is far above the difference).
template <typename T>
struct Elem;
template <>
struct Elem<float> {
  static constexpr int kPerLane = 4;
  static constexpr float kUnit = 1.0f;
  __device__ static void unpack(float2 (&f)[2], const uint4& raw) {
    f[0] = make_float2(__uint_as_float(raw.x), __uint_as_float(raw.y));
    f[1] = make_float2(__uint_as_float(raw.z), __uint_as_float(raw.w));
  }
  __device__ static float exp_of(float x) { return expf(x); }
  __device__ static float from_float(float x) { return x; }
};
template <>
struct Elem<__nv_bfloat16> {
  static constexpr int kPerLane = 8;
  static constexpr float kUnit = 1.4426950408889634f;
  __device__ static void unpack(float2 (&f)[4], const uint4& raw) {
    const uint32_t w[4] = {raw.x, raw.y, raw.z, raw.w};
#pragma unroll
    for (int i = 0; i < 4; ++i) f[i] = make_float2(__uint_as_float(w[i] << 16), __uint_as_float(w[i] & 0xffff0000u));
  }
  __device__ static float exp_of(float x) { return ptx::ex2(x); }
  __device__ static __nv_bfloat16 from_float(float x) { return __float2bfloat16_rn(x); }
};

__device__ __forceinline__ void bulk_load(void* smem_dst, const void* src, uint32_t bytes, uint64_t* bar) {
  asm volatile("cp.async.bulk.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1], %2, [%3];" ::"r"(
                   ptx::smem_u32(smem_dst)),
               "l"(src), "r"(bytes), "r"(ptx::smem_u32(bar))
               : "memory");
}
__device__ __forceinline__ void cluster_arrive() { asm volatile("barrier.cluster.arrive.release;" ::: "memory"); }
__device__ __forceinline__ void cluster_wait() { asm volatile("barrier.cluster.wait.acquire;" ::: "memory"); }
// stores to the same shared-memory variable of another CTA of the cluster
__device__ __forceinline__ uint32_t cluster_address(const void* own, int cta) {
  uint32_t a;
  asm volatile("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(a) : "r"(ptx::smem_u32(own)), "r"(cta));
  return a;
}
__device__ __forceinline__ void st_cluster(uint32_t addr, float v) {
  asm volatile("st.shared::cluster.f32 [%0], %1;" ::"r"(addr), "f"(v) : "memory");
}

// order[r] = the sequence of rank r, by a whole CTA of `threads` threads (128 of them share out the comparisons).
// Ahead of the call and a __syncthreads: lens[0..kMaxRanked) holds the lengths and INT_MIN behind the last of them,
// place[] zeros; 32 <= B <= kMaxRanked.
__device__ __forceinline__ void rank_by_length(const int* lens, int* place, int* order, int B, int threads) {
  // rank(s) = number of sequences that come before s (longer, or as long with a smaller index);
  // with the count padded to a power of two n_pad (32..256; padding is INT_MIN and comes last),
  // 128 threads share out the n_pad^2 comparisons.
  const int t = threadIdx.x;
  if (t < 128) {
    const int lg = 32 - __clz(B - 1);   // n_pad = 1 << lg, 5 <= lg <= 8
    const int n_pad = 1 << lg;
    const int groups = lg < 7 ? 128 >> lg : 1;
    const int per = n_pad / groups, g = (t >> lg) & (groups - 1);
    for (int si = t & (n_pad - 1); si < n_pad; si += 128) {
      const int mine = lens[si];
      int count = 0;
#pragma unroll 4
      for (int j = g * per; j < (g + 1) * per; j += 4) {
        const int4 o = *reinterpret_cast<const int4*>(lens + j);   // broadcast reads
        count += static_cast<int>(o.x > mine) | (static_cast<int>(o.x == mine) & static_cast<int>(j + 0 < si));
        count += static_cast<int>(o.y > mine) | (static_cast<int>(o.y == mine) & static_cast<int>(j + 1 < si));
        count += static_cast<int>(o.z > mine) | (static_cast<int>(o.z == mine) & static_cast<int>(j + 2 < si));
        count += static_cast<int>(o.w > mine) | (static_cast<int>(o.w == mine) & static_cast<int>(j + 3 < si));
      }
      if (count) atomicAdd(&place[si], count);
    }
  }
  __syncthreads();
  for (int i = t; i < B; i += threads) order[place[i]] = i;
  __syncthreads();
}

// Every CTA of the call draws a ticket once it has read the lengths; whoever holds the last one
// knows that nobody will read them again and advances them. Two levels keep the atomics off one
// address: the CTAs are dealt into kTicketGroups groups; the last of each group draws from a
// second counter, and the last of those advances.
struct LengthTickets {
  unsigned* counters;   // 1 + kTicketGroups, zero between calls
  __device__ __forceinline__ unsigned draw() const { return atomicAdd(&counters[1 + blockIdx.x % kTicketGroups], 1u); }
  __device__ __forceinline__ bool is_last(unsigned ticket) const {
    const unsigned group = blockIdx.x % kTicketGroups;
    const unsigned all_ctas = gridDim.x;
    if (ticket != (all_ctas - group + kTicketGroups - 1) / kTicketGroups - 1) return false;
    counters[1 + group] = 0;   // ready for the next call
    const unsigned groups = all_ctas < kTicketGroups ? all_ctas : kTicketGroups;
    if (atomicAdd(&counters[0], 1u) != groups - 1) return false;
    counters[0] = 0;
    return true;
  }
};

}  // namespace
}  // namespace dadattn
