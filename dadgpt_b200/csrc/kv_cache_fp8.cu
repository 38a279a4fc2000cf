// Prompts into an 8-bit KV cache: K and V heads as a prefill leaves them -> blocks of 64 tokens with a scale each, and the
// rows behind the last whole block, as bf16, into the tail buffer (fp8_block.cuh has the format).
//
// One pass: a CTA has one block (64 x D elements) in registers, finds its largest element, and writes the codes. Bound by
// HBM: 2 or 4 bytes in and 1 out per element. 64 x 12 heads of 1024 x 64: bf16 45.8 us = 6.6 TB/s, fp32 73.6 us = 6.8 TB/s;
// of lengths 1 .. 1024 26.5 us = 5.9 TB/s, where half of the CTAs find nothing to do. (Every element's exponent looked at by
// itself, for infinities, took 58.1 us: bound by instruction issue.)
#include <cuda_bf16.h>

#include "common.cuh"
#include "fp8_block.cuh"
#include "sm100_ptx.cuh"

namespace dadattn {
namespace {

constexpr int kFillThreads = 128;

struct FillParams {
  const void *k_heads, *v_heads;   // [B, H, S, D]
  uint8_t *k, *v;                  // [B, H, max_len, D]
  float *k_scale, *v_scale;        // [B, H, blocks]
  uint16_t *k_tail, *v_tail;       // [B, H, 64, D]
  int32_t* lengths;
  const int32_t* counts;           // null: S rows of every sequence
  int* status;
  int H, S, max_len, blocks;
};

// Eight consecutive elements as bf16.
template <bool BF16>
__device__ __forceinline__ uint4 load_eight(const void* heads, size_t at) {
  if (BF16) return __ldg(reinterpret_cast<const uint4*>(static_cast<const uint16_t*>(heads) + at));
  const float4* f = reinterpret_cast<const float4*>(static_cast<const float*>(heads) + at);
  const float4 a = __ldg(f), b = __ldg(f + 1);
  return make_uint4(ptx::pack_bf16(a.x, a.y), ptx::pack_bf16(a.z, a.w), ptx::pack_bf16(b.x, b.y), ptx::pack_bf16(b.z, b.w));
}

// Block x of (sequence, head) z, of K or V (y) or of both; the last x of a sequence is its open block. Both for bf16: half as
// many CTAs, as long as their registers (48 at head size 64, 80 at 128) leave the SM as many bytes on their way: the two cases
// above 46.4 -> 45.8 and 28.4 -> 26.5 us. One from fp32, whose elements take twice the registers ahead of the conversion: 77.3
// against 73.6, and 50.7 against 44.1 for 16 x 24 heads of 128, of lengths 1 .. 1024.
template <bool BF16>
constexpr int kSides = BF16 ? 2 : 1;
template <bool BF16, int D>
__global__ void __launch_bounds__(kFillThreads) kv_cache_fill_fp8_kernel(const FillParams p) {
  constexpr int kPieces = kFp8Block * D / 8 / kFillThreads;   // of eight elements, per thread and side
  constexpr int kPerRow = D / 8, kWarps = kFillThreads / 32, N = kSides<BF16>;
  __shared__ float warp_most[N][kWarps];
  pdl_wait();
  pdl_launch_dependents();
  const int block = blockIdx.x, bh = blockIdx.z, b = bh / p.H, t = threadIdx.x;
  auto is_v = [&](int side) { return N == 2 ? side == 1 : blockIdx.y == 1; };
  const int n = p.counts ? p.counts[b] : p.S;
  if (block == 0 && blockIdx.y == 0 && bh % p.H == 0 && t == 0) {
    if (n >= 0 && n <= p.S && n <= p.max_len) p.lengths[b] = n;
    else atomicExch(p.status, DADATTN_E_ARG);
  }
  if (n < 0 || n > p.S || n > p.max_len) return;   // left alone and reported
  const int row0 = block * kFp8Block, rows = min(n - row0, kFp8Block);
  if (rows <= 0) return;
  const size_t from = (static_cast<size_t>(bh) * p.S + row0) * D;
  uint4 raw[N][kPieces];
#pragma unroll
  for (int side = 0; side < N; ++side)
#pragma unroll
    for (int i = 0; i < kPieces; ++i) {
      const int piece = i * kFillThreads + t;
      raw[side][i] = piece / kPerRow < rows ? load_eight<BF16>(is_v(side) ? p.v_heads : p.k_heads, from + static_cast<size_t>(piece) * 8)
                                            : make_uint4(0, 0, 0, 0);
    }
  if (rows < kFp8Block) {
#pragma unroll
    for (int side = 0; side < N; ++side) {
      uint4* tail = reinterpret_cast<uint4*>((is_v(side) ? p.v_tail : p.k_tail) + static_cast<size_t>(bh) * kFp8Block * D);
#pragma unroll
      for (int i = 0; i < kPieces; ++i) {
        const int piece = i * kFillThreads + t;
        if (piece / kPerRow < rows) tail[piece] = raw[side][i];
      }
    }
    return;
  }
  float most[N];
  bool plain[N];
#pragma unroll
  for (int side = 0; side < N; ++side) {
    most[side] = most_of_bf16(raw[side], plain[side]);
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) most[side] = fmaxf(most[side], __shfl_xor_sync(0xffffffffu, most[side], o));
    if (t % 32 == 0) warp_most[side][t / 32] = most[side];
  }
  __syncthreads();
#pragma unroll
  for (int side = 0; side < N; ++side) {
#pragma unroll
    for (int w = 0; w < kWarps; ++w) most[side] = fmaxf(most[side], warp_most[side][w]);
    const int e = fp8_exponent(most[side]);
    uint2* codes = reinterpret_cast<uint2*>((is_v(side) ? p.v : p.k) + (static_cast<size_t>(bh) * p.max_len + row0) * D);
#pragma unroll
    for (int i = 0; i < kPieces; ++i) codes[i * kFillThreads + t] = fp8_of_bf16(raw[side][i], power_of_two(-e), plain[side]);
    if (t == 0) (is_v(side) ? p.v_scale : p.k_scale)[static_cast<size_t>(bh) * p.blocks + block] = power_of_two(e);
  }
}

template <bool BF16, int D>
int launch_fill(const FillParams& p, int B, cudaStream_t st) {
  const dim3 grid((p.S + kFp8Block - 1) / kFp8Block, 2 / kSides<BF16>, B * p.H);
  DAD_CUDA(launch_pdl(kv_cache_fill_fp8_kernel<BF16, D>, grid, dim3(kFillThreads), 0, st, p));
  return DADATTN_OK;
}

}  // namespace
}  // namespace dadattn

using namespace dadattn;

extern "C" int dadattn_fp8_scale_blocks(int max_len) { return max_len <= 0 ? 0 : fp8_scale_blocks(max_len); }

extern "C" int dadattn_kv_cache_fill_fp8(uint8_t* k_cache, uint8_t* v_cache, float* k_scale, float* v_scale, uint16_t* k_tail,
                                         uint16_t* v_tail, int32_t* lengths, const void* k_heads, const void* v_heads,
                                         const int32_t* counts, int B, int H, int S, int max_len, int D, int heads_are_bf16,
                                         dadattn_stream_t stream) {
  for (const void* x : {static_cast<const void*>(k_cache), static_cast<const void*>(v_cache), static_cast<const void*>(k_scale),
                        static_cast<const void*>(v_scale), static_cast<const void*>(k_tail), static_cast<const void*>(v_tail),
                        static_cast<const void*>(lengths), k_heads, v_heads})
    if (!x) return fail(DADATTN_E_ARG, "8-bit cache fill: null pointer");
  if (B <= 0 || H <= 0 || S <= 0 || max_len <= 0)
    return fail(DADATTN_E_ARG, "8-bit cache fill: bad sizes B=%d H=%d S=%d max_len=%d", B, H, S, max_len);
  if (!counts && S > max_len)
    return fail(DADATTN_E_ARG, "8-bit cache fill: %d rows do not fit max_len %d", S, max_len);
  if (max_len > DADATTN_MAX_CACHE_LEN || S > DADATTN_MAX_CACHE_LEN)
    return fail(DADATTN_E_UNSUPPORTED, "8-bit cache fill: S %d and max_len %d may not exceed %d", S, max_len, DADATTN_MAX_CACHE_LEN);
  if (static_cast<long long>(B) * H > 65535)
    return fail(DADATTN_E_UNSUPPORTED, "8-bit cache fill: B*H=%lld exceeds 65535 per call", static_cast<long long>(B) * H);
  if (D != 64 && D != 128) return fail(DADATTN_E_UNSUPPORTED, "8-bit cache fill: unsupported D %d", D);
  for (const void* x : {static_cast<const void*>(k_cache), static_cast<const void*>(v_cache), static_cast<const void*>(k_tail),
                        static_cast<const void*>(v_tail), k_heads, v_heads})
    if (!aligned(x, 16)) return fail(DADATTN_E_ARG, "8-bit cache fill: pointers must be 16-byte aligned");
  for (const void* x : {static_cast<const void*>(k_scale), static_cast<const void*>(v_scale), static_cast<const void*>(lengths),
                        static_cast<const void*>(counts)})
    if (!aligned(x, 4)) return fail(DADATTN_E_ARG, "8-bit cache fill: scales, lengths and counts must be 4-byte aligned");
  FillParams p = {k_heads, v_heads, k_cache, v_cache, k_scale, v_scale, k_tail, v_tail, lengths, counts, device_status_word(),
                  H, S, max_len, fp8_scale_blocks(max_len)};
  if (!p.status) return DADATTN_E_CUDA;
  cudaStream_t st = static_cast<cudaStream_t>(stream);
  if (heads_are_bf16) return D == 64 ? launch_fill<true, 64>(p, B, st) : launch_fill<true, 128>(p, B, st);
  return D == 64 ? launch_fill<false, 64>(p, B, st) : launch_fill<false, 128>(p, B, st);
}
