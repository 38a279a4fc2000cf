// Blocks of an 8-bit KV cache: 64 tokens of one head as e4m3 codes and one scale.
//
// The scale is the least power of two 2^e, e >= -126, with max |x| <= 448 2^e over the block's finite elements (448 is
// the largest e4m3 number). A code is x / 2^e rounded to nearest even; an infinity or NaN becomes NaN. Division by a
// power of two is exact, so an element is rounded once: by at most 2^-4 of itself, or 2^-10 steps of 2^e where it is
// below 2^-6 2^e. A floating format gains nothing from the last factor below two that a scale of max / 448 would use,
// and loses the exactness.
#pragma once

#include <cuda_fp16.h>
#include <cuda_fp8.h>

#include <cstdint>

#include "common.cuh"
#include "sm100_ptx.cuh"

namespace dadattn {

constexpr int kFp8Block = DADATTN_FP8_BLOCK;
// Whole blocks of a cache, and scales of a head (one at least, so that no array is empty)
inline int fp8_scale_blocks(int max_len) { return max_len < kFp8Block ? 1 : max_len / kFp8Block; }

namespace {

// |x| if it is finite, else 0
__device__ __forceinline__ float finite_abs(float x) {
  const float a = fabsf(x);
  return a < INFINITY ? a : 0.f;
}

// e of a block whose largest finite |x| is `most`: most = m 2^x with 1 <= m < 2 needs x - 8, or x - 7 where m > 1.75.
// (A denormal `most` has exponent field 0 and is far below what the least e holds.)
__device__ __forceinline__ int fp8_exponent(float most) {
  const uint32_t bits = __float_as_uint(most);
  const int x = static_cast<int>(bits >> 23) - 127;
  return max(x - 8 + ((bits & 0x7fffffu) > 0x600000u ? 1 : 0), -126);
}
__device__ __forceinline__ float power_of_two(int e) { return __uint_as_float(static_cast<uint32_t>(e + 127) << 23); }

// Largest finite |x| of a thread's pieces of eight bf16 elements; `plain`: none is infinite or NaN. Absolute values are
// compared as 16-bit integers, two at a time, and looked at one by one only where one of them is not finite.
template <int N>
__device__ __forceinline__ float most_of_bf16(const uint4 (&raw)[N], bool& plain) {
  uint32_t m = 0;
#pragma unroll
  for (int i = 0; i < N; ++i)
    for (const uint32_t w : {raw[i].x, raw[i].y, raw[i].z, raw[i].w}) m = __vmaxu2(m, w & 0x7fff7fffu);
  const uint32_t top = max(m >> 16, m & 0xffffu);
  plain = top < 0x7f80u;
  if (plain) return __uint_as_float(top << 16);
  float most = 0.f;
#pragma unroll
  for (int i = 0; i < N; ++i)
    for (const uint32_t w : {raw[i].x, raw[i].y, raw[i].z, raw[i].w})
      most = fmaxf(most, fmaxf(finite_abs(__uint_as_float(w << 16)), finite_abs(__uint_as_float(w & 0xffff0000u))));
  return most;
}

// Eight bf16 elements -> eight codes, the first in the lowest byte. `inv` = 2^-e.
__device__ __forceinline__ uint2 fp8_of_bf16(const uint4& raw, float inv, bool plain) {
  const uint32_t w[4] = {raw.x, raw.y, raw.z, raw.w};
  uint32_t c[4];
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    float a = __uint_as_float(w[i] << 16) * inv, b = __uint_as_float(w[i] & 0xffff0000u) * inv;
    if (!plain) {   // (the conversion would make an infinity 448)
      if (fabsf(a) == INFINITY) a = NAN;
      if (fabsf(b) == INFINITY) b = NAN;
    }
    c[i] = __nv_cvt_float2_to_fp8x2(make_float2(a, b), __NV_SATFINITE, __NV_E4M3);
  }
  return make_uint2(c[0] | c[1] << 16, c[2] | c[3] << 16);
}

}  // namespace
}  // namespace dadattn
