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

// Two codes, the first in the low byte. `inv` = 2^-e.
__device__ __forceinline__ uint32_t fp8_pair(float a, float b, float inv) {
  a *= inv;
  b *= inv;
  if (fabsf(a) == INFINITY) a = NAN;   // (the conversion would make it 448)
  if (fabsf(b) == INFINITY) b = NAN;
  return __nv_cvt_float2_to_fp8x2(make_float2(a, b), __NV_SATFINITE, __NV_E4M3);
}

// Eight bf16 elements -> eight codes.
__device__ __forceinline__ uint2 fp8_of_bf16(const uint4& raw, float inv) {
  const uint32_t w[4] = {raw.x, raw.y, raw.z, raw.w};
  uint32_t c[4];
#pragma unroll
  for (int i = 0; i < 4; ++i)
    c[i] = fp8_pair(__uint_as_float(w[i] << 16), __uint_as_float(w[i] & 0xffff0000u), inv);
  return make_uint2(c[0] | c[1] << 16, c[2] | c[3] << 16);
}
__device__ __forceinline__ float most_of_bf16(const uint4& raw) {
  const uint32_t w[4] = {raw.x, raw.y, raw.z, raw.w};
  float m = 0.f;
#pragma unroll
  for (int i = 0; i < 4; ++i)
    m = fmaxf(m, fmaxf(finite_abs(__uint_as_float(w[i] << 16)), finite_abs(__uint_as_float(w[i] & 0xffff0000u))));
  return m;
}

}  // namespace
}  // namespace dadattn
