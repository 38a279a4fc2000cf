// Rotary positions: the angle of a (position, pair), and the turn of 16 elements of a head.
//
// Pair i of a head of which `rot` elements are turned has the frequency w_i (radians per position). At position p
//   y1 = f (cos(p w_i) x1 - sin(p w_i) x2),  y2 = f (cos(p w_i) x2 + sin(p w_i) x1)
// with (x1, x2) elements (i, i + rot / 2), or (2 i, 2 i + 1) where pairs are interleaved. The gradient is turned by -p.
//
// Angles: p w in 32 bits loses 2^-24 of itself, 0.06 radians at a million positions, and in 64-bit arithmetic the reduction
// of a large angle would cost more than the rotation. So a frequency becomes a 64-bit fraction of a turn, and p times it,
// modulo 2^64, is the angle modulo a turn without any rounding: what is left is the fraction's own, 2^-53 of the frequency
// and 2^-65 of a turn, times p. The nearest quarter turn is taken off in integers too, so that the sine and cosine are those
// of at most an eighth of a turn, whose conversion to a float is off by 2^-28 of a turn at most (2.4e-8 radians).
#pragma once

#include <cuda_bf16.h>

#include "common.cuh"
#include "sm100_ptx.cuh"

namespace dadattn {

constexpr int kTurnUnit = 16;            // elements that a thread turns at a time
constexpr int kMaxRotaryHead = 256;      // largest head size

// What a kernel needs to know of the rotation. rot = 0: none.
struct RotaryParams {
  const double* freq;   // [rot / 2], radians per position
  float factor;         // of the turned elements
  int rot;
  int interleaved;
  int back;             // 1: by the negative angle (gradients)
};

// What every call with a rotation checks.
inline int check_rotary(const char* name, const double* freq, float factor, int rot, int D) {
  if (rot == 0) return DADATTN_OK;
  if (rot < 0 || rot > D) return fail(DADATTN_E_ARG, "%s: rot_dim %d must be within the head's %d elements", name, rot, D);
  if (rot % kTurnUnit) return fail(DADATTN_E_UNSUPPORTED, "%s: rot_dim %d is not a multiple of %d", name, rot, kTurnUnit);
  if (!freq || !aligned(freq, 8)) return fail(DADATTN_E_ARG, "%s: freq must be an 8-byte aligned device pointer", name);
  if (!(factor > -INFINITY && factor < INFINITY)) return fail(DADATTN_E_ARG, "%s: factor must be finite", name);
  return DADATTN_OK;
}

inline int current_sm_count() {
  int dev = 0, sms = 0;
  if (cudaGetDevice(&dev) != cudaSuccess || cudaDeviceGetAttribute(&sms, cudaDevAttrMultiProcessorCount, dev) != cudaSuccess)
    return 148;   // (only rules of speed go by it; a call without a device fails at its launch)
  return sms;
}

#ifdef __CUDACC__
// Turns per position, modulo 1, times 2^64.
__device__ __forceinline__ uint64_t turns_of(double freq) {
  const double t = freq * 0.15915494309189533577;   // 1 / (2 pi)
  return __double2ull_rn((t - floor(t)) * 18446744073709551616.0);   // (a fraction that rounds to 1 saturates)
}

// (cos, sin) of position * turns, times the factor. EXACT: to fp32 accuracy, else to 2^-21 (for results in bf16, whose
// rounding is 2^-9).
template <bool EXACT>
__device__ __forceinline__ float2 cos_sin(int64_t position, uint64_t turns, float factor) {
  const uint64_t a = static_cast<uint64_t>(position) * turns;
  const uint64_t quarter = (a + (1ull << 61)) >> 62;          // to the nearest, 0..3 (wraps with the turn)
  const int32_t rest = static_cast<int32_t>(static_cast<int64_t>(a - (quarter << 62)) >> 32);   // [-1/8, 1/8] turns * 2^32
  float s, c;
  if (EXACT) sincospif(static_cast<float>(rest) * 4.656612873077393e-10f, &s, &c);              // 2^-31: half turns
  else __sincosf(static_cast<float>(rest) * 1.4629180792671596e-9f, &s, &c);                    // 2 pi / 2^32
  const float cq = (quarter & 1) ? s : c, sq = (quarter & 1) ? c : s;
  return make_float2((quarter == 1 || quarter == 2 ? -cq : cq) * factor, (quarter >= 2 ? -sq : sq) * factor);
}

// 16 elements of a head, as they lie in memory in two pieces of eight.
template <typename T>
struct Sixteen;
template <>
struct Sixteen<__nv_bfloat16> {
  uint4 a, b;
  __device__ __forceinline__ void load(const void* base, int64_t at, int64_t to_second) {
    const __nv_bfloat16* p = static_cast<const __nv_bfloat16*>(base) + at;
    a = *reinterpret_cast<const uint4*>(p);
    b = *reinterpret_cast<const uint4*>(p + to_second);
  }
  __device__ __forceinline__ void to_floats(float (&x)[16]) const {
    const uint32_t w[8] = {a.x, a.y, a.z, a.w, b.x, b.y, b.z, b.w};
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      x[2 * i] = __uint_as_float(w[i] << 16);
      x[2 * i + 1] = __uint_as_float(w[i] & 0xffff0000u);
    }
  }
  __device__ __forceinline__ void from_floats(const float (&x)[16]) {
    a = make_uint4(ptx::pack_bf16(x[0], x[1]), ptx::pack_bf16(x[2], x[3]), ptx::pack_bf16(x[4], x[5]), ptx::pack_bf16(x[6], x[7]));
    b = make_uint4(ptx::pack_bf16(x[8], x[9]), ptx::pack_bf16(x[10], x[11]), ptx::pack_bf16(x[12], x[13]),
                   ptx::pack_bf16(x[14], x[15]));
  }
  __device__ __forceinline__ void store(void* base, int64_t at, int64_t to_second) const {
    __nv_bfloat16* p = static_cast<__nv_bfloat16*>(base) + at;
    *reinterpret_cast<uint4*>(p) = a;
    *reinterpret_cast<uint4*>(p + to_second) = b;
  }
};
template <>
struct Sixteen<float> {
  float4 v[4];
  __device__ __forceinline__ void load(const void* base, int64_t at, int64_t to_second) {
    const float* p = static_cast<const float*>(base) + at;
    v[0] = *reinterpret_cast<const float4*>(p);
    v[1] = *reinterpret_cast<const float4*>(p + 4);
    v[2] = *reinterpret_cast<const float4*>(p + to_second);
    v[3] = *reinterpret_cast<const float4*>(p + to_second + 4);
  }
  __device__ __forceinline__ void to_floats(float (&x)[16]) const {
#pragma unroll
    for (int i = 0; i < 4; ++i) x[4 * i] = v[i].x, x[4 * i + 1] = v[i].y, x[4 * i + 2] = v[i].z, x[4 * i + 3] = v[i].w;
  }
  __device__ __forceinline__ void from_floats(const float (&x)[16]) {
#pragma unroll
    for (int i = 0; i < 4; ++i) v[i] = make_float4(x[4 * i], x[4 * i + 1], x[4 * i + 2], x[4 * i + 3]);
  }
  __device__ __forceinline__ void store(void* base, int64_t at, int64_t to_second) const {
    float* p = static_cast<float*>(base) + at;
    *reinterpret_cast<float4*>(p) = v[0];
    *reinterpret_cast<float4*>(p + 4) = v[1];
    *reinterpret_cast<float4*>(p + to_second) = v[2];
    *reinterpret_cast<float4*>(p + to_second + 4) = v[3];
  }
};

// Where piece u of 16 elements lies in a head: its first element, and how far behind that its second eight begin. Pieces
// 0 .. rot / 16 - 1 are turned, the others pass.
__device__ __forceinline__ int unit_first(int u, const RotaryParams& r) {
  return u * kTurnUnit < r.rot && !r.interleaved ? u * 8 : u * kTurnUnit;
}
__device__ __forceinline__ int unit_second(int u, const RotaryParams& r) {
  return u * kTurnUnit < r.rot && !r.interleaved ? r.rot / 2 : 8;
}

// (cos, sin) of a token's pairs lie in shared memory, eight pairs (64 bytes) for a piece. The four 16-byte words of piece u
// change places by u, so that the threads of eight neighbouring pieces, which read the same word at a time, find it in
// different banks.
__device__ __forceinline__ int cos_sin_place(int pair) {   // in float2
  const int u = pair >> 3, word = (pair >> 1) & 3;
  return u * 8 + ((word ^ (u >> 1 & 3)) << 1) + (pair & 1);
}
// Turns the 16 elements of piece u of a token, whose table is cs.
__device__ __forceinline__ void turn_unit(float (&x)[16], const float2* cs, int u, const RotaryParams& r) {
  const float4* table = reinterpret_cast<const float4*>(cs + u * 8);
  const int move = u >> 1 & 3;
  auto turn = [&](float& a, float& b, float c, float s) {
    const float y = c * a - s * b;
    b = c * b + s * a;
    a = y;
  };
#pragma unroll
  for (int w = 0; w < 4; ++w) {
    float4 t = table[w ^ move];
    if (r.back) t.y = -t.y, t.w = -t.w;
    if (r.interleaved) {
      turn(x[4 * w], x[4 * w + 1], t.x, t.y);
      turn(x[4 * w + 2], x[4 * w + 3], t.z, t.w);
    } else {
      turn(x[2 * w], x[2 * w + 8], t.x, t.y);
      turn(x[2 * w + 1], x[2 * w + 9], t.z, t.w);
    }
  }
}

// idx / d for idx and d below 2^16 and idx * d below 2^32.
struct SmallDivisor {
  uint32_t d, m;
  SmallDivisor(int by = 1) : d(by), m(by == 1 ? 0 : static_cast<uint32_t>((0x100000000ull + by - 1) / by)) {}
  __device__ __forceinline__ uint32_t divide(uint32_t i) const { return m ? __umulhi(i, m) : i; }
};
#endif

}  // namespace dadattn
