// Rotary positions: the angle of a (position, pair), and the turn of 16 elements of a head.
//
// Pair i of a head of which `rot` elements are turned has the frequency w_i (radians per position). At position p
//   y1 = f (cos(p w_i) x1 - sin(p w_i) x2),  y2 = f (cos(p w_i) x2 + sin(p w_i) x1)
// with (x1, x2) elements (i, i + rot / 2), or (2 i, 2 i + 1) where pairs are interleaved. The gradient is turned by -p.
//
// Angles: p w in 32 bits loses 2^-24 of itself, 0.06 radians at a million positions, and in 64-bit floating point the reduction
// of a large angle would cost more than the rotation. So a frequency comes as a 64-bit fraction of a turn (dadattn_rotary_turns),
// and p times it, modulo 2^64, is the angle modulo a turn without any rounding: what is left is the fraction's own, half a unit,
// times p. The nearest quarter turn is taken off in integers too, so that the sine and cosine are those of at most an eighth of
// a turn, whose conversion to a float is off by 2^-28 of a turn at most (2.4e-8 radians).
#pragma once

#include <cuda_bf16.h>

#include "common.cuh"
#include "sm100_ptx.cuh"

namespace dadattn {

constexpr int kTurnUnit = 16;            // elements that a thread turns at a time
constexpr int kMaxRotaryHead = 256;      // largest head size

// What a kernel needs to know of the rotation. rot = 0: none.
struct RotaryParams {
  const uint64_t* turns;   // [rot / 2], 2^-64 turns per position
  float factor;            // of the turned elements
  int rot;
  int interleaved;
  int back;                // 1: by the negative angle (gradients)
};

// What every call with a rotation checks.
inline int check_rotary(const char* name, const uint64_t* turns, float factor, int rot, int D) {
  if (rot == 0) return DADATTN_OK;
  if (rot < 0 || rot > D) return fail(DADATTN_E_ARG, "%s: rot_dim %d must be within the head's %d elements", name, rot, D);
  if (rot % kTurnUnit) return fail(DADATTN_E_UNSUPPORTED, "%s: rot_dim %d is not a multiple of %d", name, rot, kTurnUnit);
  if (!turns || !aligned(turns, 16)) return fail(DADATTN_E_ARG, "%s: turns must be a 16-byte aligned device pointer", name);
  if (!(factor > -INFINITY && factor < INFINITY)) return fail(DADATTN_E_ARG, "%s: factor must be finite", name);
  return DADATTN_OK;
}

inline int current_sm_count() {
  static std::atomic<int> seen[64];   // by device
  int dev = 0, sms = 0;
  if (cudaGetDevice(&dev) != cudaSuccess || dev < 0 || dev >= 64) return 148;   // (only rules of speed go by it; a call without a
  if ((sms = seen[dev].load(std::memory_order_relaxed))) return sms;            // device fails at its launch)
  if (cudaDeviceGetAttribute(&sms, cudaDevAttrMultiProcessorCount, dev) != cudaSuccess) return 148;
  seen[dev].store(sms, std::memory_order_relaxed);
  return sms;
}

// Groups that `heads` heads are dealt out to, a thread going through one, where a head takes `blocks` CTAs and all heads of the
// call are `all`: so many that the call has `per_sm` CTAs an SM.
inline int head_groups(long long blocks, int heads, int all, int per_sm) {
  const long long groups = (static_cast<long long>(per_sm) * current_sm_count() * heads + blocks * all - 1) / (blocks * all);
  return static_cast<int>(groups < heads ? groups : heads);
}

#ifdef __CUDACC__
// sin and cos of r half turns, |r| <= 1/4, by polynomials in r^2 that were fitted for the least error over that range: off by
// 4.6e-8 and 5.9e-8 in fp32 over all their arguments (pi comes in two parts). 12 operations; sincospif, which takes any r, made a short fp32 call 1 us
// longer, at eight pairs a thread.
__device__ __forceinline__ void sin_cos_eighth(float r, float* s, float* c) {
  const float z = r * r;
  float p = fmaf(fmaf(-0.5894796f, z, 2.5498104f), z, -5.1677094f);
  p = fmaf(r, p * z, r * -8.742278e-8f);
  *s = fmaf(r, 3.14159274f, p);
  *c = fmaf(fmaf(fmaf(fmaf(0.23142955f, z, -1.3350585f), z, 4.0587077f), z, -4.934802f), z, 1.0f);
}

// (cos, sin) of position * turns, times the factor. EXACT: to fp32 accuracy, else to 2^-21 (for results in bf16, whose
// rounding is 2^-8).
template <bool EXACT>
__device__ __forceinline__ float2 cos_sin(int64_t position, uint64_t turns, float factor) {
  const uint64_t a = static_cast<uint64_t>(position) * turns;
  const uint64_t quarter = (a + (1ull << 61)) >> 62;          // to the nearest, 0..3 (wraps with the turn)
  const int32_t rest = static_cast<int32_t>(static_cast<int64_t>(a - (quarter << 62)) >> 32);   // [-1/8, 1/8] turns * 2^32
  float s, c;
  if (EXACT) sin_cos_eighth(static_cast<float>(rest) * 4.656612873077393e-10f, &s, &c);         // 2^-31: half turns
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

// The eight (cos, sin) of piece u of a token at this position, for a thread that turns that piece of several heads.
template <bool EXACT>
__device__ __forceinline__ void cos_sin_of(float2 (&cs)[8], int u, int64_t position, const RotaryParams& r) {
  const ulonglong2* turns = reinterpret_cast<const ulonglong2*>(r.turns + u * 8);
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const ulonglong2 two = __ldg(turns + i);
    cs[2 * i] = cos_sin<EXACT>(position, two.x, r.factor);
    cs[2 * i + 1] = cos_sin<EXACT>(position, two.y, r.factor);
  }
  if (r.back) {
#pragma unroll
    for (int i = 0; i < 8; ++i) cs[i].y = -cs[i].y;
  }
}
// 16 elements by eight (cos, sin); both layouts of the pairs.
__device__ __forceinline__ void turn_unit(float (&x)[16], const float2 (&cs)[8], bool interleaved) {
  auto turn = [&](float& a, float& b, float2 c) {
    const float y = c.x * a - c.y * b;
    b = c.x * b + c.y * a;
    a = y;
  };
  if (interleaved) {
#pragma unroll
    for (int i = 0; i < 8; ++i) turn(x[2 * i], x[2 * i + 1], cs[i]);
  } else {
#pragma unroll
    for (int i = 0; i < 8; ++i) turn(x[i], x[i + 8], cs[i]);
  }
}

template <typename To, typename From>
__device__ __forceinline__ Sixteen<To> converted(const Sixteen<From>& x) {
  Sixteen<To> y;
  float f[16];
  x.to_floats(f);
  y.from_floats(f);
  return y;
}
template <>
__device__ __forceinline__ Sixteen<__nv_bfloat16> converted(const Sixteen<__nv_bfloat16>& x) { return x; }   // (NaN as it is)
template <>
__device__ __forceinline__ Sixteen<float> converted(const Sixteen<float>& x) { return x; }

// One piece of `n` heads, `in_step` and `out_step` elements apart, turned or passed on. AHEAD heads are on their way at a time.
template <int AHEAD, typename From, typename To>
__device__ __forceinline__ void turn_heads(const From* in, int64_t in_step, To* out, int64_t out_step, int n, int second,
                                           bool turned, const float2 (&cs)[8], bool interleaved) {
  for (int h = 0; h < n; h += AHEAD) {
    Sixteen<From> x[AHEAD];
#pragma unroll
    for (int k = 0; k < AHEAD; ++k)
      if (h + k < n) x[k].load(in, (h + k) * in_step, second);
#pragma unroll
    for (int k = 0; k < AHEAD; ++k) {
      if (h + k >= n) break;
      Sixteen<To> y;
      if (turned) {
        float f[16];
        x[k].to_floats(f);
        turn_unit(f, cs, interleaved);
        y.from_floats(f);
      } else {
        y = converted<To>(x[k]);
      }
      y.store(out, (h + k) * out_step, second);
    }
  }
}
#endif

}  // namespace dadattn
