// Rotary positions for training: queries and keys turned by their positions ahead of the attention, their gradients turned
// back behind it. The mathematics and the angles: rotary.cuh.
//
// Bound by HBM: every element is read and written once. A thread has one piece of 16 elements (two runs of 16 bytes in bf16) of a
// token and goes through a group of its heads, with (cos, sin) of the piece's eight pairs in registers. (From a table in shared
// memory, heads side by side in a warp, the table's reads alone were 16 wavefronts for every 8 of the tensors': 41 us instead of
// 35.6 for forward and backward of 16 x 1024 x 24 heads of 64.)
// Measured: 16 x 1024 x 24 heads of 64, bf16, heads split 17.8 us (5.7 TB/s), fp32 33.6 (6.0); 8192 tokens of 40 heads of 128
// 28.0 (6.0); 140 tokens of 8 heads of 32, fp32, 2.3.
#include "rotary.cuh"

#include <algorithm>
#include <cmath>
#include <initializer_list>

namespace dadattn {
namespace {

constexpr int kThreads = 128;

struct Strides {
  int64_t batch, token, head;
};
struct TurnParams {
  const void* in[2];     // q, k
  void* out[2];
  Strides from[2], to[2];
  const int32_t* positions;   // [B, S] or null: first + s
  int64_t first;
  int S, heads[2], units;      // units: pieces of a head that are worked on
  int groups[2];               // of q's heads, and of k's behind them; a thread goes through one
  int64_t tokens;              // B * S
  RotaryParams r;
};

template <typename T>
__global__ void __launch_bounds__(kThreads) rotary_kernel(const TurnParams p) {
  constexpr bool kExact = sizeof(T) == 4;
  pdl_wait();
  pdl_launch_dependents();
  const int64_t i = static_cast<int64_t>(blockIdx.x) * kThreads + threadIdx.x, token = i / p.units;
  if (token >= p.tokens) return;
  const int u = static_cast<int>(i - token * p.units);
  const int64_t b = token / p.S, s = token - b * p.S;
  const int which = static_cast<int>(blockIdx.y) >= p.groups[0], g = blockIdx.y - (which ? p.groups[0] : 0);
  const int head0 = g * p.heads[which] / p.groups[which], n = (g + 1) * p.heads[which] / p.groups[which] - head0;
  const bool turned = u * kTurnUnit < p.r.rot;
  float2 cs[8];
  if (turned) cos_sin_of<kExact>(cs, u, p.positions ? p.positions[token] : p.first + s, p.r);
  const Strides &f = p.from[which], &t = p.to[which];
  const int x = unit_first(u, p.r);
  const T* in = static_cast<const T*>(p.in[which]) + b * f.batch + s * f.token + head0 * f.head + x;
  T* out = static_cast<T*>(p.out[which]) + b * t.batch + s * t.token + head0 * t.head + x;
  turn_heads<sizeof(T) == 4 ? 2 : 4>(in, f.head, out, t.head, n, unit_second(u, p.r), turned, cs, p.r.interleaved);
}

}  // namespace
}  // namespace dadattn

using namespace dadattn;

extern "C" int dadattn_rotary_frequencies(double* freq, int rot_dim, double base, int scaling, double stretch,
                                          double trained_len, double low, double high) {
  if (!freq) return fail(DADATTN_E_ARG, "rotary frequencies: null pointer");
  if (rot_dim <= 0 || rot_dim % 2 || rot_dim > kMaxRotaryHead)
    return fail(DADATTN_E_ARG, "rotary frequencies: rot_dim %d must be even, positive and at most %d", rot_dim, kMaxRotaryHead);
  if (!(base > 1.0 && base < INFINITY)) return fail(DADATTN_E_ARG, "rotary frequencies: base must be above 1 and finite");
  if (scaling < DADATTN_ROTARY_PLAIN || scaling > DADATTN_ROTARY_PARTS)
    return fail(DADATTN_E_ARG, "rotary frequencies: unknown scaling %d", scaling);
  if (scaling != DADATTN_ROTARY_PLAIN && !(stretch >= 1.0 && stretch < INFINITY))
    return fail(DADATTN_E_ARG, "rotary frequencies: stretch must be at least 1 and finite");
  if (scaling == DADATTN_ROTARY_PARTS &&
      !(trained_len > 0.0 && trained_len < INFINITY && low >= 0.0 && high > low && high < INFINITY))
    return fail(DADATTN_E_ARG, "rotary frequencies: by parts needs a trained length above 0 and 0 <= low < high");
  if (scaling == DADATTN_ROTARY_BASE) base *= std::pow(stretch, rot_dim > 2 ? rot_dim / (rot_dim - 2.0) : 2.0);
  for (int i = 0; i < rot_dim / 2; ++i) {
    double f = std::pow(base, -2.0 * i / rot_dim);
    if (scaling == DADATTN_ROTARY_LINEAR) f /= stretch;
    if (scaling == DADATTN_ROTARY_PARTS) {
      const double turns = trained_len * f / 6.283185307179586477;
      double keep = (turns - low) / (high - low);
      keep = keep < 0.0 ? 0.0 : keep > 1.0 ? 1.0 : keep;
      f = keep * f + (1.0 - keep) * f / stretch;
    }
    freq[i] = f;
  }
  return DADATTN_OK;
}

extern "C" int dadattn_rotary_turns(uint64_t* turns, const double* freq, int count) {
  if (!turns || !freq) return fail(DADATTN_E_ARG, "rotary turns: null pointer");
  if (count <= 0) return fail(DADATTN_E_ARG, "rotary turns: count %d must be positive", count);
  for (int i = 0; i < count; ++i) {
    if (!(freq[i] > -1e15 && freq[i] < 1e15)) return fail(DADATTN_E_ARG, "rotary turns: frequency %d is not finite, or too large", i);
    long double t = freq[i] * 0.159154943091895335768883763372514362L;   // 1 / (2 pi)
    t = (t - std::floor(t)) * 18446744073709551616.0L;
    const long double whole = std::floor(t + 0.5L);
    turns[i] = whole >= 18446744073709551616.0L ? 0 : static_cast<uint64_t>(whole);
  }
  return DADATTN_OK;
}

extern "C" int dadattn_rotary(void* q_out, void* k_out, const void* q, const void* k, const int64_t* q_out_strides,
                              const int64_t* k_out_strides, const int64_t* q_strides, const int64_t* k_strides,
                              const int32_t* positions, int64_t first, int B, int S, int Hq, int Hk, int D,
                              const uint64_t* turns, float factor, int rot_dim, int interleaved, int backward, int is_bf16,
                              dadattn_stream_t stream) {
  if (!q || !q_out || !q_strides || !q_out_strides) return fail(DADATTN_E_ARG, "rotary: null pointer");
  if (B <= 0 || S <= 0 || Hq <= 0 || Hk < 0 || D <= 0)
    return fail(DADATTN_E_ARG, "rotary: bad sizes B=%d S=%d Hq=%d Hk=%d D=%d", B, S, Hq, Hk, D);
  if (Hk > 0 && (!k || !k_out || !k_strides || !k_out_strides)) return fail(DADATTN_E_ARG, "rotary: null pointer");
  if (D % kTurnUnit || D > kMaxRotaryHead)
    return fail(DADATTN_E_UNSUPPORTED, "rotary: unsupported D %d (a multiple of %d up to %d)", D, kTurnUnit, kMaxRotaryHead);
  if (rot_dim <= 0) return fail(DADATTN_E_ARG, "rotary: rot_dim %d must be positive", rot_dim);
  if (int rc = check_rotary("rotary", turns, factor, rot_dim, D)) return rc;
  if (!aligned(positions, 4)) return fail(DADATTN_E_ARG, "rotary: positions must be 4-byte aligned");
  if (Hq > 65535 - Hk) return fail(DADATTN_E_UNSUPPORTED, "rotary: Hq=%d and Hk=%d exceed 65535 together", Hq, Hk);
  const int64_t piece = is_bf16 ? 8 : 4;   // elements of 16 bytes
  TurnParams p = {};
  const int64_t* strides[4] = {q_strides, k_strides, q_out_strides, k_out_strides};
  const void* tensors[4] = {q, k, q_out, k_out};
  for (int i = 0; i < 4; ++i) {
    if (i % 2 && Hk == 0) continue;
    const int64_t* s = strides[i];
    if (!aligned(tensors[i], 16) || s[0] % piece || s[1] % piece || s[2] % piece)
      return fail(DADATTN_E_ARG, "rotary: rows must begin at multiples of 16 bytes (pointers and strides)");
    if (s[0] < 0 || s[1] < 0 || s[2] < 0) return fail(DADATTN_E_ARG, "rotary: strides must not be negative");
    if (i >= 2 && ((B > 1 && s[0] == 0) || (S > 1 && s[1] == 0) || ((i % 2 ? Hk : Hq) > 1 && s[2] == 0)))
      return fail(DADATTN_E_ARG, "rotary: the results' rows must not lie over each other");
    (i < 2 ? p.from : p.to)[i % 2] = Strides{s[0], s[1], s[2]};
  }
  for (int i = 0; i < 2; ++i) {   // written in place: element for element
    const Strides &f = p.from[i], &t = p.to[i];
    if (tensors[i] && tensors[i] == tensors[2 + i] && (f.batch != t.batch || f.token != t.token || f.head != t.head))
      return fail(DADATTN_E_ARG, "rotary: a tensor that is turned in place has one set of strides");
  }
  p.in[0] = q, p.in[1] = k, p.out[0] = q_out, p.out[1] = k_out;
  p.positions = positions;
  p.first = first;
  p.S = S, p.heads[0] = Hq, p.heads[1] = Hk;
  // in place, what is not turned is where it belongs
  const bool same = q == q_out && (Hk == 0 || k == k_out);
  p.units = (same ? rot_dim : D) / kTurnUnit;
  p.r = RotaryParams{turns, factor, rot_dim, interleaved != 0, backward != 0};
  p.tokens = static_cast<int64_t>(B) * S;
  const long long blocks = (p.tokens * p.units + kThreads - 1) / kThreads;
  if (blocks > 0x7fffffffll) return fail(DADATTN_E_UNSUPPORTED, "rotary: B*S=%lld is too many tokens", static_cast<long long>(p.tokens));
  // Four heads a thread, which are all on their way at once, or fewer where the call has less than four CTAs an SM. (us of
  // forward and backward, 16 x 1024 x 24 heads of 64 and 8192 x 40 of 128: two or three heads 41 and -, four 35.6 and 56.5, five
  // or six 37 and 59, eight - and 60.)
  const auto groups = [&](int heads) { return heads ? std::max(head_groups(blocks, heads, Hq + Hk, 4), (heads + 3) / 4) : 0; };
  p.groups[0] = groups(Hq);
  p.groups[1] = groups(Hk);
  const dim3 grid(static_cast<unsigned>(blocks), p.groups[0] + p.groups[1]);
  cudaStream_t st = static_cast<cudaStream_t>(stream);
  if (is_bf16) DAD_CUDA(launch_pdl(rotary_kernel<__nv_bfloat16>, grid, dim3(kThreads), 0, st, p));
  else DAD_CUDA(launch_pdl(rotary_kernel<float>, grid, dim3(kThreads), 0, st, p));
  return DADATTN_OK;
}
