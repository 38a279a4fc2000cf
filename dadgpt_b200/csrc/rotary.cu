// Rotary positions for training: queries and keys turned by their positions ahead of the attention, their gradients turned
// back behind it. The mathematics and the angles: rotary.cuh.
//
// Bound by HBM: every element is read and written once. A CTA takes a few tokens and all their heads: (cos, sin) of a token's
// pairs are computed once, into shared memory, and serve every head of q and of k; the first elements are on their way
// meanwhile. A thread turns 16 elements at a time, two 16-byte pieces (bf16) of a head's two halves or of one run.
#include "rotary.cuh"

#include <cmath>
#include <initializer_list>

namespace dadattn {
namespace {

constexpr int kThreads = 256;
constexpr int kMaxTokens = 32;          // of a CTA
constexpr int kTable = 2048;            // (cos, sin) pairs of a CTA

struct Strides {
  int64_t batch, token, head;
};
struct TurnParams {
  const void* in[2];     // q, k
  void* out[2];
  Strides from[2], to[2];
  const int32_t* positions;   // [B, S] or null: first + s
  int64_t first;
  int S, heads_q, heads, units;       // heads of q; of q and k; pieces of a head that are worked on
  int tokens, tiles, heads_first;     // of a CTA; tiles of a sequence; the order: 1 = a head's tokens next to each other
  SmallDivisor by_units, by_inner;
  RotaryParams r;
};

template <typename T>
__global__ void __launch_bounds__(kThreads) rotary_kernel(const TurnParams p) {
  constexpr bool kExact = sizeof(T) == 4;
  __shared__ __align__(16) float2 table[kTable];
  pdl_wait();
  pdl_launch_dependents();
  const int b = blockIdx.x / p.tiles, s0 = (blockIdx.x - b * p.tiles) * p.tokens, n = min(p.tokens, p.S - s0);
  const int half = p.r.rot / 2;
  const uint32_t all = static_cast<uint32_t>(p.tokens) * p.heads * p.units;
  struct At {
    int token, u, which;
    int64_t from, to;
  };
  auto locate = [&](uint32_t i) {
    const uint32_t j = p.by_units.divide(i), u = i - j * p.units;
    const uint32_t outer = p.by_inner.divide(j), inner = j - outer * p.by_inner.d;
    At at;
    at.token = p.heads_first ? inner : outer;
    at.u = u;
    int head = p.heads_first ? outer : inner;
    at.which = head >= p.heads_q;
    if (at.which) head -= p.heads_q;
    const Strides &f = p.from[at.which], &t = p.to[at.which];
    const int64_t x = unit_first(u, p.r);
    at.from = b * f.batch + (s0 + at.token) * f.token + head * f.head + x;
    at.to = b * t.batch + (s0 + at.token) * t.token + head * t.head + x;
    return at;
  };
  uint32_t i = threadIdx.x;
  At at = locate(i);
  Sixteen<T> now;
  if (i < all && at.token < n) now.load(p.in[at.which], at.from, unit_second(at.u, p.r));
  for (int e = threadIdx.x; e < n * half; e += kThreads) {
    const int token = e / half, pair = e - token * half;
    const int64_t position = p.positions ? p.positions[static_cast<int64_t>(b) * p.S + s0 + token] : p.first + s0 + token;
    table[token * half + cos_sin_place(pair)] = cos_sin<kExact>(position, turns_of(p.r.freq[pair]), p.r.factor);
  }
  __syncthreads();
  while (i < all) {
    const At here = at;
    Sixteen<T> next;
    const uint32_t j = i + kThreads;
    if (j < all) {
      at = locate(j);
      if (at.token < n) next.load(p.in[at.which], at.from, unit_second(at.u, p.r));
    }
    if (here.token < n) {
      if (here.u * kTurnUnit < p.r.rot) {
        float x[16];
        now.to_floats(x);
        turn_unit(x, table + here.token * half, here.u, p.r);
        now.from_floats(x);
      }
      now.store(p.out[here.which], here.to, unit_second(here.u, p.r));
    }
    now = next;
    i = j;
  }
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

extern "C" int dadattn_rotary(void* q_out, void* k_out, const void* q, const void* k, const int64_t* q_out_strides,
                              const int64_t* k_out_strides, const int64_t* q_strides, const int64_t* k_strides,
                              const int32_t* positions, int64_t first, int B, int S, int Hq, int Hk, int D,
                              const double* freq, float factor, int rot_dim, int interleaved, int backward, int is_bf16,
                              dadattn_stream_t stream) {
  if (!q || !q_out || !q_strides || !q_out_strides) return fail(DADATTN_E_ARG, "rotary: null pointer");
  if (B <= 0 || S <= 0 || Hq <= 0 || Hk < 0 || D <= 0)
    return fail(DADATTN_E_ARG, "rotary: bad sizes B=%d S=%d Hq=%d Hk=%d D=%d", B, S, Hq, Hk, D);
  if (Hk > 0 && (!k || !k_out || !k_strides || !k_out_strides)) return fail(DADATTN_E_ARG, "rotary: null pointer");
  if (D % kTurnUnit || D > kMaxRotaryHead)
    return fail(DADATTN_E_UNSUPPORTED, "rotary: unsupported D %d (a multiple of %d up to %d)", D, kTurnUnit, kMaxRotaryHead);
  if (rot_dim <= 0) return fail(DADATTN_E_ARG, "rotary: rot_dim %d must be positive", rot_dim);
  if (int rc = check_rotary("rotary", freq, factor, rot_dim, D)) return rc;
  if (!aligned(positions, 4)) return fail(DADATTN_E_ARG, "rotary: positions must be 4-byte aligned");
  if ((static_cast<long long>(Hq) + Hk) * (D / kTurnUnit) > 32768)
    return fail(DADATTN_E_UNSUPPORTED, "rotary: %lld heads of %d are too many for a call", static_cast<long long>(Hq) + Hk, D);
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
  p.S = S, p.heads_q = Hq, p.heads = Hq + Hk;
  // in place, what is not turned is where it belongs
  const bool same = q == q_out && (Hk == 0 || k == k_out);
  p.units = (same ? rot_dim : D) / kTurnUnit;
  p.r = RotaryParams{freq, factor, rot_dim, interleaved != 0, backward != 0};
  p.heads_first = p.from[0].head > p.from[0].token;
  // Tokens of a CTA: about 1024 pieces, four a thread, but no fewer than two CTAs for each SM.
  int tokens = 1;
  const int sms = current_sm_count();
  while (tokens * 2 <= kMaxTokens && tokens * p.heads * p.units < 1024 && tokens * 2 * (rot_dim / 2) <= kTable &&
         static_cast<long long>(B) * ((S + tokens * 2 - 1) / (tokens * 2)) >= 2 * sms)
    tokens *= 2;
  p.tokens = tokens;
  p.tiles = (S + tokens - 1) / tokens;
  p.by_units = SmallDivisor(p.units);
  p.by_inner = SmallDivisor(p.heads_first ? tokens : p.heads);
  const long long blocks = static_cast<long long>(B) * p.tiles;
  if (blocks > 0x7fffffffll) return fail(DADATTN_E_UNSUPPORTED, "rotary: B*S=%lld is too many tokens", static_cast<long long>(B) * S);
  const dim3 grid(static_cast<unsigned>(blocks));
  cudaStream_t st = static_cast<cudaStream_t>(stream);
  if (is_bf16) DAD_CUDA(launch_pdl(rotary_kernel<__nv_bfloat16>, grid, dim3(kThreads), 0, st, p));
  else DAD_CUDA(launch_pdl(rotary_kernel<float>, grid, dim3(kThreads), 0, st, p));
  return DADATTN_OK;
}
