// New tokens into a paged KV cache: the K and V rows of a packed, ragged batch to the pages of their sequences, keys and
// queries turned by their positions on the way (rotary.cuh), fp32 rows rounded to bf16 once, behind the rotation.
//
// Bound by HBM: every element is read and written once. As in rotary.cu a CTA takes a few tokens and all their heads, of q, k
// and v; which sequence a token belongs to is counted from `starts` by the whole CTA, while the first elements are on their
// way. A page holds the rows of a head one after the other, so a token's row of a head is a run of 128 or 256 bytes.
#include <initializer_list>

#include "paged.cuh"
#include "rotary.cuh"

namespace dadattn {
namespace {

constexpr int kThreads = 256;
constexpr int kMaxTokens = 32;
constexpr int kTable = 2048;

struct PackedStrides {
  int64_t token, head;
};
struct AppendParams {
  const void *q, *k, *v;           // [T, heads, D]
  uint16_t *q_out, *k_pages, *v_pages;
  PackedStrides from[3], to_q;     // q, k, v
  PagedCache cache;
  int T, D, heads_q, heads, units;     // heads: of q, k and v together
  int tokens, heads_first;
  SmallDivisor by_units, by_inner;
  RotaryParams r;
  int* status;
};

using bf16 = __nv_bfloat16;
template <typename T>
__device__ __forceinline__ Sixteen<bf16> rounded(const Sixteen<T>& x) {
  Sixteen<bf16> y;
  float f[16];
  x.to_floats(f);
  y.from_floats(f);
  return y;
}
template <>
__device__ __forceinline__ Sixteen<bf16> rounded(const Sixteen<bf16>& x) { return x; }

template <typename T>
__global__ void __launch_bounds__(kThreads) paged_append_kernel(const AppendParams p) {
  __shared__ __align__(16) float2 table[kTable];
  __shared__ int later[kMaxTokens], before;   // sequences that begin at each token behind the first; up to the first
  __shared__ int row_of[kMaxTokens];          // of its sequence; -1: not written
  __shared__ int64_t place_of[kMaxTokens];    // the row of head 0 in the pool
  const PagedCache& c = p.cache;
  const int t = threadIdx.x, t0 = blockIdx.x * p.tokens, n = min(p.tokens, p.T - t0);
  if (t < kMaxTokens) later[t] = 0;
  if (t == 0) before = 0;
  __syncthreads();
  pdl_wait();
  pdl_launch_dependents();
  const uint32_t all = static_cast<uint32_t>(p.tokens) * p.heads * p.units;
  struct At {
    int token, u, head, which;   // which: 0 q, 1 k, 2 v
  };
  auto locate = [&](uint32_t i) {
    const uint32_t j = p.by_units.divide(i);
    const uint32_t outer = p.by_inner.divide(j), inner = j - outer * p.by_inner.d;
    At at;
    at.u = i - j * p.units;
    at.token = p.heads_first ? inner : outer;
    at.head = p.heads_first ? outer : inner;
    at.which = at.head < p.heads_q ? 0 : at.head < p.heads_q + c.heads ? 1 : 2;
    at.head -= at.which == 0 ? 0 : at.which == 1 ? p.heads_q : p.heads_q + c.heads;
    return at;
  };
  // where a piece lies in its head: V is not turned, so its pieces are runs
  auto first_of = [&](const At& at) { return at.which == 2 ? at.u * kTurnUnit : unit_first(at.u, p.r); };
  auto second_of = [&](const At& at) { return at.which == 2 ? 8 : unit_second(at.u, p.r); };
  auto load = [&](Sixteen<T>& x, const At& at) {
    const PackedStrides& s = p.from[at.which];
    x.load(at.which == 0 ? p.q : at.which == 1 ? p.k : p.v, (t0 + at.token) * s.token + at.head * s.head + first_of(at),
           second_of(at));
  };
  uint32_t i = t;
  At at = locate(i);
  Sixteen<T> now;
  if (i < all && at.token < n) load(now, at);

  if (c.starts) {
    int count = 0;
    for (int b = 1 + t; b <= c.B; b += kThreads) {
      const int s = c.starts[b];
      if (s <= t0) ++count;
      else if (s < t0 + n) atomicAdd(&later[s - t0], 1);
    }
    count = __reduce_add_sync(0xffffffffu, count);
    if (t % 32 == 0 && count) atomicAdd(&before, count);
    __syncthreads();
  }
  if (t < n) {
    int b = t0 + t;
    if (c.starts) {
      b = before;
      for (int j = 1; j <= t; ++j) b += later[j];
    }
    int row = -1;
    if (b < c.B) {   // (tokens behind the last sequence belong to nobody)
      int ahead, first, count;
      const int in = sequence_rows(c, b, p.T, ahead, first, count) ? t0 + t - first : -1;
      if (in >= 0 && in < count) {
        const int page = c.table[static_cast<int64_t>(b) * c.max_pages + ((ahead + in) >> c.page_shift)];
        if (page >= 0 && page < c.pages) {
          row = ahead + in;
          place_of[t] = ((static_cast<int64_t>(page) * c.heads) << c.page_shift) + (row & ((1 << c.page_shift) - 1));
        }
      }
      if (row < 0) atomicExch(p.status, DADATTN_E_ARG);
    }
    row_of[t] = row;
  }
  __syncthreads();
  const int half = p.r.rot / 2;
  if (half) {
    for (int e = t; e < n * half; e += kThreads) {
      const int token = e / half, pair = e - token * half;
      table[token * half + cos_sin_place(pair)] = cos_sin<false>(row_of[token], turns_of(p.r.freq[pair]), p.r.factor);
    }
    __syncthreads();
  }
  while (i < all) {
    const At here = at;
    Sixteen<T> next;
    const uint32_t j = i + kThreads;
    if (j < all) {
      at = locate(j);
      if (at.token < n) load(next, at);
    }
    if (here.token < n && row_of[here.token] >= 0) {
      Sixteen<bf16> y;
      if (here.which < 2 && here.u * kTurnUnit < p.r.rot) {
        float x[16];
        now.to_floats(x);
        turn_unit(x, table + here.token * half, here.u, p.r);
        y.from_floats(x);
      } else {
        y = rounded(now);
      }
      if (here.which == 0) {
        y.store(p.q_out, (t0 + here.token) * p.to_q.token + here.head * p.to_q.head + first_of(here), second_of(here));
      } else {
        const int64_t row = place_of[here.token] + (static_cast<int64_t>(here.head) << c.page_shift);
        y.store(here.which == 1 ? p.k_pages : p.v_pages, row * p.D + first_of(here), second_of(here));
      }
    }
    now = next;
    i = j;
  }
}

__global__ void __launch_bounds__(kThreads) paged_advance_kernel(int32_t* lengths, const PagedCache c, int T, int* status) {
  pdl_wait();
  pdl_launch_dependents();
  const int b = blockIdx.x * kThreads + threadIdx.x;
  if (b >= c.B) return;
  int ahead, first, count;
  if (sequence_rows(c, b, T, ahead, first, count)) lengths[b] = ahead + count;
  else atomicExch(status, DADATTN_E_ARG);
}

}  // namespace
}  // namespace dadattn

using namespace dadattn;

extern "C" int dadattn_paged_append_bf16(uint16_t* k_pages, uint16_t* v_pages, const int32_t* page_table,
                                         const int32_t* lengths, const int32_t* starts, uint16_t* q_out, const void* q,
                                         const void* k_new, const void* v_new, const int64_t* q_out_strides,
                                         const int64_t* q_strides, const int64_t* k_strides, const int64_t* v_strides, int B,
                                         int T, int Hq, int Hkv, int D, int pages, int page_size, int max_pages,
                                         const double* freq, float factor, int rot_dim, int interleaved, int new_is_bf16,
                                         dadattn_stream_t stream) {
  const char* name = "paged append";
  if (int rc = check_paged(name, k_pages, v_pages, page_table, lengths, starts, B, Hkv, D, pages, page_size, max_pages)) return rc;
  if (T <= 0 || Hq < 0) return fail(DADATTN_E_ARG, "%s: bad sizes T=%d Hq=%d", name, T, Hq);
  if (!starts && T != B) return fail(DADATTN_E_ARG, "%s: without starts T=%d is B=%d", name, T, B);
  if (int rc = check_rotary(name, freq, factor, rot_dim, D)) return rc;
  const int64_t piece = new_is_bf16 ? 8 : 4;
  if (Hq > 0) {
    if (int rc = check_packed(name, q, q_strides, piece, false, T, Hq)) return rc;
    if (int rc = check_packed(name, q_out, q_out_strides, 8, true, T, Hq)) return rc;
    if (static_cast<const void*>(q_out) == q &&
        (!new_is_bf16 || q_strides[0] != q_out_strides[0] || q_strides[1] != q_out_strides[1]))
      return fail(DADATTN_E_ARG, "%s: queries that are turned in place are bf16 and have one set of strides", name);
  }
  if (int rc = check_packed(name, k_new, k_strides, piece, false, T, Hkv)) return rc;
  if (int rc = check_packed(name, v_new, v_strides, piece, false, T, Hkv)) return rc;
  if ((static_cast<long long>(Hq) + 2ll * Hkv) * (D / kTurnUnit) > 32768)
    return fail(DADATTN_E_UNSUPPORTED, "%s: Hq=%d and Hkv=%d are too many heads for a call", name, Hq, Hkv);
  AppendParams p = {};
  p.q = q, p.k = k_new, p.v = v_new;
  p.q_out = q_out, p.k_pages = k_pages, p.v_pages = v_pages;
  if (Hq > 0) p.from[0] = PackedStrides{q_strides[0], q_strides[1]}, p.to_q = PackedStrides{q_out_strides[0], q_out_strides[1]};
  p.from[1] = PackedStrides{k_strides[0], k_strides[1]};
  p.from[2] = PackedStrides{v_strides[0], v_strides[1]};
  p.cache = PagedCache{page_table, lengths, starts, B, pages, log2_of(page_size), max_pages, Hkv};
  p.T = T, p.D = D, p.heads_q = Hq, p.heads = Hq + 2 * Hkv, p.units = D / kTurnUnit;
  p.heads_first = k_strides[1] > k_strides[0];
  p.r = RotaryParams{freq, factor, rot_dim, interleaved != 0, 0};
  p.status = device_status_word();
  if (!p.status) return DADATTN_E_CUDA;
  // tokens of a CTA: as in dadattn_rotary
  int tokens = 1;
  const int sms = current_sm_count();
  while (tokens * 2 <= kMaxTokens && tokens * p.heads * p.units < 1024 && tokens * 2 * (rot_dim / 2) <= kTable &&
         (T + tokens * 2 - 1) / (tokens * 2) >= 2 * sms)
    tokens *= 2;
  p.tokens = tokens;
  p.by_units = SmallDivisor(p.units);
  p.by_inner = SmallDivisor(p.heads_first ? tokens : p.heads);
  const dim3 grid((T + tokens - 1) / tokens);
  cudaStream_t st = static_cast<cudaStream_t>(stream);
  if (new_is_bf16) DAD_CUDA(launch_pdl(paged_append_kernel<bf16>, grid, dim3(kThreads), 0, st, p));
  else DAD_CUDA(launch_pdl(paged_append_kernel<float>, grid, dim3(kThreads), 0, st, p));
  return DADATTN_OK;
}

extern "C" int dadattn_paged_advance(int32_t* lengths, const int32_t* starts, int B, int T, int page_size, int max_pages,
                                     dadattn_stream_t stream) {
  const int32_t* any = reinterpret_cast<const int32_t*>(16);   // (there is no pool in this call)
  if (int rc = check_paged("paged advance", any, any, any, lengths, starts, B, 1, 64, 1, page_size, max_pages)) return rc;
  if (T <= 0) return fail(DADATTN_E_ARG, "paged advance: T=%d must be positive", T);
  if (!starts && T != B) return fail(DADATTN_E_ARG, "paged advance: without starts T=%d is B=%d", T, B);
  int* status = device_status_word();
  if (!status) return DADATTN_E_CUDA;
  const PagedCache c = {nullptr, lengths, starts, B, 1, log2_of(page_size), max_pages, 1};
  DAD_CUDA(launch_pdl(paged_advance_kernel, dim3((B + kThreads - 1) / kThreads), dim3(kThreads), 0,
                      static_cast<cudaStream_t>(stream), lengths, c, T, status));
  return DADATTN_OK;
}
