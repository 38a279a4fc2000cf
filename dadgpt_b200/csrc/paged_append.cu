// New tokens into a paged KV cache: the K and V rows of a packed, ragged batch to the pages of their sequences, keys and
// queries turned by their positions on the way (rotary.cuh), fp32 rows rounded to bf16 once, behind the rotation.
//
// Bound by HBM: every element is read and written once. As in rotary.cu a thread has one piece of 16 elements of a token and goes
// through a group of its heads, of q, k or v. A CTA's tokens are next to each other; which sequences they belong to is counted
// from `starts` by the whole CTA. A page holds the rows of a head one after the other, so a token's row of a head is a run of 128
// or 256 bytes.
// Measured: 14747 tokens of 16 sequences, 32 query and 8 key heads of 128, turned, bf16 59.5 us (6.1 TB/s); 301 tokens of 12 heads of
// 64, fp32, 3.0.
#include <initializer_list>

#include "paged.cuh"
#include "rotary.cuh"

namespace dadattn {
namespace {

constexpr int kThreads = 128;
constexpr int kMaxTokens = 64;           // of a CTA: a head has four pieces at least

struct PackedStrides {
  int64_t token, head;
};
struct AppendParams {
  const void *q, *k, *v;           // [T, heads, D]
  uint16_t *q_out, *k_pages, *v_pages;
  PackedStrides from[3], to_q;     // q, k, v
  PagedCache cache;
  int T, D, heads_q, units;            // units: pieces of a head
  int groups_q, groups_kv;             // of q's heads, of k's, and those of v's behind them; a thread goes through one
  RotaryParams r;
  int* status;
};

using bf16 = __nv_bfloat16;

template <typename T>
__global__ void __launch_bounds__(kThreads) paged_append_kernel(const AppendParams p) {
  __shared__ int later[kMaxTokens], before;   // sequences that begin at each token behind the first; up to the first
  const PagedCache& c = p.cache;
  const int t = threadIdx.x, tokens = kThreads / p.units, t0 = blockIdx.x * tokens, n = min(tokens, p.T - t0);
  if (t < kMaxTokens) later[t] = 0;
  if (t == 0) before = 0;
  __syncthreads();
  pdl_wait();
  pdl_launch_dependents();
  const int at = t / p.units, u = t - at * p.units;   // this thread's token and piece
  int b = t0 + at;
  if (c.starts) {
    int count = 0;
    for (int i = 1 + t; i <= c.B; i += kThreads) {
      const int s = c.starts[i];
      if (s <= t0) ++count;
      else if (s < t0 + n) atomicAdd(&later[s - t0], 1);
    }
    count = __reduce_add_sync(0xffffffffu, count);
    if (t % 32 == 0 && count) atomicAdd(&before, count);
    // A sequence without new rows is reported here: the CTAs of V's last heads, which form no angles, look at some each. (us
    // without / by all these CTAs / by one: 2000 sequences 10.2 / 10.5 / 12.8, 300 6.75 / 6.95 / 6.95, 16 3.4 / 3.45 / 3.45.)
    if (blockIdx.y == gridDim.y - 1) {
      int ahead, first, many;
      for (int64_t i = static_cast<int64_t>(blockIdx.x) * kThreads + t; i < c.B; i += static_cast<int64_t>(gridDim.x) * kThreads)
        if (!sequence_rows(c, static_cast<int>(i), p.T, ahead, first, many)) atomicExch(p.status, DADATTN_E_ARG);
    }
    __syncthreads();
    b = before;
    for (int j = 1; j <= at && j < n; ++j) b += later[j];
  }
  // (tokens behind the last sequence and ahead of the first belong to nobody)
  if (at >= n || b >= c.B || (c.starts && t0 + at < c.starts[0])) return;
  int ahead, first, count;
  const int in = sequence_rows(c, b, p.T, ahead, first, count) ? t0 + at - first : -1;
  int page = -1;
  const int row = ahead + in;
  if (in >= 0 && in < count) page = c.table[static_cast<int64_t>(b) * c.max_pages + (row >> c.page_shift)];
  if (page < 0 || page >= c.pages) {
    if (u == 0 && blockIdx.y == 0) atomicExch(p.status, DADATTN_E_ARG);
    return;
  }
  // the heads of this CTA: of q, k or v
  int g = blockIdx.y, which = 0;
  if (g >= p.groups_q) {
    g -= p.groups_q;
    which = 1 + (g >= p.groups_kv);
    if (which == 2) g -= p.groups_kv;
  }
  const int all = which == 0 ? p.heads_q : c.heads, groups = which == 0 ? p.groups_q : p.groups_kv;
  const int head0 = g * all / groups, heads = (g + 1) * all / groups - head0;
  const bool turned = which < 2 && u * kTurnUnit < p.r.rot;
  float2 cs[8];
  if (turned) cos_sin_of<false>(cs, u, row, p.r);
  const int x = which == 2 ? u * kTurnUnit : unit_first(u, p.r), second = which == 2 ? 8 : unit_second(u, p.r);
  const PackedStrides& s = p.from[which];
  const T* from = static_cast<const T*>(which == 0 ? p.q : which == 1 ? p.k : p.v) + (t0 + at) * s.token + head0 * s.head + x;
  int64_t step;
  uint16_t* to;
  if (which == 0) {
    to = p.q_out + (t0 + at) * p.to_q.token + head0 * p.to_q.head;
    step = p.to_q.head;
  } else {
    const int64_t first_row = ((static_cast<int64_t>(page) * c.heads + head0) << c.page_shift) + (row & ((1 << c.page_shift) - 1));
    to = (which == 1 ? p.k_pages : p.v_pages) + first_row * p.D;
    step = static_cast<int64_t>(p.D) << c.page_shift;
  }
  turn_heads<sizeof(T) == 4 ? 2 : 4>(from, s.head, reinterpret_cast<bf16*>(to) + x, step, heads, second, turned, cs,
                                     p.r.interleaved);
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
                                         const uint64_t* turns, float factor, int rot_dim, int interleaved, int new_is_bf16,
                                         dadattn_stream_t stream) {
  const char* name = "paged append";
  if (int rc = check_paged(name, k_pages, v_pages, page_table, lengths, starts, B, Hkv, D, pages, page_size, max_pages)) return rc;
  if (T <= 0 || Hq < 0) return fail(DADATTN_E_ARG, "%s: bad sizes T=%d Hq=%d", name, T, Hq);
  if (!starts && T != B) return fail(DADATTN_E_ARG, "%s: without starts T=%d is B=%d", name, T, B);
  if (int rc = check_rotary(name, turns, factor, rot_dim, D)) return rc;
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
  if (static_cast<long long>(Hq) + 2ll * Hkv > 65535)
    return fail(DADATTN_E_UNSUPPORTED, "%s: Hq=%d and Hkv=%d are too many heads for a call", name, Hq, Hkv);
  AppendParams p = {};
  p.q = q, p.k = k_new, p.v = v_new;
  p.q_out = q_out, p.k_pages = k_pages, p.v_pages = v_pages;
  if (Hq > 0) p.from[0] = PackedStrides{q_strides[0], q_strides[1]}, p.to_q = PackedStrides{q_out_strides[0], q_out_strides[1]};
  p.from[1] = PackedStrides{k_strides[0], k_strides[1]};
  p.from[2] = PackedStrides{v_strides[0], v_strides[1]};
  p.cache = PagedCache{page_table, lengths, starts, B, pages, log2_of(page_size), max_pages, Hkv};
  p.T = T, p.D = D, p.heads_q = Hq, p.units = D / kTurnUnit;
  p.r = RotaryParams{turns, factor, rot_dim, interleaved != 0, 0};
  p.status = device_status_word();
  if (!p.status) return DADATTN_E_CUDA;
  const int tokens = kThreads / p.units, blocks = static_cast<int>((static_cast<long long>(T) + tokens - 1) / tokens);
  // (few groups: each finds its tokens' sequences and pages for itself. With four heads a thread, as in rotary.cu, 14747 tokens of
  // 32 + 16 heads took 69.3 us instead of 60.3, by direct calls.)
  p.groups_q = Hq ? head_groups(blocks, Hq, Hq + 2 * Hkv, 8) : 0;
  p.groups_kv = head_groups(blocks, Hkv, Hq + 2 * Hkv, 8);
  const dim3 grid(blocks, p.groups_q + 2 * p.groups_kv);
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
