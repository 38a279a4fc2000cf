// A KV cache in pages: k, v [pages, heads, page_size, D] bf16. Row j of sequence b is row j % page_size of page
// page_table[b, j / page_size]. lengths[b] rows are there ahead of a call, whose new tokens lie packed: sequence b's are rows
// starts[b] .. starts[b + 1] - 1 of [T, heads, D], and are its rows lengths[b] and on.
#pragma once

#include "common.cuh"

namespace dadattn {

constexpr int kMinPage = 16, kMaxPage = 1024;

struct PagedCache {
  const int32_t* table;     // [B, max_pages]
  const int32_t* lengths;   // [B]
  const int32_t* starts;    // [B + 1], or null: one token for each sequence
  int B, pages, page_shift, max_pages, heads;
};

inline int log2_of(int x) {
  int n = 0;
  while ((1 << n) < x) ++n;
  return n;
}

// What every call on such a cache checks of it.
inline int check_paged(const char* name, const void* k, const void* v, const int32_t* table, const int32_t* lengths,
                       const int32_t* starts, int B, int heads, int D, int pages, int page_size, int max_pages) {
  if (!k || !v || !table || !lengths) return fail(DADATTN_E_ARG, "%s: null pointer", name);
  if (B <= 0 || heads <= 0 || pages <= 0 || max_pages <= 0)
    return fail(DADATTN_E_ARG, "%s: bad sizes B=%d heads=%d pages=%d max_pages=%d", name, B, heads, pages, max_pages);
  if (D != 64 && D != 128) return fail(DADATTN_E_UNSUPPORTED, "%s: unsupported D %d", name, D);
  if (page_size < kMinPage || page_size > kMaxPage || (page_size & (page_size - 1)))
    return fail(DADATTN_E_UNSUPPORTED, "%s: unsupported page size %d (a power of two from %d to %d)", name, page_size, kMinPage,
                kMaxPage);
  if (static_cast<long long>(max_pages) * page_size > DADATTN_MAX_CACHE_LEN)
    return fail(DADATTN_E_UNSUPPORTED, "%s: max_pages=%d of %d rows exceed %d", name, max_pages, page_size, DADATTN_MAX_CACHE_LEN);
  if (static_cast<long long>(pages) * heads > 0x7fffffffll / page_size)   // rows have 32-bit coordinates
    return fail(DADATTN_E_UNSUPPORTED, "%s: %d pages of %d heads and %d rows are too many", name, pages, heads, page_size);
  if (!aligned(k, 16) || !aligned(v, 16)) return fail(DADATTN_E_ARG, "%s: the pages must be 16-byte aligned", name);
  if (!aligned(table, 4) || !aligned(lengths, 4) || !aligned(starts, 4))
    return fail(DADATTN_E_ARG, "%s: page_table, lengths and starts must be 4-byte aligned", name);
  return DADATTN_OK;
}

// Strides (token, head) in elements of a packed [T, heads, D] tensor.
inline int check_packed(const char* name, const void* p, const int64_t* s, int64_t piece, bool written, int T, int heads) {
  if (!p || !s) return fail(DADATTN_E_ARG, "%s: null pointer", name);
  if (!aligned(p, 16) || s[0] % piece || s[1] % piece)
    return fail(DADATTN_E_ARG, "%s: rows must begin at multiples of 16 bytes (pointers and strides)", name);
  if (s[0] < 0 || s[1] < 0) return fail(DADATTN_E_ARG, "%s: strides must not be negative", name);
  if (written && ((T > 1 && s[0] == 0) || (heads > 1 && s[1] == 0)))
    return fail(DADATTN_E_ARG, "%s: the results' rows must not lie over each other", name);
  return DADATTN_OK;
}

#ifdef __CUDACC__
// Rows that sequence b has ahead of the call and brings, by its own numbers; false: not those of a sequence of this cache.
__device__ __forceinline__ bool sequence_rows(const PagedCache& c, int b, int T, int& ahead, int& first, int& count) {
  first = c.starts ? c.starts[b] : b;
  const int end = c.starts ? c.starts[b + 1] : b + 1;
  ahead = c.lengths[b];
  count = end - first;
  if (first < 0 || end < first || end > T) return false;
  return ahead >= 0 && static_cast<int64_t>(ahead) + count <= static_cast<int64_t>(c.max_pages) << c.page_shift;
}
#endif

}  // namespace dadattn
