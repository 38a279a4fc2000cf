// delta of rows that see few keys, for the windowed backward.
//
// delta_i = dO_i.O_i = sum_j P_ij dP_ij. The first form is what a backward has, from O as the forward rounded it; it is off by
// dO_i times that rounding. dS_ij = P_ij (dP_ij - delta_i) of a row that sees n keys is off by that much in relation to about
// sqrt(n) times as much: by nothing to speak of where n is large, by more than dS's own rounding to bf16 where n is small (and
// with n = 1, where dS is 0, there is nothing else). So rows that see up to kFewKeys form the second sum. These are the first
// rows of a unit, or all of them under a narrow window. Norms of the error of dQ and dK in a model of the arithmetic (48 x 32 x
// 64; one rounding of dS and one of the results make 2.35e-3): 2.65e-3 with the first form for all rows, 2.36e-3 so. Over
// windows from 16 to 70 at most 2.5e-3 with 8 keys, 2.45e-3 with 16, 2.43e-3 with 24, 2.42e-3 with 32.
//
// A warp takes 16 rows: scores and dP by warp-wide matrix instructions, eight keys at a time, operands straight from memory
// (a sum over the head's dimensions may take them in any order, so a thread's are 16 consecutive bytes of a row). The block of a
// tcgen05 product, 128 rows, would be mostly hidden pairs here. Backward with the first rows' sums and without, us: 192 x 1024 x
// 64, window 256, 102.8 / 101.5; 72 x 777 x 64, window 128, 37.0 / 36.3; 24 x 8192 x 128 the same. Where all rows have so few
// keys (192 x 1024 x 64, window 16, 4 first tokens) the kernel ahead of the gradient takes 49 us, 21 without (332 with a lane
// per key, which reads 32 rows side by side). A kernel of its own would add a launch to each backward.
#pragma once

#include <cuda_bf16.h>

#include <cstdint>

#include "sm100_ptx.cuh"

namespace dadattn {

constexpr int kFewKeys = 32;

struct NoRows {};   // a backward without a window
struct FewKeys {
  static constexpr int kThreads = 256;   // of the blocks that take these rows
  const __nv_bfloat16 *q, *k, *v;        // [BH, S, D]
  const float* lse;
  int S, window, sinks, rows;            // rows 0 .. rows - 1 of every unit
  int groups, split;                     // of 16 rows, a unit's; warps that share one (their tiles of keys)
  int64_t first_block, n;                // the kernel's blocks from here on take them, n = BH groups in all
  float scale_log2;
};

// 1 <= window <= S, 0 <= sinks <= S. Row i sees min(i + 1, window) keys and, beyond those, min(sinks, i + 1 - window) first ones.
inline FewKeys few_keys(const uint16_t* q, const uint16_t* k, const uint16_t* v, const float* lse, int BH, int S, float scale,
                        int window, int sinks, int64_t first_block) {
  using BF = __nv_bfloat16;
  const int rows = static_cast<int64_t>(window) + sinks <= kFewKeys || S <= kFewKeys ? S : kFewKeys;
  // All rows: what counts is the work. The first 32: that it is done before the others' blocks are.
  const int groups = (rows + 15) / 16, split = rows > kFewKeys ? 1 : 4;
  return {reinterpret_cast<const BF*>(q), reinterpret_cast<const BF*>(k), reinterpret_cast<const BF*>(v), lse, S, window, sinks,
          rows, groups, split, first_block, static_cast<int64_t>(BH) * groups, scale * 1.4426950408889634f};
}
inline int64_t few_keys_blocks(const FewKeys& f) { return (f.n * f.split * 32 + FewKeys::kThreads - 1) / FewKeys::kThreads; }

namespace {

// c += A B^T: A 16 rows, B 8 rows, 16 of the head's dimensions. Thread (g, t) = (lane / 4, lane % 4) has two words of A's rows g
// and g + 8 and of B's row g, and of c rows g (x, y) and g + 8 (z, w), columns 2t and 2t + 1.
__device__ __forceinline__ void mma_16x8(float4& c, uint32_t a0, uint32_t a0_low, uint32_t a1, uint32_t a1_low, uint32_t b0, uint32_t b1) {
  asm("mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
      : "+f"(c.x), "+f"(c.y), "+f"(c.z), "+f"(c.w)
      : "r"(a0), "r"(a0_low), "r"(a1), "r"(a1_low), "r"(b0), "r"(b1));
}

// By a block of FewKeys::kThreads threads, `block` counted from 0.
template <int D>
__device__ __forceinline__ void few_keys_delta(const FewKeys& f, int64_t block, const __nv_bfloat16* __restrict__ dout,
                                               float* __restrict__ delta) {
  constexpr int kChunks = D / 32;   // 16-byte pieces of a row per thread
  __shared__ float part_sum[FewKeys::kThreads / 32][16];
  const int warp = threadIdx.x / 32, part = warp % f.split;
  const int64_t mine = block * (FewKeys::kThreads / 32 / f.split) + warp / f.split, at = min(mine, f.n - 1);
  const int lane = threadIdx.x % 32, g = lane / 4, t = lane % 4;
  const int64_t unit = at / f.groups, row0 = unit * f.S;
  const int i0 = static_cast<int>(at - unit * f.groups) * 16;
  const int rows[2] = {i0 + g, i0 + g + 8};
  auto piece = [&](const __nv_bfloat16* x, int row, int c) {   // (rows behind the last one: the last; they are not used)
    return reinterpret_cast<const uint4*>(x + (row0 + min(row, f.S - 1)) * D)[t + 4 * c];
  };
  const float neg_lse[2] = {-f.lse[row0 + min(rows[0], f.S - 1)] * 1.4426950408889634f,
                            -f.lse[row0 + min(rows[1], f.S - 1)] * 1.4426950408889634f};
  float sum[2] = {0.f, 0.f};
  auto tile = [&](int k0) {   // keys k0 .. k0 + 7
    float4 s = make_float4(0.f, 0.f, 0.f, 0.f), dp = s;
    auto products = [&](float4& to, const __nv_bfloat16* a, const __nv_bfloat16* b, int c) {
      const uint4 a0 = piece(a, rows[0], c), a1 = piece(a, rows[1], c), x = piece(b, k0 + g, c);
      mma_16x8(to, a0.x, a1.x, a0.y, a1.y, x.x, x.y);
      mma_16x8(to, a0.z, a1.z, a0.w, a1.w, x.z, x.w);
    };
#pragma unroll 2
    for (int c = 0; c < kChunks; ++c) {   // (the rows' own pieces again for every tile: few registers)
      products(s, f.q, f.k, c);
      products(dp, dout, f.v, c);
    }
    const float sc[4] = {s.x, s.y, s.z, s.w}, d[4] = {dp.x, dp.y, dp.z, dp.w};
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      const int i = rows[e / 2], j = k0 + 2 * t + e % 2;
      if (j <= i && (i - j < f.window || j < f.sinks)) sum[e / 2] += ptx::ex2(fmaf(sc[e], f.scale_log2, neg_lse[e / 2])) * d[e];
    }
  };
  // the first keys' tiles, then the window's
  const int from = max(i0 - f.window + 1, 0) / 8 * 8, n_first = (min(f.sinks, from) + 7) / 8;
  const int n_tiles = n_first + (min(i0 + 16, f.S) - from + 7) / 8;
#pragma unroll 1
  for (int n = part; n < n_tiles; n += f.split) tile(n < n_first ? n * 8 : from + (n - n_first) * 8);
#pragma unroll
  for (int h = 0; h < 2; ++h) {
    sum[h] += __shfl_xor_sync(0xffffffffu, sum[h], 1);
    sum[h] += __shfl_xor_sync(0xffffffffu, sum[h], 2);
    if (t == 0) part_sum[warp][g + 8 * h] = sum[h];
  }
  __syncthreads();
  if (part == 0 && lane < 16 && mine < f.n && i0 + lane < f.rows) {
    float all = 0.f;
    for (int j = 0; j < f.split; ++j) all += part_sum[warp + j][lane];
    delta[row0 + i0 + lane] = all;
  }
}

}  // namespace
}  // namespace dadattn
