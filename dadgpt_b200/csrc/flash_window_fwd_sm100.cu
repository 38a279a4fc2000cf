// bf16 causal attention forward with a sliding window and a few first tokens that stay visible, for sm_100a:
// query i sees key j iff j <= i and (i - j < window or j < sinks).
//
//   out_i = sum_j p_ij v_j,  p_ij = exp(scale q_i.k_j - lse_i),  lse_i = ln sum_j exp(scale q_i.k_j)   over the visible j
//
// One CTA per 128 query rows of one (batch, head) goes through the 64-key tiles that any of its rows sees: those of the
// first tokens, then from the one where its first row's window begins to the diagonal. Tiles of 64 keys, not 128: a
// narrow window has few interior tiles, and half a tile less of hidden keys at either end is a third of the work at
// window 128.
//   warp 0      TMA producer: Q once, K and V tiles through a ring
//   warp 1      MMA issuer (one elected lane) and owner of the tensor memory:
//               S = Q K^T (128 x 64 fp32), O += P V with P read back from tensor memory
//   warps 2-5   softmax, one thread per row
// A CTA does six tiles or so, and setting up and ending take as long as four: what counts is that others work meanwhile. So
// an SM holds four CTAs of head size 64: 128 columns of tensor memory, P over S in one score buffer, whose next scores follow
// the product with it, and 80 registers, for which a thread reads half of its scores twice. (Two CTAs with two threads per
// row and two buffers: 46.3 us for 192 x 1024 with window 256, which take 41.) At head size 128 two, whose scores have two buffers: S of the next
// tile is formed while the exponentials of the current one are computed.
// The accumulator is rescaled only when a row's maximum has grown by 2^8 (exact all the same); warps that see nothing of a
// tile store zeros.
// Measured (us): 192 x 1024 x 64, window 256, 4 first tokens 41 (101 MB and 11.4 GFLOP), 72 x 777 x 64, window 128 14,
// 24 x 8192 x 128, window 1024 114 (97 GFLOP: 850 TFLOP/s). No unit is near its limit in either (issue slots 50 %, exp2 41 %,
// tensor pipe 24 % in the first, 40, 48 and 50 % in the last): a tile's steps wait for each other, and a CTA's start and end
// are as long as some tiles. Of six tiles or so of 64 keys a third is hidden in the first case. A window that hides little is
// better taken by the causal kernels, to which nothing here turns: 192 x 1024 x 64 60 us with a window of 1024 and 46 there,
// 53 with 512; 24 x 8192 x 128 413 and 409.
// Every wait is bounded (sm100_ptx.cuh). Barriers as in flash_bf16_sm100.cu.
#include <cuda_bf16.h>

#include <cfloat>

#include "common.cuh"
#include "sm100_ptx.cuh"

namespace dadattn {
namespace {

using namespace ptx;

// (four polls ahead of the suspending wait: 1 %)
#define window_wait(bar, parity, abort_flag) mbar_wait_at<4>(bar, parity, abort_flag, __LINE__)

constexpr int kBM = 128;                   // query rows per CTA
constexpr int kBN = 64;                    // keys per tile
constexpr int kPanelBytes = kBM * 128;     // [128 rows][64 bf16], swizzled
constexpr int kSubPanelBytes = kBN * 128;  // [64 rows][64 bf16]
constexpr float kLog2e = 1.4426950408889634f;
constexpr float kLn2 = 0.6931471805599453f;
constexpr float kRescaleThreshold = 8.0f;  // log2 units: P stays below 2^8

template <int D>
struct WindowFwd {
  static constexpr int kPanels = D / 64;
  static constexpr int kBufs = D == 64 ? 1 : 2;            // score buffers
  static constexpr int kPerSm = D == 64 ? 4 : 2;           // CTAs
  static constexpr int kSoftmax = kBM;
  static constexpr int kThreads = 64 + kSoftmax;
  static constexpr int kStages = 2;                        // K / V ring depth
  static constexpr int kTile = kPanels * kSubPanelBytes;   // a [64, D] tile
  static constexpr int kQ = 0;
  static constexpr int kK = kQ + kPanels * kPanelBytes;
  static constexpr int kV = kK + kStages * kTile;
  static constexpr int kBars = kV + kStages * kTile;
  static constexpr int kBytes = kBars + 256;
  static constexpr uint32_t kColS = 0, kColO = kBufs * kBN, kTmemCols = kColO + D;
  static_assert(kTmemCols * kPerSm <= 512 && kPerSm * (kBytes + 1024) <= 228 * 1024, "the CTAs of an SM");
};

struct WindowBars {
  uint64_t q_full, k_full[2], v_full[2], k_empty[2], v_empty[2];
  uint64_t s_full[2], p_full[2], o_done[2], settled;
  uint32_t tmem_base;
  int abort_flag;
};
static_assert(sizeof(WindowBars) <= 256, "barrier block");

// The lowest n bits
__device__ __forceinline__ uint32_t low_bits(int n) { return n <= 0 ? 0u : n >= 32 ? 0xffffffffu : (1u << n) - 1u; }

template <int D>
__global__ void __launch_bounds__(WindowFwd<D>::kThreads, WindowFwd<D>::kPerSm)
flash_window_fwd_kernel(const __grid_constant__ CUtensorMap map_q, const __grid_constant__ CUtensorMap map_k,
                        const __grid_constant__ CUtensorMap map_v, const __grid_constant__ CUtensorMap map_out,
                        float* __restrict__ lse, int S, float scale, int window, int sinks, LeveledGrid order,
                        int* __restrict__ status) {
  using L = WindowFwd<D>;
  constexpr int kStages = L::kStages, kBufs = L::kBufs;
  extern __shared__ __align__(1024) uint8_t smem[];
  WindowBars* bars = reinterpret_cast<WindowBars*>(smem + L::kBars);
  volatile int* abort_flag = &bars->abort_flag;

  const int warp = threadIdx.x / 32, lane = threadIdx.x % 32;
  int level, bh;
  if (!leveled_block(order, level, bh)) return;
  const int q0 = ((S + kBM - 1) / kBM - 1 - level) * kBM;
  // key tiles: n_first of the first tokens, then those from `from` to the diagonal (1 <= window <= S)
  int from = max(q0 - window + 1, 0) / kBN;
  int n_first = (min(sinks, q0 + kBM) + kBN - 1) / kBN;
  if (n_first >= from) n_first = from = 0;   // no gap between them
  const int last = (min(q0 + kBM, S) - 1) / kBN, n = n_first + last - from + 1;
  auto tile_at = [&](int j) { return j < n_first ? j : from + j - n_first; };

  if ((smem_u32(smem) & 1023u) != 0) {  // the swizzled layouts need a 1024-byte aligned base
    if (threadIdx.x == 0) atomicExch(status, DADATTN_E_CUDA);
    return;
  }
  // The tiles of the ring's stage s, by the producing thread
  auto load_k = [&](int s, int j) {
    mbar_arrive_expect_tx(&bars->k_full[s], L::kTile);
    for (int p = 0; p < L::kPanels; ++p)
      tma_load_3d(smem + L::kK + s * L::kTile + p * kSubPanelBytes, &map_k, &bars->k_full[s], p * 64, tile_at(j) * kBN, bh);
  };
  auto load_v = [&](int s, int j) {
    mbar_arrive_expect_tx(&bars->v_full[s], L::kTile);
    for (int p = 0; p < L::kPanels; ++p)
      tma_load_3d(smem + L::kV + s * L::kTile + p * kSubPanelBytes, &map_v, &bars->v_full[s], p * 64, tile_at(j) * kBN, bh);
  };
  if (threadIdx.x == 0) {
    prefetch_tensormap(&map_q);
    prefetch_tensormap(&map_k);
    prefetch_tensormap(&map_v);
    prefetch_tensormap(&map_out);
    mbar_init(&bars->q_full, 1);
    for (int s = 0; s < kStages; ++s) {
      mbar_init(&bars->k_full[s], 1);
      mbar_init(&bars->v_full[s], 1);
      mbar_init(&bars->k_empty[s], 1);
      mbar_init(&bars->v_empty[s], 1);
    }
    for (int b = 0; b < 2; ++b) {
      mbar_init(&bars->s_full[b], 1);
      mbar_init(&bars->p_full[b], L::kSoftmax);
      mbar_init(&bars->o_done[b], 1);
    }
    mbar_init(&bars->settled, 1);
    bars->abort_flag = 0;
    fence_mbar_init();
    // the first tiles need this thread's barriers and nothing of what the others set up
    pdl_wait();
    mbar_arrive_expect_tx(&bars->q_full, L::kPanels * kPanelBytes);
    for (int p = 0; p < L::kPanels; ++p)
      tma_load_3d(smem + L::kQ + p * kPanelBytes, &map_q, &bars->q_full, p * 64, q0, bh);
    load_k(0, 0);
    load_v(0, 0);
  }
  __syncwarp();
  if (warp == 1) {
    tmem_alloc(&bars->tmem_base, L::kTmemCols);
    tmem_relinquish();
  }
  tc_fence_before_sync();
  __syncthreads();
  tc_fence_after_sync();
  const uint32_t tmem = bars->tmem_base;
  pdl_wait();
  pdl_launch_dependents();

  if (warp == 0) {
    // ------------------------------ TMA producer ------------------------------
    if (lane == 0) {
      int n_k = 1, n_v = 1;   // tiles loaded
      for (int j = 1; j < n; ++j) {
        const int s = j % kStages, use = j / kStages;
        if (use > 0 && !window_wait(&bars->k_empty[s], (use - 1) & 1, abort_flag)) break;
        load_k(s, j);
        ++n_k;
        if (use > 0 && !window_wait(&bars->v_empty[s], (use - 1) & 1, abort_flag)) break;
        load_v(s, j);
        ++n_v;
      }
      settle(&bars->q_full, 0);
      settle_ring(bars->k_full, kStages, n_k);
      settle_ring(bars->v_full, kStages, n_v);
    }
  } else if (warp == 1) {
    // ------------------------------ MMA issuer ------------------------------
    if (elect_one()) {
      constexpr uint32_t idesc_s = make_idesc_bf16(kBM, kBN, 0, 0);  // Q, K: K-major
      constexpr uint32_t idesc_o = make_idesc_bf16(kBM, D, 0, 1);    // P K-major, V MN-major
      const SmemDescBase q_desc = make_desc_base_sw128(smem_u32(smem + L::kQ), 0);
      const SmemDescBase k_desc0 = make_desc_base_sw128(smem_u32(smem + L::kK), 0);
      const SmemDescBase v_desc0 = make_desc_base_sw128(smem_u32(smem + L::kV), kSubPanelBytes);
      bool ok = window_wait(&bars->q_full, 0, abort_flag);

      // O (+)= P_i V_i
      auto issue_pv = [&](int i) -> bool {
        const int s = i % kStages, buf = i % kBufs;
        if (!window_wait(&bars->v_full[s], (i / kStages) & 1, abort_flag)) return false;
        if (!window_wait(&bars->p_full[buf], (i / kBufs) & 1, abort_flag)) return false;
        tc_fence_after_sync();
        const SmemDescBase v_desc{v_desc0.lo + s * (L::kTile >> 4), v_desc0.hi};
#pragma unroll
        for (int kk = 0; kk < kBN / 16; ++kk)
          mma_ts(tmem + L::kColO, tmem + L::kColS + buf * kBN + kk * 8, desc_at(v_desc, kk * 2048), idesc_o, (i > 0 || kk > 0) ? 1u : 0u);
        mma_commit(&bars->v_empty[s]);
        mma_commit(&bars->o_done[i & 1]);
        return true;
      };

      for (int j = 0; ok && j < n; ++j) {
        const int s = j % kStages, buf = j % kBufs;
        // Two buffers: S_j goes over P_{j-2}, behind P_{j-2} V_{j-2}, which this thread issued earlier, and ahead of
        // P_{j-1} V_{j-1}. One: behind P_{j-1} V_{j-1}.
        if (kBufs == 1 && j > 0 && !(ok = issue_pv(j - 1))) break;
        if (!(ok = window_wait(&bars->k_full[s], (j / kStages) & 1, abort_flag))) break;
        tc_fence_after_sync();
        const SmemDescBase k_desc{k_desc0.lo + s * (L::kTile >> 4), k_desc0.hi};
#pragma unroll
        for (int kk = 0; kk < D / 16; ++kk)
          mma_ss(tmem + L::kColS + buf * kBN, desc_at(q_desc, (kk / 4) * kPanelBytes + (kk % 4) * 32),
                 desc_at(k_desc, (kk / 4) * kSubPanelBytes + (kk % 4) * 32), idesc_s, kk > 0 ? 1u : 0u);
        mma_commit(&bars->k_empty[s]);
        mma_commit(&bars->s_full[buf]);
        if (kBufs == 2 && j > 0) ok = issue_pv(j - 1);
      }
      if (ok) issue_pv(n - 1);
      settle_products(&bars->settled);
    }
  } else {
    // ------------------------------ softmax ------------------------------
    const int quad = warp % 4;                 // TMEM lane quadrant this warp may touch
    const int row = quad * 32 + lane, r = q0 + row;
    const uint32_t tlane = tmem + (static_cast<uint32_t>(quad * 32) << 16);
    const uint32_t tO = tlane + L::kColO;
    const float scale_log2 = scale * kLog2e;
    auto wait_pv = [&](int i) { return window_wait(&bars->o_done[i & 1], (i >> 1) & 1, abort_flag); };
    float m = -INFINITY, l = 0.f;   // running max (log2 units, scaled) and sum
    bool ok = true;

    for (int j = 0; j < n; ++j) {
      const int buf = j % kBufs, t0 = tile_at(j) * kBN;
      const uint32_t tS = tlane + L::kColS + buf * kBN;
      // tiles in which any row of the CTA does not see a key: across the diagonal, or across the window's beginning
      const bool edge = t0 + kBN - 1 > q0 || (t0 <= q0 + kBM - 1 - window && t0 + kBN > sinks);
      uint32_t seen[2] = {0xffffffffu, 0xffffffffu};
      bool any = true, masked = false;   // whether the warp's rows see anything, and not everything
      if (edge) {
#pragma unroll
        for (int w = 0; w < 2; ++w) {
          const int c = t0 + 32 * w;
          seen[w] = low_bits(r - c + 1) & (~low_bits(r - window - c + 1) | low_bits(sinks - c));
        }
        any = __any_sync(0xffffffffu, (seen[0] | seen[1]) != 0);
        masked = __any_sync(0xffffffffu, (seen[0] & seen[1]) != 0xffffffffu);
      }
      // 32 of the thread's scores
      auto load = [&](uint32_t (&x)[32], int w) {
        tmem_ld32(tS + 32 * w, x);
        tmem_wait_ld();
        if (masked) {
#pragma unroll
          for (int i = 0; i < 32; ++i)
            if (!(seen[w] >> i & 1u)) x[i] = 0xff800000u;   // -inf
        }
      };
      // max of the raw scores (scale > 0 commutes with max)
      auto most_of = [&](const uint32_t (&x)[32], float most) -> float {
        float mx[4] = {most, -INFINITY, -INFINITY, -INFINITY};
#pragma unroll
        for (int i = 0; i < 32; i += 2) mx[(i >> 1) & 3] = fmax3(mx[(i >> 1) & 3], __uint_as_float(x[i]), __uint_as_float(x[i + 1]));
        return fmaxf(fmaxf(mx[0], mx[1]), fmaxf(mx[2], mx[3]));
      };
      if (!(ok = window_wait(&bars->s_full[buf], (j / kBufs) & 1, abort_flag))) break;
      tc_fence_after_sync();
      if (any) {
        uint32_t xa[32], xb[32];
        load(xa, 0);
        float mx = most_of(xa, -INFINITY);
        load(xb, 1);
        mx = __fmul_rn(most_of(xb, mx), scale_log2);
        if (j == 0) {
          m = mx;   // O is first written by an MMA with accumulate = 0: nothing to rescale
        } else if (__any_sync(0xffffffffu, mx > m + kRescaleThreshold)) {
          if (!(ok = wait_pv(j - 1))) break;
          tc_fence_after_sync();
          const float m_new = fmaxf(m, mx);
          // m = -inf: nothing but zeros has been accumulated so far
          const float corr = (m == -INFINITY) ? 0.f : ex2(m - m_new);
#pragma unroll 1
          for (int c = 0; c < D / 16; ++c) {
            uint32_t o[16];
            tmem_ld16(tO + c * 16, o);
            tmem_wait_ld();
#pragma unroll
            for (int i = 0; i < 16; ++i) o[i] = __float_as_uint(__uint_as_float(o[i]) * corr);
            tmem_st16(tO + c * 16, o);
          }
          tmem_wait_st();
          l = __fmul_rn(l, corr);
          m = m_new;
        }
        // p = exp2(s scale log2e - m). A row that has seen no key yet has m = -inf: its scores are all -inf and must give
        // p = 0, not exp2(nan).
        float2 sum2[2] = {make_float2(0.f, 0.f), make_float2(0.f, 0.f)};
        const float2 sl = make_float2(scale_log2, scale_log2);
        const float neg_m = (m == -INFINITY) ? 0.f : -m;
        const float2 nm = make_float2(neg_m, neg_m);
        auto weights = [&](const uint32_t (&x)[32], uint32_t (&pk)[16]) {   // packed P
#pragma unroll
          for (int i = 0; i < 32; i += 2) {
            const float2 e = ffma2(make_float2(__uint_as_float(x[i]), __uint_as_float(x[i + 1])), sl, nm);
            const float2 p = make_float2(ex2(e.x), ex2(e.y));
            sum2[(i >> 1) & 1] = fadd2(sum2[(i >> 1) & 1], p);
            pk[i / 2] = pack_bf16(p.x, p.y);
          }
        };
        // P goes over S, into its first 32 columns: the second half's scores are read by then, the first half's, where
        // registers do not hold both, a second time
        uint32_t pa[16], pb[16];
        weights(xb, pb);
        if (kBufs == 1) load(xa, 0);
        weights(xa, pa);
        l += (sum2[0].x + sum2[1].x) + (sum2[0].y + sum2[1].y);
        tmem_st16(tS, pa);
        tmem_st16(tS + 16, pb);
      } else {
        uint32_t none[16];
#pragma unroll
        for (int i = 0; i < 16; ++i) none[i] = 0u;
        tmem_st16(tS, none);
        tmem_st16(tS + 16, none);
      }
      tmem_wait_st();
      tc_fence_before_sync();
      mbar_arrive(&bars->p_full[buf]);
    }

    // out = O / l; lse in natural-log units of the scaled scores. Results leave through the Q tile, which every product has
    // read, and TMA.
    if (ok && wait_pv(n - 1)) {
      tc_fence_after_sync();
      const float f = 1.f / l;   // (a row sees its own key)
      uint8_t* stage = smem + L::kQ + quad * 32 * 128;
#pragma unroll
      for (int c = 0; c < D / 32; ++c) {
        uint32_t o[32];
        tmem_ld32(tO + c * 32, o);
        tmem_wait_ld();
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          float y[8];
#pragma unroll
          for (int e = 0; e < 8; ++e) y[e] = __uint_as_float(o[8 * i + e]) * f;
          *reinterpret_cast<uint4*>(stage + (c / 2) * kPanelBytes + lane * 128 + ((((c & 1) * 4 + i) ^ (lane & 7)) << 4)) =
              make_uint4(pack_bf16(y[0], y[1]), pack_bf16(y[2], y[3]), pack_bf16(y[4], y[5]), pack_bf16(y[6], y[7]));
        }
      }
      fence_proxy_async_smem();
      __syncwarp();
      if (lane == 0 && q0 + quad * 32 < S) {   // (rows beyond S are not written)
        for (int p = 0; p < L::kPanels; ++p) tma_store_3d(&map_out, stage + p * kPanelBytes, p * 64, q0 + quad * 32, bh);
        bulk_commit();
      }
      if (r < S) lse[static_cast<size_t>(bh) * S + r] = (m + log2f(l)) * kLn2;
      if (lane == 0) bulk_wait_read<0>();
    }
  }

  // ------------------------------ common exit ------------------------------
  tc_fence_before_sync();
  __syncthreads();
  if (warp == 1) {
    __syncwarp();
    tc_fence_after_sync();
    tmem_dealloc(tmem, L::kTmemCols);
  }
  if (threadIdx.x == 0 && bars->abort_flag) report_timeout(status, bars->abort_flag);
}

template <int D>
int launch_window_fwd(uint16_t* out, float* lse, const uint16_t* q, const uint16_t* k, const uint16_t* v, int BH, int S,
                      float scale, int window, int sinks, cudaStream_t st) {
  using L = WindowFwd<D>;
  CUtensorMap mq, mk, mv, mo;
  if (int rc = make_tensor_map_bf16(&mq, q, BH, S, D, kBM)) return rc;
  if (int rc = make_tensor_map_bf16(&mk, k, BH, S, D, kBN)) return rc;
  if (int rc = make_tensor_map_bf16(&mv, v, BH, S, D, kBN)) return rc;
  if (int rc = make_tensor_map_bf16(&mo, out, BH, S, D, 32)) return rc;
  int* status = device_status_word();
  if (!status) return DADATTN_E_CUDA;
  auto kern = flash_window_fwd_kernel<D>;
  DAD_CUDA(cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, L::kBytes));
  const LeveledGrid order = leveled_grid(32768, S, BH);
  DAD_CUDA(launch_pdl(kern, leveled_blocks(order, (S + kBM - 1) / kBM), dim3(L::kThreads), L::kBytes, st, mq, mk, mv, mo,
                      lse, S, scale, window, sinks, order, status));
  return DADATTN_OK;
}

int check_window(const char* name, std::initializer_list<const void*> tensors, int BH, int S, int D, float scale, int window,
                 int sinks) {
  for (const void* x : tensors)
    if (!x) return fail(DADATTN_E_ARG, "%s: null tensor pointer", name);
  if (BH <= 0 || S <= 0) return fail(DADATTN_E_ARG, "%s: BH=%d and S=%d must be positive", name, BH, S);
  if (BH > 65535) return fail(DADATTN_E_UNSUPPORTED, "%s: BH=%d exceeds 65535 per call", name, BH);
  if (S > DADATTN_MAX_CACHE_LEN) return fail(DADATTN_E_UNSUPPORTED, "%s: S=%d exceeds %d", name, S, DADATTN_MAX_CACHE_LEN);
  if (!dadattn_flash_bf16_supported(D)) return fail(DADATTN_E_UNSUPPORTED, "%s: unsupported d_head %d", name, D);
  if (!(scale > 0.0f && scale < INFINITY)) return fail(DADATTN_E_ARG, "%s: scale must be positive and finite", name);
  if (window < 0 || sinks < 0) return fail(DADATTN_E_ARG, "%s: window %d and sinks %d must not be negative", name, window, sinks);
  for (const void* x : tensors)
    if (!aligned(x, 16)) return fail(DADATTN_E_ARG, "%s: tensors and workspace must be 16-byte aligned", name);
  return DADATTN_OK;
}

// Neither says more than S keys; a window of 0 is one of S.
int within(int keys, int S) { return keys < S ? keys : S; }

}  // namespace
}  // namespace dadattn

using namespace dadattn;

extern "C" int dadattn_flash_fwd_bf16_window(uint16_t* out, float* lse, const uint16_t* q, const uint16_t* k,
                                             const uint16_t* v, int BH, int S, int D, float scale, int window, int sinks,
                                             dadattn_stream_t stream) {
  if (int rc = check_window("windowed forward", {out, q, k, v}, BH, S, D, scale, window, sinks)) return rc;
  if (!lse || !aligned(lse, 4)) return fail(DADATTN_E_ARG, "windowed forward: lse must be a 4-byte aligned device pointer");
  auto* launch = D == 64 ? launch_window_fwd<64> : launch_window_fwd<128>;
  return launch(out, lse, q, k, v, BH, S, scale, window == 0 ? S : within(window, S), within(sinks, S),
                static_cast<cudaStream_t>(stream));
}

extern "C" size_t dadattn_flash_bwd_bf16_window_workspace_bytes(int BH, int S, int D) {
  return dadattn_flash_bwd_bf16_workspace_bytes(BH, S, D);
}

extern "C" int dadattn_flash_bwd_bf16_window(uint16_t* dq, uint16_t* dk, uint16_t* dv, void* workspace,
                                             size_t workspace_bytes, const uint16_t* dout, const uint16_t* out,
                                             const float* lse, const uint16_t* q, const uint16_t* k, const uint16_t* v,
                                             int BH, int S, int D, float scale, int window, int sinks,
                                             dadattn_stream_t stream) {
  if (int rc = check_window("windowed backward", {dq, dk, dv, workspace, dout, out, q, k, v}, BH, S, D, scale, window, sinks))
    return rc;
  if (!lse || !aligned(lse, 4)) return fail(DADATTN_E_ARG, "windowed backward: lse must be a 4-byte aligned device pointer");
  if (!bwd_single_pass())
    return fail(DADATTN_E_UNSUPPORTED, "windowed backward: taken by the single-pass backward only (dadattn_set_bwd_deterministic(0))");
  if (!aligned(workspace, 256)) return fail(DADATTN_E_ARG, "windowed backward: workspace must be 256-byte aligned");
  const size_t need = dadattn_flash_bwd_bf16_window_workspace_bytes(BH, S, D);
  if (workspace_bytes < need)
    return fail(DADATTN_E_WORKSPACE, "windowed backward: workspace %zu < %zu bytes", workspace_bytes, need);
  auto* launch = D == 64 ? launch_bwd_window_d64 : launch_bwd_window_d128;
  return launch(dq, dk, dv, workspace, dout, out, lse, q, k, v, BH, S, scale, window == 0 ? S : within(window, S),
                within(sinks, S), static_cast<cudaStream_t>(stream));
}
