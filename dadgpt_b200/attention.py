"""Host-side mirror of DadGPT's fused-attention interface (reference cuda/gpu_ops.cuh:112-122).

Function names, argument order and meaning follow the reference; torch tensors stand in for its
raw device pointers, and the current torch CUDA stream for its default stream. Every function
enqueues the library's kernels and returns without synchronising, as the reference does. Errors
raise (the reference throws std::runtime_error / std::out_of_range).
"""
from __future__ import annotations

import math

import torch

from . import _lib
from ._lib import native as _native


def _ptr(t: torch.Tensor | None) -> int | None:
    return None if t is None else t.data_ptr()


def _stream() -> int:
    return torch.cuda.current_stream().cuda_stream


def _need(t: torch.Tensor, dtype, shape=None, name="tensor"):
    if not t.is_cuda:
        raise ValueError(f"{name} must be a CUDA tensor (there is no CPU path)")
    if t.dtype != dtype or not t.is_contiguous():
        raise ValueError(f"{name} must be contiguous {dtype}, got {t.dtype} contiguous={t.is_contiguous()}")
    if shape is not None and tuple(t.shape) != tuple(shape):
        raise ValueError(f"{name} has shape {tuple(t.shape)}, expected {tuple(shape)}")


def gpu_flash_attention_supported(d_head: int) -> bool:
    """reference cuda/attention.cu:232 — true for head sizes 32 and 64."""
    return d_head in (32, 64)


def gpu_flash_attention_forward(out, lse, q, k, v, BH, S, d_head, scale, *, rate=0.0, seed=0,
                                offset=0, unit0=0):
    """fp32 fused causal attention forward (reference cuda/attention.cu:234-239).

    out,q,k,v: [BH,S,d_head] fp32; lse: [BH,S] fp32. Keyword arguments add the
    attention-probability dropout of the reference's materialized branch (src/model.cpp:406-415).
    """
    _native().fwd_f32(out, lse, q, k, v, BH, S, d_head, scale, rate, seed, offset, unit0)


def gpu_flash_attention_backward(dq, dk, dv, delta, dout, out, lse, q, k, v, BH, S, d_head,
                                 scale, *, rate=0.0, seed=0, offset=0, unit0=0):
    """fp32 fused backward; writes dq, dk, dv (reference cuda/attention.cu:241-252)."""
    _native().bwd_f32(dq, dk, dv, delta, dout, out, lse, q, k, v, BH, S, d_head, scale, rate, seed, offset, unit0)


def gpu_flash_attention_forward_bf16(out, lse, q, k, v, BH, S, d_head, scale, *, rate=0.0,
                                     seed=0, offset=0, unit0=0, mask_bits=None):
    """bf16 tensor-core forward (tcgen05); same argument order as the fp32 call. With
    ``mask_bits`` (from :func:`dropout_mask_bits`) the dropout mask is read, not drawn."""
    _native().fwd_bf16(out, lse, q, k, v, BH, S, d_head, scale, rate, seed, offset, unit0, mask_bits)


def dropout_mask_bits(BH, S, rate, seed, offset=0, unit0=0, out=None):
    """Bit-packed keep mask of the reference's attention dropout (cuda/gpu_ops.cu:712-734 drawn
    per probability, here packed per 128 x 128 tile of the causal lower triangle) for the
    ``mask_bits`` argument of the bf16 calls below. Returns the int32 device tensor."""
    if out is None:
        nbytes = int(_lib.load().dadattn_dropout_mask_bits_bytes(BH, S))
        out = torch.empty(nbytes // 4, dtype=torch.int32, device="cuda")
    _native().mask_bits(out, BH, S, rate, seed, offset, unit0)
    return out


def flash_backward_bf16_workspace_bytes(BH, S, d_head) -> int:
    return int(_lib.load().dadattn_flash_bwd_bf16_workspace_bytes(BH, S, d_head))


def gpu_flash_attention_backward_bf16(dq, dk, dv, workspace, dout, out, lse, q, k, v, BH, S,
                                      d_head, scale, *, rate=0.0, seed=0, offset=0, unit0=0,
                                      mask_bits=None):
    """bf16 tensor-core backward; ``workspace`` replaces the fp32 call's ``delta`` scratch. With
    ``mask_bits`` (from :func:`dropout_mask_bits`) the dropout mask is read, not drawn."""
    _native().bwd_bf16(dq, dk, dv, workspace, dout, out, lse, q, k, v, BH, S, d_head, scale, rate, seed, offset,
                       unit0, mask_bits)


def gpu_flash_attention_forward_bf16_interleaved(out, lse, q, k, v, B, H, S, d_head, scale, *, rate=0.0,
                                                 seed=0, offset=0, unit0=0):
    """bf16 forward on the activations as the projections leave them, [B*S, H*d_head] (reference
    src/model.cpp:372-387): no gpu_split_heads / gpu_merge_heads copies around the call."""
    _native().fwd_bf16_strided(out, lse, q, k, v, B, H, S, d_head, scale, rate, seed, offset, unit0)


def gpu_flash_attention_backward_bf16_interleaved(dq, dk, dv, workspace, dout, out, lse, q, k, v, B, H, S,
                                                  d_head, scale, *, rate=0.0, seed=0, offset=0, unit0=0):
    """Backward of the call above; every bf16 tensor is [B*S, H*d_head]."""
    _native().bwd_bf16_strided(dq, dk, dv, workspace, dout, out, lse, q, k, v, B, H, S, d_head, scale, rate, seed,
                               offset, unit0)


def gpu_flash_attention_forward_bf16_window(out, lse, q, k, v, BH, S, d_head, scale, window, sinks=0):
    """bf16 forward with a sliding window: query i sees key j <= i iff i - j < window or j < sinks (window = 0: every
    j <= i). Arguments as in :func:`gpu_flash_attention_forward_bf16`; head sizes 64 and 128."""
    _native().fwd_bf16_window(BH, S, d_head, scale, window, sinks, out, lse, q, k, v)


def flash_backward_bf16_window_workspace_bytes(BH, S, d_head) -> int:
    return int(_lib.load().dadattn_flash_bwd_bf16_window_workspace_bytes(BH, S, d_head))


def gpu_flash_attention_backward_bf16_window(dq, dk, dv, workspace, dout, out, lse, q, k, v, BH, S, d_head, scale,
                                             window, sinks=0):
    """Backward of the call above, with its ``window`` and ``sinks``."""
    _native().bwd_bf16_window(BH, S, d_head, scale, window, sinks, dq, dk, dv, workspace, dout, out, lse, q, k, v)


def flash_f32_via_bf16_workspace_bytes(BH, S, d_head) -> int:
    return int(_lib.load().dadattn_flash_f32_via_bf16_workspace_bytes(BH, S, d_head))


def gpu_flash_attention_forward_via_bf16(out, lse, q, k, v, BH, S, d_head, scale, workspace):
    """fp32 tensors, bf16 tensor-core arithmetic: what the reference's fp32 signature
    (cuda/attention.cu:234-239) computes when its GEMM precision is BF16 (cuda/gpu_ops.cuh:43-44)."""
    _native().fwd_via_bf16(out, lse, q, k, v, BH, S, d_head, scale, workspace)


def gpu_flash_attention_backward_via_bf16(dq, dk, dv, dout, out, lse, q, k, v, BH, S, d_head, scale,
                                          workspace):
    """Backward of the call above (reference cuda/attention.cu:241-252; no ``delta`` argument:
    the workspace holds it)."""
    _native().bwd_via_bf16(dq, dk, dv, dout, out, lse, q, k, v, BH, S, d_head, scale, workspace)


def set_backward_deterministic(on: bool) -> None:
    """Head size 64: choose between the single-pass backward (default; dQ summed across key tiles
    in arrival order, so its last bits may vary between runs) and the two-kernel backward that,
    like the reference, accumulates nothing across thread blocks."""
    _lib.check(_lib.load().dadattn_set_bwd_deterministic(1 if on else 0))


def dropout_mask(mask: torch.Tensor, rate: float, seed: int, offset: int = 0, first: int = 0):
    """Fill ``mask`` (uint8, flat) with the reference's keep(1)/drop(0) mask
    (reference cuda/gpu_ops.cu:712-734) for elements first .. first+numel-1."""
    _need(mask, torch.uint8, None, "mask")
    _lib.check(_lib.load().dadattn_dropout_mask(_ptr(mask), mask.numel(), rate, seed, offset,
                                                first, _stream()))


def decode_attention_f32(out, q, k_new, v_new, k_cache, v_cache, pos, scale):
    """Attention part of model_forward_cached (reference src/model.cpp:745-790) for one sequence:
    caches [H,max_len,D] fp32, q/k_new/v_new/out [H*D]. Raises IndexError when pos is outside
    the cache (the reference throws std::out_of_range, src/model.cpp:693-696)."""
    _native().decode_f32(out, q, k_new, v_new, k_cache, v_cache, pos, scale)


class KVCacheBF16:
    """Batched counterpart of the reference's ``struct KVCache`` (src/model.hpp:140-152) for one
    layer: k, v [B,H,max_len,D] bf16, per-sequence lengths on the device, the decode kernel's workspace.
    With ``weights``, also the rows' accumulated attention weights [B,H,max_len] fp32, which
    :func:`decode_attention_bf16_window` adds up and :func:`kv_cache_evict_bf16` goes by."""

    def __init__(self, B, H, max_len, D, device="cuda", weights=False):
        self.B, self.H, self.max_len, self.D = B, H, max_len, D
        self.k = torch.zeros(B, H, max_len, D, dtype=torch.bfloat16, device=device)
        self.v = torch.zeros_like(self.k)
        self.lengths = torch.zeros(B, dtype=torch.int32, device=device)
        self.weights = torch.zeros(B, H, max_len, dtype=torch.float32, device=device) if weights else None
        lib = _lib.load()
        nbytes = max(lib.dadattn_decode_workspace_bytes(B, H, D, max_len),
                     lib.dadattn_decode_window_workspace_bytes(B, H, D, max_len, 1 if weights else 0))
        # zero-filled once: the counters must start at zero (include/dadattn.h)
        self.workspace = torch.zeros(int(nbytes), dtype=torch.uint8, device=device)


def decode_attention_bf16(out, q, k_new, v_new, cache: KVCacheBF16, scale):
    """One decode step for every sequence of ``cache``: append k_new/v_new [B,H,D] at each
    sequence's length, attend, write out [B,H,D], lengths += 1."""
    _native().decode_bf16(out, q, k_new, v_new, cache.k, cache.v, cache.lengths, cache.B, cache.H, cache.D,
                          cache.max_len, scale, cache.workspace)


def decode_attention_bf16_window(out, q, k_new, v_new, cache: KVCacheBF16, scale, *, window=0, sinks=0, weights=False):
    """:func:`decode_attention_bf16` over a sliding window: the token at row L of its sequence sees row j <= L iff
    L - j < window or j < sinks (window = 0: every row). With ``weights``, each visible row's probability is added to
    ``cache.weights`` (and the appended row's weight set to its own); the cache was made with ``weights=True``, and rows
    that a prompt filled begin with the weights that the caller puts there (zeros, say). Without ``weights`` none is written,
    on a cache that has them neither: the appended row's is then what an earlier row left in its place, until the caller
    sets it."""
    if weights and cache.weights is None:
        raise ValueError("the cache has no weights: make it with weights=True")
    _native().decode_bf16_window(cache.B, cache.H, cache.D, cache.max_len, scale, window, sinks, out, q, k_new, v_new,
                                 cache.k, cache.v, cache.lengths, cache.weights if weights else None, cache.workspace)


def kv_cache_evict_bf16(dst: KVCacheBF16, src: KVCacheBF16, budget, recent=0):
    """Keeps ``budget`` rows of every sequence and head of ``src`` that has more: the last ``recent`` ones and the
    heaviest of the others by ``src.weights`` (equal ones: the lower index). K, V and weights of the rows that stay go,
    in order, to rows 0.. of ``dst``, another cache or ``src`` itself, and ``dst.lengths`` becomes min(length, budget).
    Every row needs a weight of its own, from steps with ``weights`` or from the caller: see
    :func:`decode_attention_bf16_window`."""
    if dst.weights is None or src.weights is None:
        raise ValueError("eviction goes by the weights: make the caches with weights=True")
    _native().evict_bf16(src.B, src.H, src.D, dst.max_len, src.max_len, budget, recent, dst.k, dst.v, dst.weights,
                         dst.lengths, src.k, src.v, src.weights, src.lengths)


FP8_BLOCK = 64   # tokens that share a scale (DADATTN_FP8_BLOCK)


class KVCacheFP8:
    """A cache of one layer in 8 bits: k, v [B,H,max_len,D] e4m3 codes in blocks of 64 tokens, k_scale, v_scale
    [B,H,max_len // 64] powers of two, the rows behind the last whole block in k_tail, v_tail [B,H,64,D] bf16,
    per-sequence lengths on the device, the decode kernel's workspace. Row j of a whole block stands for
    ``k[b,h,j] * k_scale[b,h,j // 64]``, a later one is ``k_tail[b,h,j % 64]``."""

    def __init__(self, B, H, max_len, D, device="cuda"):
        self.B, self.H, self.max_len, self.D = B, H, max_len, D
        lib = _lib.load()
        self.k = torch.zeros(B, H, max_len, D, dtype=torch.uint8, device=device).view(torch.float8_e4m3fn)
        self.v = torch.zeros_like(self.k)
        self.k_scale = torch.ones(B, H, lib.dadattn_fp8_scale_blocks(max_len), dtype=torch.float32, device=device)
        self.v_scale = torch.ones_like(self.k_scale)
        self.k_tail = torch.zeros(B, H, FP8_BLOCK, D, dtype=torch.bfloat16, device=device)
        self.v_tail = torch.zeros_like(self.k_tail)
        self.lengths = torch.zeros(B, dtype=torch.int32, device=device)
        nbytes = int(lib.dadattn_decode_window_workspace_bytes(B, H, D, max_len, 0))
        self.workspace = torch.zeros(nbytes, dtype=torch.uint8, device=device)


def kv_cache_fill_fp8(cache: KVCacheFP8, k_heads, v_heads, counts=None):
    """A prefill's heads [B,H,S,D] (fp32 or bf16) into ``cache``: the first counts[b] rows (int32 [B] on the device;
    None: all S) of every sequence, which becomes that long."""
    S = k_heads.shape[2] if k_heads.dim() == 4 else 0   # (other shapes are refused by name)
    _native().fill_fp8(cache.B, cache.H, S, cache.max_len, cache.D, cache.k, cache.v, cache.k_scale, cache.v_scale,
                       cache.k_tail, cache.v_tail, cache.lengths, k_heads, v_heads, counts)


def decode_attention_fp8(out, q, k_new, v_new, cache: KVCacheFP8, scale, *, window=0, sinks=0):
    """One decode step for every sequence of an 8-bit ``cache``: append k_new / v_new [B,H,D] bf16, attend over the
    rows that :func:`decode_attention_bf16_window` would, write out [B,H,D], lengths += 1."""
    _native().decode_fp8(cache.B, cache.H, cache.D, cache.max_len, scale, window, sinks, out, q, k_new, v_new, cache.k,
                         cache.v, cache.k_scale, cache.v_scale, cache.k_tail, cache.v_tail, cache.lengths,
                         cache.workspace)


class RotaryPositions:
    """How heads are turned by their positions: the first ``rot_dim`` elements of each, in pairs (i, i + rot_dim / 2) or,
    ``interleaved``, (2 i, 2 i + 1), pair i by ``position * freq[i]`` radians. ``scaling`` for contexts ``stretch`` times as
    long as those trained on: None, "linear", "base" or "parts" (by turns over ``trained_len``, from ``low`` to ``high``);
    include/dadattn.h has the formulas. ``factor`` multiplies the turned elements; None: 0.1 ln(stretch) + 1 with "parts",
    else 1. ``freq``: radians per position (float64, on the host); ``turns``: as the kernels take them, on the device."""

    SCALINGS = {None: 0, "linear": 1, "base": 2, "parts": 3}   # DADATTN_ROTARY_*

    def __init__(self, rot_dim, *, base=10000.0, interleaved=False, scaling=None, stretch=1.0, trained_len=0, low=1.0,
                 high=32.0, factor=None, device="cuda"):
        if scaling not in self.SCALINGS:
            raise ValueError(f"unknown scaling {scaling!r}")
        host = torch.empty(max(rot_dim, 0) // 2, dtype=torch.float64)
        _lib.check(_lib.load().dadattn_rotary_frequencies(host.data_ptr() or 8, rot_dim, base, self.SCALINGS[scaling], stretch,
                                                          trained_len, low, high))
        self.rot_dim, self.interleaved = rot_dim, bool(interleaved)
        if factor is None:
            factor = 0.1 * math.log(stretch) + 1.0 if scaling == "parts" else 1.0
        self.factor = float(factor)
        self.freq = host
        turns = torch.empty(rot_dim // 2, dtype=torch.int64)
        _lib.check(_lib.load().dadattn_rotary_turns(turns.data_ptr(), host.data_ptr(), rot_dim // 2))
        self.turns = turns.to(device)


def rotary_forward(q_out, k_out, q, k, rotary: RotaryPositions, *, positions=None, first=0):
    """Queries [B,S,H,D] and keys [B,S,Hk,D] (fp32 or bf16) turned by their positions: ``positions`` [B,S] int32 on the device,
    or first + s. Any order in memory with neighbouring elements in a row: heads-split tensors are passed as
    ``x.view(B, H, S, D).transpose(1, 2)``, activations [B*S, H*D] as ``x.view(B, S, H, D)``. The results may be the tensors
    themselves; k and k_out may be None."""
    _native().rotary(0, first, rotary.turns, rotary.factor, rotary.rot_dim, rotary.interleaved, q_out, k_out, q, k, positions)


def rotary_backward(dq, dk, dq_turned, dk_turned, rotary: RotaryPositions, *, positions=None, first=0):
    """Backward of the call above: gradients of the turned tensors to those of the tensors."""
    _native().rotary(1, first, rotary.turns, rotary.factor, rotary.rot_dim, rotary.interleaved, dq, dk, dq_turned, dk_turned,
                     positions)


class KVCachePagedBF16:
    """A cache of one layer in pages: k, v [pages,H,page_size,D] bf16. Row j of sequence b is row j % page_size of page
    ``page_table[b, j // page_size]`` (int32 [B,max_pages], filled by the caller); ``lengths`` [B] int32 rows are there ahead
    of a call. Layers of a model share table and lengths: pass those of the first. H: key heads. Small calls are faster with a
    table no wider than the longest sequence needs."""

    def __init__(self, B, H, pages, page_size, max_pages, D, device="cuda", page_table=None, lengths=None):
        self.B, self.H, self.pages, self.page_size, self.max_pages, self.D = B, H, pages, page_size, max_pages, D
        self.k = torch.zeros(pages, H, page_size, D, dtype=torch.bfloat16, device=device)
        self.v = torch.zeros_like(self.k)
        self.page_table = torch.zeros(B, max_pages, dtype=torch.int32, device=device) if page_table is None else page_table
        self.lengths = torch.zeros(B, dtype=torch.int32, device=device) if lengths is None else lengths

    def _args(self):
        return (self.B, self.H, self.D, self.pages, self.page_size, self.max_pages, self.k, self.v, self.page_table,
                self.lengths)


def _rotary_args(rotary):
    return (None, 1.0, 0, 0) if rotary is None else (rotary.turns, rotary.factor, rotary.rot_dim, rotary.interleaved)


def kv_cache_append_paged(cache: KVCachePagedBF16, k_new, v_new, starts=None, *, q=None, q_out=None, rotary=None):
    """The new rows of a packed batch, k_new and v_new [T,H,D] bf16 or fp32, to their pages: sequence b's are rows
    starts[b] .. starts[b+1]-1 (int32 [B+1]; None: one for each sequence) and become its rows lengths[b] and on, which stay the
    lengths until :func:`kv_cache_advance_paged`. With ``rotary``, keys are turned by their rows, and so are queries q
    [T,Hq,D], into q_out (bf16: they are rounded, which :func:`decode_attention_paged_bf16` does not do, so that the two ways
    differ in their last bits)."""
    _native().append_paged(*cache._args(), *_rotary_args(rotary), starts, q_out, q, k_new, v_new)


def paged_attention_bf16(out, q, cache: KVCachePagedBF16, starts, max_new, scale, *, lse=None):
    """Causal attention of a packed batch's new tokens, q [T,Hq,D] bf16, over all rows of their sequences, whose pages hold
    theirs already (:func:`kv_cache_append_paged`): token i of sequence b sees rows j <= lengths[b] + i. ``max_new``: no sequence
    brings more tokens. Hq a multiple of the cache's heads. out [T,Hq,D]; lse [T,Hq] fp32 where it is wanted."""
    _native().paged_attention(*cache._args(), max_new, scale, starts, out, lse, q)


def decode_attention_paged_bf16(out, q, k_new, v_new, cache: KVCachePagedBF16, scale, *, rotary=None, lse=None):
    """One decode step for every sequence of a paged cache: the token is turned by its row (with ``rotary``), appended and
    attended for, q, out [B,Hq,D], k_new, v_new [B,H,D] bf16. The lengths stay what they are until
    :func:`kv_cache_advance_paged`: layers share them."""
    _native().decode_paged(*cache._args(), *_rotary_args(rotary), scale, out, lse, q, k_new, v_new)


def kv_cache_advance_paged(cache: KVCachePagedBF16, starts=None, tokens=None):
    """The end of a step, behind its last layer: every sequence becomes longer by its new tokens (``starts`` and ``tokens``, the
    packed batch's rows, as for the step; None: one for each)."""
    T = cache.B if starts is None else tokens
    if T is None:
        raise ValueError("tokens, the rows of the packed batch, goes with starts")
    _native().advance_paged(cache.B, T, cache.page_size, cache.max_pages, cache.lengths, starts)


def set_decode_early_start(on: bool) -> None:
    """Let :func:`decode_attention_bf16` calls of this thread fetch the lengths and their first
    cache rows while the kernel ahead of them in the stream drains. Only valid when that kernel
    does not write this call's cache, lengths or workspace (layers of a model with two or more
    layers, each with its own :class:`KVCacheBF16`); see include/dadattn.h."""
    _lib.check(_lib.load().dadattn_set_decode_early_start(1 if on else 0))


def device_status() -> int:
    """Synchronise and return (then clear) the device-side status word; 0 = no condition."""
    return int(_lib.load().dadattn_device_status(_stream()))
