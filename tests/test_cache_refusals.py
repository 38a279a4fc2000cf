"""CPU: what the cache calls refuse, before anything reaches a GPU."""
import pytest
import torch

import dadgpt_b200 as dad
from dadgpt_b200 import _lib

P = 1 << 20   # a pointer that is not looked at


def _far(i):
    return P + (i << 40)   # arrays that do not overlap


def _window(lib, **change):
    a = dict(out=P, q=P, k_new=P, v_new=P, k=P, v=P, lengths=P, weights=None, B=2, H=3, D=64, max_len=100, scale=0.125,
             window=8, sinks=2, workspace=P, bytes=1 << 30, stream=None)
    a.update(change)
    return lib.dadattn_decode_bf16_window(*a.values())


def _fp8(lib, **change):
    a = dict(out=P, q=P, k_new=P, v_new=P, k=P, v=P, k_scale=P, v_scale=P, k_tail=P, v_tail=P, lengths=P, B=2, H=3, D=64,
             max_len=100, scale=0.125, window=0, sinks=0, workspace=P, bytes=1 << 30, stream=None)
    a.update(change)
    return lib.dadattn_decode_fp8(*a.values())


def _fill(lib, **change):
    a = dict(k=P, v=P, k_scale=P, v_scale=P, k_tail=P, v_tail=P, lengths=P, k_heads=P, v_heads=P, counts=None, B=2, H=3,
             S=50, max_len=100, D=64, bf16=1, stream=None)
    a.update(change)
    return lib.dadattn_kv_cache_fill_fp8(*a.values())


def _evict(lib, **change):
    a = dict(kd=_far(0), vd=_far(1), wd=_far(2), ld=_far(3), ks=_far(4), vs=_far(5), ws=_far(6), ls=_far(7), B=2, H=3, D=64,
             max_dst=100, max_src=200, budget=50, recent=5, stream=None)
    a.update(change)
    return lib.dadattn_kv_cache_evict_bf16(*a.values())


BAD = [(_window, c, rc) for c, rc in [
    (dict(q=None), -1), (dict(lengths=None), -1), (dict(B=0), -1), (dict(H=-1), -1), (dict(max_len=0), -1),
    (dict(B=1 << 20, H=1 << 15), -1), (dict(max_len=(1 << 30) + 1), -2), (dict(D=32), -2), (dict(window=-1), -1),
    (dict(sinks=-1), -1), (dict(scale=float("nan")), -1), (dict(scale=float("inf")), -1), (dict(k=P + 8), -1),
    (dict(lengths=P + 2), -1), (dict(weights=P + 2), -1), (dict(workspace=None), -1), (dict(workspace=P + 4), -1),
    (dict(bytes=255), -5), (dict(weights=P, bytes=256 + 2 * 3 * 100 * 4 - 1), -5)]]
BAD += [(_fp8, c, rc) for c, rc in [
    (dict(v_tail=None), -1), (dict(k_scale=None), -1), (dict(v_scale=P + 2), -1), (dict(k_tail=P + 8), -1), (dict(D=96), -2),
    (dict(window=-5), -1), (dict(bytes=0), -5)]]
BAD += [(_fill, c, rc) for c, rc in [
    (dict(k_heads=None), -1), (dict(S=0), -1), (dict(S=101), -1), (dict(B=70000, H=1), -2), (dict(D=16), -2),
    (dict(v_heads=P + 8), -1), (dict(counts=P + 1), -1), (dict(k_scale=P + 2), -1), (dict(max_len=-4), -1)]]
BAD += [(_evict, c, rc) for c, rc in [
    (dict(ws=None), -1), (dict(budget=0), -1), (dict(budget=101), -1), (dict(recent=51), -1), (dict(recent=-1), -1),
    (dict(D=256), -2), (dict(max_src=196609), -2), (dict(kd=_far(0) + 8), -1), (dict(kd=_far(4)), -1), (dict(kd=_far(4) + 1024), -1),
    (dict(vd=_far(0)), -1), (dict(wd=_far(6)), -1), (dict(ld=_far(7)), -1),
    (dict(kd=_far(4), vd=_far(5), wd=_far(6), ld=_far(7)), -1)]]   # (the two max_len differ)


@pytest.mark.parametrize("call,change,code", BAD, ids=lambda x: x.__name__ if callable(x) else str(x))
def test_refused(lib, call, change, code):
    assert call(lib, **change) == code
    assert lib.dadattn_last_error()


def test_sizes(lib):
    assert [lib.dadattn_fp8_scale_blocks(n) for n in (-1, 0, 1, 63, 64, 127, 128, 1280)] == [0, 0, 1, 1, 1, 1, 2, 20]
    size = lib.dadattn_decode_window_workspace_bytes
    assert size(64, 12, 64, 1280, 0) == 3328 and size(1, 1, 64, 10, 0) == 256 and size(0, 1, 64, 10, 0) == 0
    assert size(64, 12, 64, 1280, 1) == 3328 + 64 * 12 * 1280 * 4
    # as much as the plain decode call's counters take, so that one zeroed workspace serves both
    assert size(64, 12, 64, 1280, 0) <= lib.dadattn_decode_workspace_bytes(64, 12, 64, 1280)


def test_tensors_are_checked_in_python(lib):
    cache = dad.KVCacheFP8(2, 3, 100, 64, device="cpu")
    x = torch.zeros(2, 3, 64, dtype=torch.bfloat16)
    with pytest.raises(ValueError, match="CUDA tensor"):
        dad.decode_attention_fp8(x, x, x, x, cache, 0.125)
    heads = torch.zeros(2, 3, 10, 64)
    with pytest.raises(ValueError, match="CUDA tensor"):
        dad.kv_cache_fill_fp8(cache, heads, heads)
    plain, weighted = dad.KVCacheBF16(2, 3, 100, 64, device="cpu"), dad.KVCacheBF16(2, 3, 100, 64, device="cpu", weights=True)
    with pytest.raises(ValueError, match="CUDA tensor"):
        dad.decode_attention_bf16_window(x, x, x, x, plain, 0.125, window=4)
    with pytest.raises(ValueError, match="weights=True"):
        dad.decode_attention_bf16_window(x, x, x, x, plain, 0.125, weights=True)
    with pytest.raises(ValueError, match="weights=True"):
        dad.kv_cache_evict_bf16(weighted, plain, 10)
    with pytest.raises(ValueError, match="CUDA tensor"):
        dad.kv_cache_evict_bf16(weighted, weighted, 10)
    assert issubclass(_lib.DadAttnError, RuntimeError)


def _forward(lib, **change):
    a = dict(out=P, lse=P, q=P, k=P, v=P, BH=4, S=100, D=64, scale=0.125, window=8, sinks=2, stream=None)
    a.update(change)
    return lib.dadattn_flash_fwd_bf16_window(*a.values())


def _backward(lib, **change):
    a = dict(dq=P, dk=P, dv=P, workspace=P, bytes=1 << 30, dout=P, out=P, lse=P, q=P, k=P, v=P, BH=4, S=100, D=64, scale=0.125,
             window=8, sinks=2, stream=None)
    a.update(change)
    return lib.dadattn_flash_bwd_bf16_window(*a.values())


COMMON = [(dict(q=None), -1), (dict(lse=None), -1), (dict(lse=P + 2), -1), (dict(v=P + 8), -1), (dict(BH=0), -1), (dict(S=-1), -1),
          (dict(BH=65536), -2), (dict(S=(1 << 30) + 1), -2), (dict(D=32), -2), (dict(scale=0.0), -1), (dict(scale=-1.0), -1),
          (dict(scale=float("nan")), -1), (dict(scale=float("inf")), -1), (dict(window=-1), -1), (dict(sinks=-2), -1)]


@pytest.mark.parametrize("call,change,code", [(_forward, *c) for c in COMMON] + [(_backward, *c) for c in COMMON] +
                         [(_backward, dict(workspace=P + 16), -1), (_backward, dict(bytes=100), -5), (_backward, dict(dout=None), -1)],
                         ids=lambda x: x.__name__ if callable(x) else str(x))
def test_windowed_attention_refuses(lib, call, change, code):
    assert call(lib, **change) == code and lib.dadattn_last_error()


def test_windowed_attention_checks_tensors(lib):
    x, lse = torch.zeros(2, 8, 64, dtype=torch.bfloat16), torch.zeros(2, 8)
    with pytest.raises(ValueError, match="CUDA tensor"):
        dad.gpu_flash_attention_forward_bf16_window(x, lse, x, x, x, 2, 8, 64, 0.125, 4)
    with pytest.raises(ValueError, match="CUDA tensor"):
        dad.gpu_flash_attention_backward_bf16_window(x, x, x, x, x, x, lse, x, x, x, 2, 8, 64, 0.125, 4)
