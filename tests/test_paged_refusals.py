"""CPU: what the rotary and paged-cache calls refuse, before anything reaches a GPU, and the frequencies."""
import ctypes as C
import math

import pytest
import torch

import dadgpt_b200 as dad
from tests import paged_reference

P = 1 << 20   # a pointer that is not looked at


def _strides(*s):
    return (C.c_int64 * len(s))(*s)


def _rotary(lib, **change):
    s = _strides(10 * 4 * 64, 4 * 64, 64)
    a = dict(q_out=P, k_out=P, q=P, k=P, qo=s, ko=s, qs=s, ks=s, positions=None, first=0, B=2, S=10, Hq=4, Hk=4, D=64, turns=P,
             factor=1.0, rot=64, interleaved=0, backward=0, bf16=1, stream=None)
    a.update(change)
    return lib.dadattn_rotary(*a.values())


def _append(lib, **change):
    s = _strides(4 * 64, 64)
    a = dict(k=P, v=P, table=P, lengths=P, starts=P, q_out=P, q=P, k_new=P, v_new=P, qo=s, qs=s, ks=s, vs=s, B=2, T=10, Hq=4,
             Hkv=4, D=64, pages=9, page=16, max_pages=4, turns=P, factor=1.0, rot=64, interleaved=0, bf16=1, stream=None)
    a.update(change)
    return lib.dadattn_paged_append_bf16(*a.values())


def _attention(lib, **change):
    s = _strides(8 * 64, 64)
    a = dict(out=P, lse=P, q=P, os=s, qs=s, k=P, v=P, table=P, lengths=P, starts=P, B=2, T=10, max_new=9, Hq=8, Hkv=4, D=64,
             pages=9, page=16, max_pages=4, scale=0.125, stream=None)
    a.update(change)
    return lib.dadattn_paged_attention_bf16(*a.values())


def _decode(lib, **change):
    s = _strides(8 * 64, 64)
    a = dict(out=P, lse=None, q=P, k_new=P, v_new=P, os=s, qs=s, ks=s, vs=s, k=P, v=P, table=P, lengths=P, B=2, Hq=8, Hkv=4,
             D=64, pages=9, page=16, max_pages=4, scale=0.125, turns=P, factor=1.0, rot=64, interleaved=0, stream=None)
    a.update(change)
    return lib.dadattn_decode_paged_bf16(*a.values())


def _advance(lib, **change):
    a = dict(lengths=P, starts=P, B=2, T=10, page=16, max_pages=4, stream=None)
    a.update(change)
    return lib.dadattn_paged_advance(*a.values())


NAN, INF = float("nan"), float("inf")
BAD = [(_rotary, c, rc) for c, rc in [
    (dict(q=None), -1), (dict(k_out=None), -1), (dict(qs=None), -1), (dict(B=0), -1), (dict(S=-1), -1), (dict(Hk=-1), -1),
    (dict(D=72), -2), (dict(D=272), -2), (dict(rot=0), -1), (dict(rot=80), -1), (dict(rot=8), -2), (dict(turns=None), -1),
    (dict(turns=P + 8), -1), (dict(factor=NAN), -1), (dict(factor=INF), -1), (dict(q=P + 8), -1), (dict(positions=P + 2), -1),
    (dict(qs=_strides(640, 64, 4)), -1), (dict(qs=_strides(640, 64, -64)), -1), (dict(qo=_strides(640, 0, 64)), -1),
    (dict(q_out=2 * P, qo=_strides(0, 256, 64)), -1), (dict(qs=_strides(2560, 64, 640)), -1), (dict(Hq=1 << 20), -2)]]
PAGED = [(dict(k=None), -1), (dict(table=None), -1), (dict(lengths=None), -1), (dict(B=0), -1), (dict(Hkv=0), -1), (dict(pages=0), -1),
         (dict(max_pages=-1), -1), (dict(D=32), -2), (dict(D=96), -2), (dict(page=8), -2), (dict(page=48), -2), (dict(page=2048), -2),
         (dict(max_pages=1 << 27), -2), (dict(pages=1 << 30), -2), (dict(k=P + 8), -1), (dict(table=P + 2), -1)]
BAD += [(call, c, rc) for call in (_append, _attention, _decode) for c, rc in PAGED]
BAD += [(_append, c, rc) for c, rc in [
    (dict(T=0), -1), (dict(starts=None), -1), (dict(starts=P + 2), -1), (dict(rot=8), -2), (dict(rot=-16), -1), (dict(rot=128), -1),
    (dict(turns=None), -1), (dict(q_out=None), -1), (dict(q=None), -1), (dict(k_new=None), -1), (dict(v_new=P + 8), -1),
    (dict(ks=None), -1), (dict(ks=_strides(256, 60)), -1), (dict(ks=_strides(-256, 64)), -1), (dict(qo=_strides(0, 64)), -1),
    (dict(bf16=0), -1), (dict(q_out=2 * P, Hq=1 << 20), -2), (dict(qs=_strides(512, 64)), -1)]]   # (bf16=0: fp32 queries in place)
BAD += [(_attention, c, rc) for c, rc in [
    (dict(out=None), -1), (dict(q=None), -1), (dict(T=0), -1), (dict(max_new=0), -1), (dict(starts=None), -1), (dict(Hq=6), -1),
    (dict(Hq=0), -1), (dict(Hq=4 * 129), -2), (dict(scale=0.0), -1), (dict(scale=-1.0), -1), (dict(scale=NAN), -1),
    (dict(scale=INF), -1), (dict(out=P + 8), -1), (dict(lse=P + 2), -1), (dict(os=_strides(0, 64)), -1), (dict(qs=_strides(0, 64)), -1),
    (dict(qs=_strides(512, 0)), -1), (dict(qs=_strides(512, 4)), -1), (dict(T=1 << 30, B=1 << 29), -2), (dict(T=1 << 26, Hkv=1024, Hq=1024), -2)]]
BAD += [(_decode, c, rc) for c, rc in [
    (dict(out=None), -1), (dict(v_new=None), -1), (dict(Hq=6), -1), (dict(scale=0.0), -1), (dict(scale=NAN), -1), (dict(rot=24), -2),
    (dict(turns=None), -1), (dict(lse=P + 1), -1), (dict(q=P + 4), -1), (dict(os=_strides(512, 0)), -1), (dict(B=1 << 27), -2)]]
BAD += [(_advance, c, rc) for c, rc in [
    (dict(lengths=None), -1), (dict(lengths=P + 2), -1), (dict(B=0), -1), (dict(T=0), -1), (dict(starts=None), -1), (dict(page=10), -2),
    (dict(max_pages=0), -1)]]


@pytest.mark.parametrize("call,change,code", BAD, ids=lambda x: x.__name__ if callable(x) else None)
def test_refused(lib, call, change, code):
    assert call(lib, **change) == code
    assert lib.dadattn_last_error()


FREQ = [dict(rot_dim=64), dict(rot_dim=16, base=500000.0), dict(rot_dim=2), dict(rot_dim=128, scaling="linear", stretch=4.0),
        dict(rot_dim=64, scaling="base", stretch=8.0), dict(rot_dim=128, scaling="parts", stretch=16.0, trained_len=4096),
        dict(rot_dim=64, scaling="parts", stretch=8.0, trained_len=8192, low=1.0, high=4.0, base=500000.0, factor=1.0)]


@pytest.mark.parametrize("case", FREQ, ids=str)
def test_frequencies(lib, case):
    r = dad.RotaryPositions(**case, device="cpu")
    how = {k: v for k, v in case.items() if k not in ("rot_dim", "factor")}
    want = paged_reference.frequencies(case["rot_dim"], **how)
    # a power, a division and a sum or two in 64 bits
    assert bool(((r.freq - want).abs() <= 2.0 ** -47 * want).all()) and r.freq.dtype == torch.float64
    want = case.get("factor", 0.1 * math.log(case["stretch"]) + 1 if case.get("scaling") == "parts" else 1.0)
    assert r.factor == want


@pytest.mark.parametrize("bad", [dict(rot_dim=0), dict(rot_dim=7), dict(rot_dim=-2), dict(rot_dim=258), dict(rot_dim=64, base=1.0),
                                 dict(rot_dim=64, base=NAN), dict(rot_dim=64, base=INF), dict(rot_dim=64, scaling="linear", stretch=0.5),
                                 dict(rot_dim=64, scaling="base", stretch=NAN), dict(rot_dim=64, scaling="parts", stretch=2.0),
                                 dict(rot_dim=64, scaling="parts", stretch=2.0, trained_len=100, low=4.0, high=4.0)], ids=str)
def test_frequencies_refused(lib, bad):
    with pytest.raises(RuntimeError, match="rotary frequencies"):
        dad.RotaryPositions(**bad, device="cpu")
    with pytest.raises(ValueError, match="unknown scaling"):
        dad.RotaryPositions(64, scaling="other", device="cpu")


def test_turns(lib):
    """Fractions of a turn, rounded to 2^-64: from fractions with 50 digits of pi."""
    from fractions import Fraction
    freq = dad.RotaryPositions(128, device="cpu").freq.tolist() + [-0.25, 0.0, 6.5, 1000.125]
    a, got = (C.c_double * len(freq))(*freq), (C.c_uint64 * len(freq))()
    assert lib.dadattn_rotary_turns(got, a, len(freq)) == 0
    pi = Fraction(31415926535897932384626433832795028841971693993751, 10 ** 49)
    for w, t in zip(freq, got):
        want = Fraction(w) / (2 * pi)
        off = (Fraction(t, 2 ** 64) - want) % 1
        # half a unit, and the product's rounding in 64 bits of mantissa
        assert min(off, 1 - off) <= Fraction(1, 2 ** 64) + abs(want) / 2 ** 62
    assert lib.dadattn_rotary_turns(None, a, 1) == -1 and lib.dadattn_rotary_turns(got, None, 1) == -1
    assert lib.dadattn_rotary_turns(got, a, 0) == -1
    for bad in (NAN, INF, 1e30):
        assert lib.dadattn_rotary_turns(got, (C.c_double * 1)(bad), 1) == -1


def test_tensors_are_checked_in_python(lib):
    r = dad.RotaryPositions(64, device="cpu")
    c = dad.KVCachePagedBF16(2, 4, 9, 16, 4, 64, device="cpu")
    x = torch.zeros(2, 10, 4, 64)
    with pytest.raises(ValueError, match="CUDA tensor"):
        dad.rotary_forward(x, x, x, x, r)
    with pytest.raises(ValueError, match=r"\[B, S, heads, D\]"):
        dad.rotary_backward(x[0], None, x[0], None, r)
    with pytest.raises(ValueError, match="CUDA tensor"):
        dad.kv_cache_append_paged(c, x[0], x[0], torch.zeros(3, dtype=torch.int32))
    with pytest.raises(ValueError, match="CUDA tensor"):
        dad.paged_attention_bf16(x[0], x[0], c, None, 1, 0.125)
    with pytest.raises(ValueError, match="CUDA tensor"):
        dad.decode_attention_paged_bf16(x[0], x[0], x[0], x[0], c, 0.125)
    with pytest.raises(ValueError, match=r"\[tokens, heads, D\]"):
        dad.kv_cache_append_paged(c, x, x)
    with pytest.raises(ValueError, match="CUDA tensor"):
        dad.kv_cache_advance_paged(c)
    with pytest.raises(ValueError, match="goes with starts"):
        dad.kv_cache_advance_paged(c, torch.zeros(3, dtype=torch.int32))
