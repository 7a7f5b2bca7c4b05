"""CPU checks of the calls around a decoder layer and a beam search: what they refuse, with which code and message, before any device
work, and the tables of frequencies."""
import ctypes as C
import math

import pytest

from test_kv_cache_abi import AT, INVALID, UNSUPPORTED, cache, refused


def norm(qb, x=AT, dtype=0, xs=64, r=None, rt=0, rs=64, w=AT, eps=1e-6, m=2, n=64, q=AT, d=AT):
    return qb.lib().qnt_rms_norm_q8(x, dtype, xs, r, rt, rs, w, eps, m, n, q, d, None)


@pytest.mark.parametrize("change, code, word", [
    (dict(x=None), INVALID, "null"), (dict(w=None), INVALID, "null"), (dict(q=None), INVALID, "null"), (dict(d=None), INVALID, "null"),
    (dict(dtype=2), UNSUPPORTED, "dtype"), (dict(n=48), INVALID, "multiple of 32"), (dict(n=0), INVALID, "multiple"),
    (dict(n=32800, xs=32800), UNSUPPORTED, "32768"), (dict(m=-1), INVALID, "multiple"), (dict(xs=63), INVALID, "x_stride"),
    (dict(eps=-1e-6), INVALID, "eps"), (dict(eps=math.nan), INVALID, "eps"), (dict(x=AT + 2), INVALID, "aligned"),
    (dict(x=AT + 1, dtype=1), INVALID, "aligned"), (dict(w=AT + 2), INVALID, "aligned"), (dict(q=AT + 8), INVALID, "aligned"),
    (dict(d=AT + 4), INVALID, "aligned"), (dict(r=AT), INVALID, "not be x"), (dict(r=AT + 2048, rs=10), INVALID, "residual_stride"),
    (dict(r=AT + 2050, rt=0), INVALID, "aligned"), (dict(r=AT + 2048, rt=4), UNSUPPORTED, "residual"),
    (dict(r=AT + 2048, dtype=1, rt=4), UNSUPPORTED, "residual"), (dict(r=AT + 2049, dtype=1, rt=1), INVALID, "aligned")])
def test_norm(qb, change, code, word):
    refused(qb, norm(qb, **change), code, word)


def test_nothing_to_do(qb):
    L = qb.lib()
    assert norm(qb, m=0, x=None, q=None) == 0
    assert L.qnt_dequantize_q8(None, None, 0, 64, None, 0, None) == 0
    assert L.qnt_rope(None, 0, None, 0, 0, None, 0, None, 0, 0, 0, 64, 64, 0, None, 1.0, None, 5, None) == 0
    assert L.qnt_rope(None, 0, None, 0, 4, None, 0, None, 0, 0, 0, 64, 64, 0, None, 1.0, None, 0, None) == 0
    assert L.qnt_beam_select(None, 0, 0, None, None, 0, 0, 4, 100, 4, None, None, None, None, 0, None) == 0
    c = cache(qb)
    assert L.qnt_kv_reorder(C.byref(c), None, None, 0, 0, None, 0, None) == 0


@pytest.mark.parametrize("change, code, word", [
    (dict(q=None), INVALID, "null"), (dict(d=None), INVALID, "null"), (dict(out=None), INVALID, "null"), (dict(q=AT + 8), INVALID, "aligned"),
    (dict(out=AT + 8), INVALID, "aligned"), (dict(d=AT + 2), INVALID, "aligned"), (dict(n=40), INVALID, "multiple"), (dict(n=0), INVALID, "multiple"),
    (dict(m=-1), INVALID, "multiple"), (dict(dtype=3), UNSUPPORTED, "dtype"), (dict(m=2 ** 31 - 1, n=2 ** 20), UNSUPPORTED, "too many")])
def test_dequantize(qb, change, code, word):
    a = dict(q=AT, d=AT, m=2, n=64, out=AT, dtype=0) | change
    refused(qb, qb.lib().qnt_dequantize_q8(a["q"], a["d"], a["m"], a["n"], a["out"], a["dtype"], None), code, word)


@pytest.mark.parametrize("change, code, word", [
    (dict(q=None), INVALID, "null q"), (dict(qo=None), INVALID, "null q"), (dict(k=None), INVALID, "null k"), (dict(dtype=2), UNSUPPORTED, "dtype"),
    (dict(hd=63), INVALID, "head_dim"), (dict(hd=1026, rot=64), INVALID, "head_dim"), (dict(rot=66), INVALID, "rotary_dim"),
    (dict(rot=0), INVALID, "rotary_dim"), (dict(rot=7), INVALID, "rotary_dim"), (dict(heads=-1), INVALID, "heads"), (dict(kv=5000), INVALID, "heads"),
    (dict(m=-1), INVALID, "tokens"), (dict(qs=255), INVALID, "stride of q"), (dict(kos=127), INVALID, "stride of k"),
    (dict(qo=AT, qos=512), INVALID, "two strides"), (dict(q=AT + 2), INVALID, "aligned"), (dict(ko=AT + 1, dtype=1), INVALID, "aligned"),
    (dict(turns=None), INVALID, "turns"), (dict(turns=AT + 4), INVALID, "turns"), (dict(pos=None), INVALID, "positions"),
    (dict(pos=AT + 2), INVALID, "positions")])
def test_rope(qb, change, code, word):
    a = dict(q=AT, qs=256, qo=2 * AT, qos=256, heads=4, k=AT, ks=128, ko=3 * AT, kos=128, kv=2, dtype=0, hd=64, rot=64, inter=0, turns=AT, scale=1.0,
             pos=AT, m=2) | change
    refused(qb, qb.lib().qnt_rope(*a.values(), None), code, word)


@pytest.mark.parametrize("change, code, word", [
    (dict(x=None), INVALID, "null"), (dict(s=None), INVALID, "null"), (dict(out=None), INVALID, "null"), (dict(t=None), INVALID, "null"),
    (dict(p=None), INVALID, "null"), (dict(x=AT + 2), INVALID, "aligned"), (dict(s=AT + 1), INVALID, "aligned"), (dict(p=AT + 2), INVALID, "aligned"),
    (dict(dtype=2), UNSUPPORTED, "dtype"), (dict(k=0), INVALID, "positive"), (dict(k=65), UNSUPPORTED, "at most 64"),
    (dict(b=0), INVALID, "positive"), (dict(b=1025), UNSUPPORTED, "beams"), (dict(v=0), INVALID, "positive"), (dict(g=-1), INVALID, "positive"),
    (dict(v=1, b=2, k=3), INVALID, "fewer than k"), (dict(v=2 ** 30, b=4, stride=2 ** 30), UNSUPPORTED, "too large"),
    (dict(g=2 ** 30), UNSUPPORTED, "too large"), (dict(stride=999), INVALID, "stride"), (dict(e=AT, end=-1), INVALID, "end_id"),
    (dict(e=AT, end=1000), INVALID, "end_id"), (dict(ws=None), INVALID, "workspace"), (dict(ws=AT + 8), INVALID, "workspace"),
    (dict(nb=10), INVALID, "workspace")])
def test_beam_select(qb, change, code, word):
    a = dict(x=AT, dtype=0, stride=1000, s=AT, e=None, end=-1, g=2, b=4, v=1000, k=4, out=AT, t=AT, p=AT, ws=AT, nb=1 << 40) | change
    refused(qb, qb.lib().qnt_beam_select(*a.values(), None), code, word)


def test_beam_workspace(qb):
    need = qb.lib().qnt_beam_workspace
    assert need(1, 4, 1000, 4) > 0 and need(0, 4, 1000, 4) == 0 and need(1, 4, 1000, 65) == 0 and need(1, 0, 1000, 1) == 0
    assert need(64, 4, 151936, 8) < 64 << 20


@pytest.mark.parametrize("change, code, word", [
    (dict(seqs=None), INVALID, "null"), (dict(parents=None), INVALID, "null"), (dict(seqs=AT + 2), INVALID, "aligned"),
    (dict(parents=AT + 1), INVALID, "aligned"), (dict(n=-1), INVALID, "count"), (dict(n=5, group=5), INVALID, "count"),
    (dict(group=3), INVALID, "whole groups"), (dict(group=0), INVALID, "whole groups"), (dict(group=-4), INVALID, "whole groups"),
    (dict(ws=None), INVALID, "workspace"), (dict(ws=AT + 4), INVALID, "workspace"), (dict(nb=16), INVALID, "workspace")])
def test_reorder(qb, change, code, word):
    c = cache(qb)
    a = dict(seqs=AT, parents=AT, n=4, group=2, ws=AT, nb=1 << 40) | change
    refused(qb, qb.lib().qnt_kv_reorder(C.byref(c), *a.values(), None), code, word)
    bad = cache(qb, head_dim=96)
    refused(qb, qb.lib().qnt_kv_reorder(C.byref(bad), *a.values(), None), UNSUPPORTED, "head_dim")
    assert qb.lib().qnt_kv_reorder_workspace(C.byref(bad)) == 0 and qb.lib().qnt_kv_reorder_workspace(C.byref(c)) > 0


def test_frequencies(qb):
    f, scale = qb.Rope.frequencies(64, 1e6)
    assert scale == 1.0 and len(f) == 32 and f[0] == 1.0 and math.isclose(f[16], 1e-3)
    for bad in (dict(kind="other"), dict(kind="linear"), dict(kind="linear", factor=0.0), dict(kind="yarn", factor=2.0),
                dict(kind="bands", factor=2.0, original=100, low=4, high=4), dict(kind="linear", factor=2.0, original=5), dict(factor=2.0)):
        with pytest.raises(ValueError):
            qb.Rope.frequencies(64, 1e6, bad)
    with pytest.raises(ValueError):
        qb.Rope.frequencies(64, 1.0)
    with pytest.raises(ValueError):
        qb.Rope(7)
    with pytest.raises(ValueError):
        qb.Rope(8, frequencies=[1.0], device="cpu")
