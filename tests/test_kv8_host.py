"""Refusals of the 8-bit paged cache and of the beam selection: the library checks its
arguments on the host before any device effect, so they need no GPU (the pointers below are
never read)."""
import ctypes

import pytest
import torch

from pvlc_b200 import abi, kv8, ops

P16 = 1 << 20                     # a well-aligned address that is never read
BIG = 1 << 40


def cache(**kw):
    d = dict(codes=P16, scales=P16 * 2, tails=P16 * 3, table=P16 * 4, tokens=P16 * 5,
             refs=P16 * 6, layers=2, pages=64, slots=8, max_pages=16, kv_heads=2, code_type=0)
    d.update(kw)
    return abi.Kv8CacheStruct(**d)


CACHE_REFUSALS = [
    (dict(layers=0), abi.ZERO_DIMENSION), (dict(pages=0), abi.ZERO_DIMENSION),
    (dict(slots=0), abi.ZERO_DIMENSION), (dict(max_pages=0), abi.ZERO_DIMENSION),
    (dict(kv_heads=0), abi.ZERO_DIMENSION), (dict(code_type=2), abi.INVALID_DECODER_GEOMETRY),
    (dict(kv_heads=17), abi.INVALID_DECODER_GEOMETRY),
    (dict(slots=65537), abi.INVALID_DECODER_GEOMETRY),
    (dict(max_pages=(1 << 20) + 1), abi.INVALID_DECODER_GEOMETRY),
    (dict(layers=1025), abi.INVALID_DECODER_GEOMETRY),
    (dict(pages=1 << 24), abi.ARITHMETIC_OVERFLOW),
    (dict(codes=None), abi.NULL_POINTER), (dict(refs=None), abi.NULL_POINTER),
    (dict(tails=None), abi.NULL_POINTER), (dict(codes=P16 + 8), abi.MISALIGNED_POINTER),
    (dict(scales=P16 + 4), abi.MISALIGNED_POINTER), (dict(table=P16 + 2), abi.MISALIGNED_POINTER),
]


def decode(c, **kw):
    a = dict(layer=0, q=P16, qs=2560, k=P16, v=P16, ks=2560, heads=16, cos=P16, sin=P16, rr=10,
             row=None, slot=P16, batch=4, ws=P16, wsb=BIG, out=P16)
    a.update(kw)
    return abi.lib().pvlc_attn_kv8_decode(
        ctypes.byref(c) if c is not None else None, a["layer"], a["q"], a["qs"], a["k"], a["v"],
        a["ks"], a["heads"], a["cos"], a["sin"], a["rr"], a["row"], a["slot"], a["batch"],
        a["ws"], a["wsb"], a["out"], None)


def store(c, **kw):
    a = dict(layer=0, k=P16, v=P16, rows=100, rs=256, begin=P16, count=P16, slot=P16, batch=4,
             most=50, ws=P16, wsb=BIG)
    a.update(kw)
    return abi.lib().pvlc_attn_kv8_store(
        ctypes.byref(c), a["layer"], a["k"], a["v"], a["rows"], a["rs"], a["begin"], a["count"],
        a["slot"], a["batch"], a["most"], a["ws"], a["wsb"], None)


def grow(c, **kw):
    a = dict(slot=P16, batch=4, adv=None, advn=1, ahead=None, aheadn=1, ws=P16, wsb=BIG)
    a.update(kw)
    return abi.lib().pvlc_attn_kv8_grow(ctypes.byref(c), a["slot"], a["batch"], a["adv"],
                                        a["advn"], a["ahead"], a["aheadn"], a["ws"], a["wsb"],
                                        None)


def fork(c, **kw):
    a = dict(slot=P16, parent=P16 * 2, batch=4, adv=0, out=P16 * 3, ws=P16, wsb=BIG)
    a.update(kw)
    return abi.lib().pvlc_attn_kv8_fork(ctypes.byref(c), a["slot"], a["parent"], a["batch"],
                                        a["adv"], a["out"], a["ws"], a["wsb"], None)


@pytest.mark.parametrize("change,code", CACHE_REFUSALS)
def test_cache_refusals(change, code):
    for call in (decode, store, grow, fork):
        assert call(cache(**change)) == code, call.__name__
    L = abi.lib()
    bad, good = cache(**change), cache(codes=P16 * 7, scales=P16 * 8, tails=P16 * 9,
                                       table=P16 * 10, tokens=P16 * 11, refs=P16 * 12)
    assert L.pvlc_attn_kv8_compact(ctypes.byref(bad), ctypes.byref(good), None, P16, BIG,
                                   None) == code
    assert L.pvlc_attn_kv8_compact(ctypes.byref(good), ctypes.byref(bad), None, P16, BIG,
                                   None) == code


def test_null_cache():
    assert decode(None) == abi.NULL_POINTER
    assert abi.lib().pvlc_attn_kv8_compact(None, None, None, P16, BIG, None) == abi.NULL_POINTER


@pytest.mark.parametrize("change,code", [
    (dict(batch=0), abi.ZERO_DIMENSION), (dict(heads=0), abi.ZERO_DIMENSION),
    (dict(rr=0), abi.ZERO_DIMENSION), (dict(batch=2049), abi.INVALID_DECODER_GEOMETRY),
    (dict(layer=2), abi.INVALID_DECODER_GEOMETRY), (dict(heads=15), abi.INVALID_DECODER_GEOMETRY),
    (dict(heads=34, qs=34 * 128), abi.INVALID_DECODER_GEOMETRY),
    (dict(slot=None, batch=9), abi.INVALID_DECODER_GEOMETRY),
    (dict(qs=2040), abi.LENGTH_MISMATCH), (dict(ks=248), abi.LENGTH_MISMATCH),
    (dict(qs=2052), abi.LENGTH_MISMATCH), (dict(ks=260), abi.LENGTH_MISMATCH),
    (dict(q=None), abi.NULL_POINTER), (dict(out=None), abi.NULL_POINTER),
    (dict(cos=None), abi.NULL_POINTER), (dict(q=P16 + 8), abi.MISALIGNED_POINTER),
    (dict(out=P16 + 2), abi.MISALIGNED_POINTER), (dict(slot=P16 + 1), abi.MISALIGNED_POINTER),
    (dict(row=P16 + 2), abi.MISALIGNED_POINTER), (dict(ws=None), abi.NULL_POINTER),
    (dict(ws=P16 + 4), abi.MISALIGNED_POINTER), (dict(wsb=1000), abi.WORKSPACE_TOO_SMALL),
])
def test_decode_refusals(change, code):
    assert decode(cache(), **change) == code


@pytest.mark.parametrize("change,code", [
    (dict(batch=0), abi.ZERO_DIMENSION), (dict(rows=0), abi.ZERO_DIMENSION),
    (dict(most=0), abi.ZERO_DIMENSION), (dict(batch=2049), abi.INVALID_DECODER_GEOMETRY),
    (dict(layer=2), abi.INVALID_DECODER_GEOMETRY), (dict(most=101), abi.CAPACITY_EXHAUSTED),
    (dict(rows=10000, most=16 * 32 + 32), abi.CAPACITY_EXHAUSTED),
    (dict(rs=248), abi.LENGTH_MISMATCH), (dict(rs=260), abi.LENGTH_MISMATCH),
    (dict(k=None), abi.NULL_POINTER), (dict(slot=None), abi.NULL_POINTER),
    (dict(begin=None), abi.NULL_POINTER), (dict(v=P16 + 8), abi.MISALIGNED_POINTER),
    (dict(count=P16 + 2), abi.MISALIGNED_POINTER), (dict(wsb=100), abi.WORKSPACE_TOO_SMALL),
])
def test_store_refusals(change, code):
    assert store(cache(), **change) == code


@pytest.mark.parametrize("change,code", [
    (dict(batch=0), abi.ZERO_DIMENSION), (dict(batch=2049), abi.INVALID_DECODER_GEOMETRY),
    (dict(advn=16 * 32 + 32), abi.CAPACITY_EXHAUSTED),
    (dict(aheadn=1 << 31), abi.CAPACITY_EXHAUSTED), (dict(slot=None), abi.NULL_POINTER),
    (dict(adv=P16 + 2), abi.MISALIGNED_POINTER), (dict(wsb=1000), abi.WORKSPACE_TOO_SMALL),
])
def test_grow_refusals(change, code):
    assert grow(cache(), **change) == code


@pytest.mark.parametrize("change,code", [
    (dict(batch=0), abi.ZERO_DIMENSION), (dict(batch=2049), abi.INVALID_DECODER_GEOMETRY),
    (dict(adv=1 << 20), abi.CAPACITY_EXHAUSTED), (dict(parent=None), abi.NULL_POINTER),
    (dict(out=P16), abi.LENGTH_MISMATCH), (dict(out=P16 + 12), abi.LENGTH_MISMATCH),
    (dict(out=P16 * 2 - 8), abi.LENGTH_MISMATCH), (dict(out=P16 * 3 + 1), abi.MISALIGNED_POINTER),
    (dict(wsb=1000), abi.WORKSPACE_TOO_SMALL),
])
def test_fork_refusals(change, code):
    assert fork(cache(), **change) == code


def test_compact_refusals():
    f = abi.lib().pvlc_attn_kv8_compact
    other = dict(codes=P16 * 7, scales=P16 * 8, tails=P16 * 9, table=P16 * 10, tokens=P16 * 11,
                 refs=P16 * 12)

    def call(a, b, live=None, ws=P16, wsb=BIG):
        return f(ctypes.byref(a), ctypes.byref(b), live, ws, wsb, None)
    for kw in (dict(layers=3), dict(kv_heads=1), dict(code_type=1), dict(slots=7)):
        assert call(cache(), cache(**{**other, **kw})) == abi.INVALID_DECODER_GEOMETRY
    for name in other:
        assert call(cache(), cache(**{**other, name: getattr(cache(), name)})) == \
            abi.LENGTH_MISMATCH
    assert call(cache(), cache(**other), live=P16 + 1) == abi.MISALIGNED_POINTER
    assert call(cache(), cache(**other), wsb=1000) == abi.WORKSPACE_TOO_SMALL


@pytest.mark.parametrize("args", [(0, 16, 2, 4, 4), (2049, 16, 2, 4, 4), (4, 15, 2, 4, 4),
                                  (4, 16, 17, 4, 4), (4, 34, 2, 4, 4), (4, 0, 2, 4, 4),
                                  (4, 16, 2, 65537, 4)])
def test_workspace_bytes_out_of_range(args):
    assert abi.lib().pvlc_attn_kv8_workspace_bytes(*args) == 0


def test_workspace_bytes_grow_with_the_call():
    f = abi.lib().pvlc_attn_kv8_workspace_bytes
    assert 0 < f(1, 16, 2, 1, 1) <= f(64, 16, 2, 1, 1) <= f(64, 16, 2, 1, 1 << 20)


def beam(**kw):
    a = dict(x=P16, half=0, ld=1000, s=P16, B=2, W=4, V=1000, K=8, ws=P16, wsb=BIG, o=P16)
    a.update(kw)
    return abi.lib().pvlc_lm_head_beam_topk(a["x"], a["half"], a["ld"], a["s"], a["B"], a["W"],
                                            a["V"], a["K"], a["ws"], a["wsb"], a["o"], P16, P16,
                                            None)


@pytest.mark.parametrize("change,code", [
    (dict(B=0), abi.ZERO_DIMENSION), (dict(W=0), abi.ZERO_DIMENSION),
    (dict(V=0), abi.ZERO_DIMENSION), (dict(K=0), abi.ZERO_DIMENSION),
    (dict(W=33), abi.INVALID_DECODER_GEOMETRY), (dict(K=65), abi.INVALID_DECODER_GEOMETRY),
    (dict(B=2049), abi.INVALID_DECODER_GEOMETRY), (dict(B=2048, W=32), abi.INVALID_DECODER_GEOMETRY),
    (dict(V=(1 << 24) + 1, ld=1 << 30), abi.INVALID_DECODER_GEOMETRY),
    (dict(ld=999), abi.LENGTH_MISMATCH), (dict(half=2), abi.LENGTH_MISMATCH),
    (dict(W=1, V=7, ld=7), abi.LENGTH_MISMATCH), (dict(x=None), abi.NULL_POINTER),
    (dict(o=None), abi.NULL_POINTER), (dict(x=P16 + 2), abi.MISALIGNED_POINTER),
    (dict(half=1, x=P16 + 1), abi.MISALIGNED_POINTER), (dict(wsb=64), abi.WORKSPACE_TOO_SMALL),
])
def test_beam_refusals(change, code):
    assert beam(**change) == code
    bad = {k: v for k, v in change.items() if k in "BWVK"}
    if code in (abi.ZERO_DIMENSION, abi.INVALID_DECODER_GEOMETRY):
        a = dict(B=2, W=4, V=1000, K=8)
        a.update(bad)
        assert abi.lib().pvlc_lm_head_beam_topk_workspace_bytes(a["B"], a["W"], a["V"], a["K"]) == 0


def test_compact_refuses_overlapping_caches():
    """No array of one cache may share bytes with any of the other."""
    f = abi.lib().pvlc_attn_kv8_compact
    names = ("codes", "scales", "tails", "table", "tokens", "refs")
    step = 1 << 30                         # more than any array of the two holds
    a = cache(**{n: step * (i + 1) for i, n in enumerate(names)})
    b = {n: step * (i + 7) for i, n in enumerate(names)}
    for i, n in enumerate(names):
        for m in names:
            # 16 bytes into one of a's arrays (each is longer than that)
            at = step * (i + 1) + 16
            assert f(ctypes.byref(a), ctypes.byref(cache(**{**b, m: at})), None, P16, BIG,
                     None) == abi.LENGTH_MISMATCH, (n, m)


def test_compiled_checks_pass_nothing_by_on_the_host():
    """The compiled argument checks were built, and hand anything that is not a CUDA call back
    to the Python ones (None)."""
    abi.lib()
    c = abi.calls
    assert c is not None, "make -C paddleocr-vl-webgpu_b200 builds pvlc_b200/_calls.so"
    t, i = torch.zeros((2, 2, 128), dtype=torch.float16), torch.zeros(2, dtype=torch.int32)
    head = (0, 0, 0, 0, 0)
    for args in ((), (None,), head, (*head, 0, i, t, t, i, i, 4), (*head, -1, i, t, t, i, i, 4),
                 (*head, 0, t, t, t, t, t, i, None, None), (*head, i, i, i, None),
                 (*head, i, 1, 1), (1 << 70, *head[1:], i, 1, 1), (*head, 0, 0, None), ("x",) * 14,
                 (torch.zeros((2, 9)), torch.zeros((1, 2)), 2, torch.zeros(64, dtype=torch.uint8)),
                 (i, i, 2, i), (None, None, None, None)):
        for fn in (c.store, c.decode, c.grow, c.fork, c.compact, c.beam_topk):
            assert fn(*args) is None, (fn, args)


def test_compiled_checks_load_in_a_fresh_process():
    """Also where the library is loaded before anything has imported torch."""
    import os
    import subprocess
    import sys
    package = os.path.dirname(os.path.dirname(abi.__file__))
    code = f"import sys; sys.path.insert(0, {package!r}); from pvlc_b200 import abi; abi.lib(); " \
           "sys.exit(abi.calls is None)"
    assert subprocess.run([sys.executable, "-c", code]).returncode == 0


def test_wrappers_refuse_host_tensors():
    t = torch.zeros((1, 4, 2, 2, 32, 128), dtype=torch.int8)
    with pytest.raises(TypeError):
        kv8.Cache(t, None, None, None, None, None)
    with pytest.raises(TypeError):
        ops.beam_topk(torch.zeros((4, 100)), torch.zeros((1, 4)), 4)
    with pytest.raises(TypeError):
        kv8.grow(None, None, None)
