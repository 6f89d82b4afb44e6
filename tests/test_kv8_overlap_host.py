"""Outputs that share memory with what a call reads are refused before any device effect (the
pointers are never read: no GPU needed)."""
import ctypes

import pytest

from pvlc_b200 import abi

STEP = 1 << 30                            # more than any array below holds
NAMES = ("codes", "scales", "tails", "table", "tokens", "refs")
SIZES = dict(layers=2, pages=64, slots=8, max_pages=16, kv_heads=2, code_type=0)
BYTES = dict(codes=2 * 64 * 2 * 2 * 4096, scales=2 * 64 * 2 * 8, tails=2 * 8 * 2 * 2 * 8192,
             table=8 * 16 * 4, tokens=8 * 4, refs=64 * 4)
CACHE = abi.Kv8CacheStruct(**{n: STEP * (i + 1) for i, n in enumerate(NAMES)}, **SIZES)
WORKSPACE = 1 << 26


def decode(out, batch=4, **kw):
    """16 query and 2 KV heads; q rows 2,560 elements apart, k and v rows 1,024."""
    a = {n: STEP * (10 + i) for i, n in enumerate(("q", "k", "v", "cos", "sin", "row", "slot", "ws"))}
    a.update(kw)
    return abi.lib().pvlc_attn_kv8_decode(
        ctypes.byref(CACHE), 0, a["q"], 2560, a["k"], a["v"], 1024, 16, a["cos"], a["sin"], 10,
        a["row"], a["slot"], batch, a["ws"], WORKSPACE, out, None)


@pytest.mark.parametrize("name", NAMES)
def test_decode_into_the_cache(name):
    base = getattr(CACHE, name)
    last = (BYTES[name] - 1) // 16 * 16
    for at in (base, base + last, base - 4 * 4096 + 16):
        assert decode(at) == abi.LENGTH_MISMATCH, name


@pytest.mark.parametrize("i,size", [(3, 3 * 10 * 512), (4, 3 * 10 * 512), (5, 16), (6, 16),
                                    (7, WORKSPACE)])
def test_decode_into_tables_slots_and_workspace(i, size):
    base = STEP * (10 + i)
    for at in (base, base + (size - 1) // 16 * 16, base - 4 * 4096 + 16):
        assert decode(at) == abi.LENGTH_MISMATCH


@pytest.mark.parametrize("i,stride,row", [(0, 5120, 4096), (1, 2048, 512), (2, 2048, 512)])
def test_decode_into_its_rows(i, stride, row):
    base = STEP * (10 + i)
    for b in range(4):
        for at in (base + b * stride, base + b * stride + row - 16):
            assert decode(at) == abi.LENGTH_MISMATCH
            assert decode(at, batch=1) == abi.LENGTH_MISMATCH if b == 0 else True
    assert decode(base - 4 * 4096 + 16) == abi.LENGTH_MISMATCH


@pytest.mark.parametrize("name", NAMES + ("ws",))
def test_fork_and_compact_into_the_cache(name):
    """slot_out and live_out are written before the tables are read."""
    other = abi.Kv8CacheStruct(**{n: STEP * (i + 20) for i, n in enumerate(NAMES)}, **SIZES)
    ws = STEP * 30
    base, size = (ws, WORKSPACE) if name == "ws" else (getattr(CACHE, name), BYTES[name])
    for at in (base, base + size - 4, base - 12):
        assert abi.lib().pvlc_attn_kv8_fork(ctypes.byref(CACHE), STEP * 31, STEP * 32, 4, 1, at, ws,
                                            WORKSPACE, None) == abi.LENGTH_MISMATCH
    for a, b in ((CACHE, other), (other, CACHE)):
        for at in (base, base + size - 4):
            assert abi.lib().pvlc_attn_kv8_compact(ctypes.byref(a), ctypes.byref(b), at, ws, WORKSPACE,
                                                   None) == abi.LENGTH_MISMATCH


@pytest.mark.parametrize("half", [0, 1])
def test_beam_outputs(half):
    """3 requests of 2 beams, 100 logits 128 apart, the best 5."""
    unit = 2 if half else 4
    good = [STEP * (40 + i) for i in range(6)]           # logits, scores, workspace, the outputs

    def call(x, s, ws, *outs):
        return abi.lib().pvlc_lm_head_beam_topk(x, half, 128, s, 3, 2, 100, 5, ws, WORKSPACE, *outs, None)
    places = [good[0], good[0] + 5 * 128 * unit + 100 * unit - 4, good[0] + 128 * unit + 4, good[0] - 56,
              good[1], good[1] + 6 * 4 - 4, good[2], good[2] + WORKSPACE - 4]
    for i in (3, 4, 5):
        others = [o for o in (3, 4, 5) if o != i]
        for at in places + [good[o] + d for o in others for d in (0, 56, -56)]:
            args = list(good)
            args[i] = at
            assert call(*args) == abi.LENGTH_MISMATCH, (i, at)
