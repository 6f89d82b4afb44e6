"""The compiled argument checks (csrc/py_calls.cpp) against the Python ones: what both take gives
the same bits, and what the Python ones refuse they hand back (None)."""
import numpy as np
import pytest
import torch

import kv8_ref as R

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def kv8(cuda_lib):
    from pvlc_b200 import kv8
    return kv8


def ints(x):
    return torch.tensor(x, dtype=torch.int32, device="cuda")


def steps(kv8, ops, strided, given):
    """A prompt, a decode step, a selection, a fork, a grow and a compact; all that they left."""
    g = torch.Generator(device="cuda").manual_seed(3)
    randn = lambda *s: torch.randn(s, generator=g, device="cuda")  # noqa: E731
    c = kv8.Cache.empty(1, 24, 8, 6, 2)
    into = kv8.Cache.empty(1, 20, 8, 6, 2)
    for x in (c, into):
        for t in (x.codes.view(torch.uint8), x.scales, x.tails):
            t.zero_()
    ws = kv8.Workspace(c, 4, 16)
    slot, count = ints([2, 5, 0, 7]), ints([33, 64, 5, 31])
    kv = randn(133, 2, 2, 128).half()
    k, v = (kv[:, 0], kv[:, 1]) if strided else (kv[:, 0].contiguous(), kv[:, 1].contiguous())
    kv8.grow(c, slot, ws, ahead=count)
    kv8.store(c, 0, k, v, ints([0, 33, 97, 102]), count, slot, 64, ws)
    kv8.grow(c, slot, ws, advance=count, ahead=1)
    qkv = randn(4, 20 * 128).half()
    q, kn, vn = (x.view(4, -1, 128) for x in qkv.split([2048, 256, 256], 1))
    if not strided:
        q, kn, vn = q.contiguous(), kn.contiguous(), vn.contiguous()
    cos, sin = (torch.from_numpy(t).cuda() for t in R.rope_tables(80, 1))
    out = torch.empty((4, 16, 128), dtype=torch.float16, device="cuda") if given else None
    o = kv8.decode(c, 0, q, kn, vn, cos, sin, slot, ws, rope_row=ints([1, 2, 3, 4]) if given
                   else None, out=out)
    assert not given or o is out
    logits = randn(4, 1000)
    got = ops.beam_topk(logits.half() if strided else logits, randn(1, 4), 4,
                        ops.BeamWorkspace(1, 4, 1000, 4))
    to = torch.empty_like(slot) if given else None
    new = kv8.fork(c, slot, got[1].flatten(), ws, advance=1, out=to)
    assert not given or new is to
    kv8.grow(c, new, ws, ahead=1)
    live = ints([0])
    kv8.compact(c, into, ws, live=live if given else None)
    assert ws.errors() == 0
    return [o, *got, new, into.codes.view(torch.uint8), into.scales, into.tails, into.table,
            into.tokens, into.refs, c.codes.view(torch.uint8), c.tails, c.table]


@pytest.mark.parametrize("strided", [False, True])
@pytest.mark.parametrize("given", [False, True])
def test_both_make_the_same_calls(kv8, monkeypatch, strided, given):
    from pvlc_b200 import abi, ops
    assert abi.calls is not None
    taken = []

    class Seen:
        def __getattr__(self, name):
            def call(*args):
                r = getattr(fast, name)(*args)
                taken.append((name, r is not None))
                return r
            return call
    fast = abi.calls
    monkeypatch.setattr(abi, "calls", Seen())
    a = steps(kv8, ops, strided, given)
    assert taken and all(ok for _, ok in taken), taken
    assert {n for n, _ in taken} == {"store", "decode", "grow", "fork", "compact", "beam_topk"}
    monkeypatch.setattr(abi, "calls", None)
    b = steps(kv8, ops, strided, given)
    for x, y in zip(a, b):
        assert x.dtype == y.dtype and x.shape == y.shape and x.is_contiguous()
        assert torch.equal(x.contiguous().view(torch.uint8), y.contiguous().view(torch.uint8))


def test_the_compiled_checks_refuse_what_python_refuses(kv8):
    """Each argument in turn wrong: the compiled checks return None, the function raises."""
    from pvlc_b200 import abi, ops
    c = kv8.Cache.empty(1, 4, 2, 4, 2)
    ws = kv8.Workspace(c, 2, 16)
    slot = ints([0, 1])
    h = torch.zeros((2, 16, 128), device="cuda").half()
    kv = h[:, :2].contiguous()
    cos = torch.zeros((3, 9, 128), device="cuda")
    head = (c._p, c.index, ws._p, ws.nbytes, ws.index)
    turned = h.transpose(0, 1).contiguous().transpose(0, 1)

    def wrong(fn, name, good, bad):
        for i, values in bad.items():
            for x in values:
                args = list(good)
                args[i] = x
                assert getattr(abi.calls, name)(*head, *args) is None, (name, i, x)
                with pytest.raises((TypeError, ValueError)):
                    fn(*args)
    half = slot.long()
    wrong(lambda la, q, k, v, co, si, s, r, o: kv8.decode(c, la, q, k, v, co, si, s, ws, r, o),
          "decode", (0, h, kv, kv, cos, cos, slot, slot, None),
          {0: [1, -1], 1: [h.float(), h.cpu(), h[:1], h[0], turned, 3], 2: [kv[:, :1], kv.float(), h],
           3: [kv[:1], kv.cpu(), None], 4: [cos[:2], cos.double(), cos[:, :, :64], None],
           5: [cos[:, :8], cos.cpu(), cos[0]], 6: [half, slot[:1], slot.cpu(), slot[None]],
           7: [half, slot[:1]], 8: [h[:1], h.float(), turned]})
    wrong(lambda la, s, k, v, b, n, m: kv8.store(c, la, k, v, b, n, s, m, ws), "store",
          (0, slot, kv, kv, slot, slot, 2),
          {0: [1, -1], 1: [half, slot.cpu(), None], 2: [kv.float(), kv[:, :1], kv.cpu()],
           3: [kv[:1], h], 4: [slot[:1], half], 5: [slot[:1], slot.cpu()], 6: [-1, 1 << 32]})
    wrong(lambda s, a, b: kv8.grow(c, s, ws, a, b), "grow", (slot, 0, 1),
          {0: [half, slot.cpu()], 1: [-1, 1 << 31, slot[:1], half], 2: [-1, slot.cpu()]})
    wrong(lambda s, p, a, o: kv8.fork(c, s, p, ws, a, o), "fork", (slot, slot, 0, None),
          {0: [half], 1: [slot[:1], half, slot.cpu()], 2: [-1, 1 << 31], 3: [slot[:1], half]})
    logits, scores = torch.zeros((4, 50), device="cuda"), torch.zeros((2, 2), device="cuda")
    bw = ops.BeamWorkspace(2, 2, 50, 2)
    for i, x in ((0, logits.cpu()), (0, logits.double()), (0, logits[:3]), (0, logits.t()),
                 (0, logits[0]), (1, scores.half()), (1, scores.t()[:, :1]), (1, scores.cpu()),
                 (1, scores[0])):
        args = [logits, scores, 2, bw]
        args[i] = x
        assert abi.calls.beam_topk(*args[:3], bw.buffer) is None
        with pytest.raises((TypeError, ValueError)):
            ops.beam_topk(*args)
    # what only the library refuses comes back as its error from both
    for calls in (abi.calls, None):
        keep, abi.calls = abi.calls, calls
        try:
            with pytest.raises(abi.PvlcError):
                kv8.fork(c, slot, slot, ws, out=slot)
            with pytest.raises(abi.PvlcError):
                ops.beam_topk(logits, scores, 65, bw)
        finally:
            abi.calls = keep
    assert ws.errors() == 0


def test_subclasses_and_other_streams(kv8):
    """A tensor subclass is left to the Python checks; the call goes to the current stream."""
    from pvlc_b200 import abi

    class Mine(torch.Tensor):
        pass
    c = kv8.Cache.empty(1, 4, 2, 4, 2)
    ws = kv8.Workspace(c, 2, 16)
    torch.cuda.synchronize()
    s = torch.cuda.Stream()
    with torch.cuda.stream(s):
        slot = ints([1, 0])
        assert abi.calls.grow(c._p, c.index, ws._p, ws.nbytes, ws.index, slot.as_subclass(Mine), 0,
                              32) is None
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g, stream=s):        # captures only what goes to this stream
            kv8.grow(c, slot, ws, ahead=32)
    torch.cuda.synchronize()
    assert int(c.refs.sum()) == 0
    g.replay()
    torch.cuda.synchronize()
    assert int(c.refs.sum()) == 2 and ws.errors() == 0
