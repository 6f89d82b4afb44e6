"""What captured and concurrent calls leave in the cache."""
import numpy as np
import pytest
import torch

import kv8_ref as R

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def kv8(cuda_lib):
    from pvlc_b200 import kv8
    return kv8


def arrays(c):
    return [c.codes.view(torch.uint8), c.scales, c.tails, c.table, c.tokens, c.refs]


@pytest.mark.parametrize("code", ["e4m3", "int8"])
def test_replays_and_streams_leave_what_a_call_leaves(kv8, code):
    """Two caches, a workspace each: a captured step (decode, grow) replayed for two inputs, and
    steps on two streams at once, against the reference and bit for bit against plain calls."""
    lengths = [300, 30, 31, 1000]                    # two of them close a block within the steps
    cos, sin = R.rope_tables(1100)
    tc, ts = torch.from_numpy(cos).cuda(), torch.from_numpy(sin).cuda()
    g = torch.Generator(device="cuda").manual_seed(2)
    xs = [torch.randn((4, 20, 128), generator=g, device="cuda").half() for _ in range(2)]
    slot = torch.arange(4, dtype=torch.int32, device="cuda")
    made = [R.filled_cache(kv8, code, lengths, 2, seed=s, spare=9) for s in (16, 17)]
    for c in made:
        R.give_pages(c, range(4))
    saved = [[t.clone() for t in arrays(c)] for c in made]
    ws = [kv8.Workspace(c, 4, 16) for c in made]

    def restore():
        for c, s in zip(made, saved):
            for t, old in zip(arrays(c), s):
                t.copy_(old)

    def step(i, x):
        out = kv8.decode(made[i], 0, x[:, :16], x[:, 16:18], x[:, 18:], tc, ts, slot, ws[i])
        kv8.grow(made[i], slot, ws[i], advance=1, ahead=1)
        return out
    refs = [R.Ref(c, code) for c in made]
    outs, after = [[], []], []
    for i in (0, 1):
        for x in xs:
            outs[i].append(step(i, x).clone())
            h = x.cpu().numpy()
            for b in range(4):
                want, tol = refs[i].decode(0, b, h[b, :16], h[b, 16:18], h[b, 18:], cos, sin,
                                           int(refs[i].tokens[b]))
                assert (np.abs(outs[i][-1][b].cpu().numpy() - want) <= tol).all()
            refs[i].grow(range(4), [1] * 4, [1] * 4)
        refs[i].same(made[i])
        after.append([t.clone() for t in arrays(made[i])])

    def check(i):
        for t, want in zip(arrays(made[i]), after[i]):
            assert torch.equal(t.view(torch.uint8), want.view(torch.uint8))
    restore()
    x = xs[0].clone()
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=side):
        got = step(0, x)
    for k in (0, 1):
        x.copy_(xs[k])
        graph.replay()
        assert torch.equal(got, outs[0][k])
    check(0)
    restore()
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in made]
    both = [[], []]
    for k in (0, 1):
        for i in (0, 1):
            with torch.cuda.stream(streams[i]):
                both[i].append(step(i, xs[k]))
    torch.cuda.synchronize()
    for i in (0, 1):
        assert all(torch.equal(a, b) for a, b in zip(both[i], outs[i]))
        check(i)
        assert ws[i].errors() == 0


@pytest.mark.parametrize("code,group", [("e4m3", 1), ("int8", 2), ("e4m3", 9)])
def test_the_largest_batch(kv8, code, group):
    """2,048 sequences, whose places in shared memory leave the ring its fewest stages."""
    rng = np.random.default_rng(3)
    B = 2048
    lengths = [int(n) for n in rng.integers(0, 70, B)]
    lengths[7], lengths[-1] = 900, 1203
    c = R.filled_cache(kv8, code, lengths, 1, seed=5, spare=B // 8)
    R.give_pages(c, range(B))
    cos, sin = R.rope_tables(1300)
    q = rng.standard_normal((B, group, 128)).astype(np.float16)
    k, v = rng.standard_normal((2, B, 1, 128)).astype(np.float16)
    slot = rng.permutation(B).astype(np.int32)
    dev = lambda x: torch.from_numpy(x).cuda()  # noqa: E731
    ws = kv8.Workspace(c, B, group)
    ref = R.Ref(c, code)
    out = kv8.decode(c, 0, dev(q), dev(k), dev(v), dev(cos), dev(sin), dev(slot), ws).cpu().numpy()
    for b, s in enumerate(slot):
        want, tol = ref.decode(0, s, q[b], k[b], v[b], cos, sin, lengths[s])
        assert (np.abs(out[b] - want) <= tol).all(), (b, lengths[s])
    assert ws.errors() == 0
    ref.same(c)
