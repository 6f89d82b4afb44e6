"""8-bit paged KV cache on the GPU against its plain 64-bit restatement (kv8_ref.py).

Stored codes, scales, tails, tables and counts are compared bit for bit: a power-of-two scale
leaves one rounding, and the kernels round it as the definition does.  Attention outputs are
held to the bound that Ref.decode derives for each value.
"""
import numpy as np
import pytest
import torch

import kv8_ref as R

pytestmark = pytest.mark.gpu
CODES = ["e4m3", "int8"]


@pytest.fixture(scope="module")
def kv8(cuda_lib):
    from pvlc_b200 import kv8
    return kv8


def ints(x):
    return torch.tensor(x, dtype=torch.int32, device="cuda")


# ------------------------------------------------------------------- store
@pytest.mark.parametrize("code", CODES)
@pytest.mark.parametrize("heads", [1, 2, 5])
@pytest.mark.parametrize("held,count", [
    ([0], [1]), ([0], [31]), ([0], [32]), ([0], [33]), ([7], [24]), ([7], [25]), ([7], [26]),
    ([31], [1]), ([31], [33]), ([40], [200]),
    ([0, 5, 32, 63, 64, 100, 3], [64, 0, 1, 1, 95, 28, 5])])
def test_store(kv8, code, heads, held, count):
    c = R.filled_cache(kv8, code, held, heads, layers=2, seed=1, spare=sum(count) // 32 + 9,
                       room=max(count) // 32 + 2)
    B = len(held)
    for s in range(B):
        R.give_pages(c, [s], count[s])
    ref = R.Ref(c, code)
    rng = np.random.default_rng(2)
    total = sum(count) + 3 * B + 2
    kv = rng.standard_normal((total, 2, heads, 128)).astype(np.float16)
    begin, at = [], 2
    for n in count:                      # NaN rows between the prompts are nobody's
        begin.append(at)
        at += n + 3
    used = np.zeros(total, bool)
    for b, n in zip(begin, count):
        used[b:b + n] = True
    kv[~used] = np.nan
    t = torch.from_numpy(kv).cuda()
    ws = kv8.Workspace(c, B)
    kv8.store(c, 1, t[:, 0], t[:, 1], ints(begin), ints(count), ints(list(range(B))),
              max(count), ws)
    for s in range(B):
        rows = kv[begin[s]:begin[s] + count[s]]
        ref.store(1, s, rows[:, 0], rows[:, 1])
    assert ws.errors() == 0
    ref.same(c)


@pytest.mark.parametrize("code", CODES)
def test_store_special_values(kv8, code):
    """Zeros, subnormals, the type's largest value, exact range borders, ties, NaN and
    infinities, a block each."""
    rng = np.random.default_rng(3)
    most = R.MOST[code]
    blocks = []
    base = rng.standard_normal((32, 128))
    for f in (0.0, 2.0 ** -24, 2.0 ** -15, 1.0, 65504.0):
        x = np.clip(base * f, -f, f) if f else base * 0
        x[3, 5] = f
        blocks.append(x)
    for top in (most, most * 2, most / 2, np.nextafter(np.float16(most), np.float16(1e4)),
                np.nextafter(np.float16(most), np.float16(0))):
        x = np.clip(base, -1, 1) * float(top)
        x[0, 0] = top
        x[1, :64] = float(top) * np.arange(64) / 127 / 2      # ties among them
        blocks.append(x)
    for odd in (np.nan, np.inf, -np.inf):
        x = base.copy()
        x[31, 127] = odd
        blocks.append(x)
    x = -np.abs(base)
    x[5] = -0.0
    blocks.append(x)
    k = np.concatenate(blocks).astype(np.float16)[:, None]
    v = np.concatenate(blocks[::-1]).astype(np.float16)[:, None]
    n = len(k)
    c = kv8.Cache.empty(1, n // 32, 1, n // 32, 1, R.DTYPE[code])
    c.codes.view(torch.uint8).zero_()
    c.tails.zero_()
    ws = kv8.Workspace(c, 1)
    kv8.grow(c, ints([0]), ws, ahead=n)
    ref = R.Ref(c, code)
    kv8.store(c, 0, torch.from_numpy(k).cuda(), torch.from_numpy(v).cuda(), ints([0]), ints([n]),
              ints([0]), n, ws)
    ref.store(0, 0, k, v)
    assert ws.errors() == 0
    ref.same(c)


@pytest.mark.parametrize("code", CODES)
def test_store_in_pieces_equals_store_at_once(kv8, code):
    rng = np.random.default_rng(4)
    kv = torch.from_numpy(rng.standard_normal((300, 2, 2, 128)).astype(np.float16)).cuda()
    got = []
    for pieces in ([300], [1, 30, 1, 1, 95, 172], [64, 236], [33] * 9 + [3]):
        c = kv8.Cache.empty(1, 10, 1, 10, 2, R.DTYPE[code])
        c.tails.zero_()
        c.codes.view(torch.uint8).zero_()
        c.scales.zero_()
        ws, slot, at = kv8.Workspace(c, 1), ints([0]), 0
        for n in pieces:
            kv8.grow(c, slot, ws, ahead=n)
            kv8.store(c, 0, kv[:, 0], kv[:, 1], ints([at]), ints([n]), slot, n, ws)
            kv8.grow(c, slot, ws, advance=n)
            at += n
        assert ws.errors() == 0
        got.append((c.codes.view(torch.uint8), c.scales, c.table, c.tails[:, :, :, :, :300 % 32]))
    for other in got[1:]:
        for a, b in zip(got[0], other):
            assert torch.equal(a, b)


def test_store_flags_and_leaves_alone(kv8):
    """Bad slots, counts, row ranges and pages: flagged, nothing else of theirs is written,
    good and idle neighbours are served."""
    c = R.filled_cache(kv8, "e4m3", [0] * 8, 2, spare=12, room=3)
    R.give_pages(c, range(8), 32)
    c.table[6, 0] = 99                                   # no such page
    ref = R.Ref(c, "e4m3")
    rng = np.random.default_rng(5)
    kv = rng.standard_normal((64, 2, 2, 128)).astype(np.float16)
    t = torch.from_numpy(kv).cuda()
    ws = kv8.Workspace(c, 8)
    c.tokens[5] = -4
    ref.tokens[5] = -4
    slot = [0, 8, -7, 1, 2, 5, 6, -1]
    count = [33, 32, 32, 32, 40, 8, 33, 32]
    begin = [0, 0, 0, 33, 30, 0, 0, 0]                   # 33 + 32 > 64 rows, 30 + 40 too
    kv8.store(c, 0, t[:, 0], t[:, 1], ints(begin), ints(count), ints(slot), 40, ws)
    assert ws.errors() == kv8.FLAG_SLOT | kv8.FLAG_ROWS_HELD | kv8.FLAG_INPUT_ROWS | kv8.FLAG_PAGE
    ref.store(0, 0, kv[:33, 0], kv[:33, 1])
    ref.tails[0, 6, 0, :, 0], ref.tails[0, 6, 1, :, 0] = kv[32, 0], kv[32, 1]
    ref.same(c)
    assert ws.errors() == 0
    c.tokens[5] = 0
    # over the capacity of 3 pages and 31 rows, over max_count, negative
    kv8.store(c, 0, t[:, 0], t[:, 1], ints([0, 0, 0]), ints([40, 33, -1]), ints([2, 3, 4]), 32, ws)
    assert ws.errors() == kv8.FLAG_INPUT_ROWS | kv8.FLAG_ROWS_HELD
    c.tokens[2] = 3 * 32 + 31
    kv8.store(c, 0, t[:, 0], t[:, 1], ints([0]), ints([1]), ints([2]), 32, ws)
    assert ws.errors() == kv8.FLAG_ROWS_HELD
    ref.tokens[5], ref.tokens[2] = 0, 3 * 32 + 31
    ref.same(c)


# ------------------------------------------------------------------ decode
def decode_case(kv8, code, lengths, heads, group, seed, slot=None, strided=False, rope_row=True,
                layers=1, layer=0, cache=None, scale_q=1.0):
    rng = np.random.default_rng(seed)
    B = len(lengths) if slot is None else len(slot)
    c = cache or R.filled_cache(kv8, code, lengths, heads, layers, seed, spare=len(lengths) + 3)
    R.give_pages(c, range(len(lengths)))
    QH = heads * group
    qkv = rng.standard_normal((B, (QH + 2 * heads) * 128)).astype(np.float16)
    qkv[:, :QH * 128] *= np.float16(scale_q)
    cos, sin = R.rope_tables(max(lengths) + 10, seed)
    t = torch.from_numpy(qkv).cuda()
    q = t[:, :QH * 128].view(B, QH, 128)
    k = t[:, QH * 128:(QH + heads) * 128].view(B, heads, 128)
    v = t[:, (QH + heads) * 128:].view(B, heads, 128)
    if not strided:
        q, k, v = q.contiguous(), k.contiguous(), v.contiguous()
    names = list(range(B)) if slot is None else slot
    rows = [(lengths[s] + (5 if rope_row else 0)) if 0 <= s < len(lengths) else 0 for s in names]
    ws = kv8.Workspace(c, B, QH)
    ref = R.Ref(c, code)
    kw = dict(rope_row=ints(rows) if rope_row else None)
    out = torch.full((B, QH, 128), 7.0, dtype=torch.float16, device="cuda")
    tc, ts = torch.from_numpy(cos).cuda(), torch.from_numpy(sin).cuda()

    def run():
        return kv8.decode(c, layer, q, k, v, tc, ts, ints(names) if slot is not None else None,
                          ws, out=out, **kw)
    run()
    host = lambda x: x.cpu().numpy()  # noqa: E731
    hq, hk, hv = host(q), host(k), host(v)
    got = host(out).astype(np.float64)
    for b, s in enumerate(names):
        if s == -1:
            assert (got[b] == 7.0).all(), "an idle sequence's output was written"
            continue
        want, tol = ref.decode(layer, s, hq[b], hk[b], hv[b], cos, sin, rows[b])
        off = np.abs(got[b] - want)
        assert (off <= tol).all(), (b, s, lengths[s], float((off / tol).max()))
    assert ws.errors() == 0
    ref.same(c)
    return c, ws, run, out


SHORT = [0, 1, 2, 15, 16, 30, 31, 32, 33, 62, 63, 64, 65, 95, 96, 127]


@pytest.mark.parametrize("code", CODES)
@pytest.mark.parametrize("heads,group", [(2, 8), (1, 1), (3, 5), (1, 16), (2, 9), (8, 4), (16, 2)])
def test_decode_short(kv8, code, heads, group):
    decode_case(kv8, code, SHORT, heads, group, seed=heads * 31 + group)


@pytest.mark.parametrize("code", CODES)
def test_decode_projection_views_and_default_rows(kv8, code):
    decode_case(kv8, code, [40, 3, 191, 64], 2, 8, seed=6, strided=True, rope_row=False)


def test_decode_slots_in_any_order_and_idle(kv8):
    decode_case(kv8, "e4m3", [70, 5, 31, 200, 0], 2, 8, seed=7, slot=[3, -1, 0, 4, -1, 2],
                layers=3, layer=2)


@pytest.mark.parametrize("code,heads,group,lengths", [
    ("e4m3", 2, 8, [700, 3, 1500, 64, 65, 4000]), ("int8", 2, 8, [5000]),
    ("e4m3", 1, 8, [9000]), ("int8", 4, 7, [2049, 1023, 1, 511]),
    ("int8", 1, 16, [3000, 2999]), ("e4m3", 2, 8, [1024 + 31])])
def test_decode_long(kv8, code, heads, group, lengths):
    decode_case(kv8, code, lengths, heads, group, seed=8)


@pytest.mark.parametrize("code", CODES)
def test_decode_many_ragged(kv8, code):
    rng = np.random.default_rng(9)
    lengths = [int(x) for x in rng.integers(0, 300, 150)] + [0, 31, 1200]
    decode_case(kv8, code, lengths, 2, 8, seed=9)


@pytest.mark.parametrize("scale_q", [0.0, 30.0])
def test_decode_flat_and_peaked_scores(kv8, scale_q):
    """All scores equal, and scores so far apart that one row takes all the weight."""
    decode_case(kv8, "e4m3", [100, 1000, 31], 2, 8, seed=10, scale_q=scale_q)
    decode_case(kv8, "int8", [100, 1000, 31], 2, 8, seed=10, scale_q=scale_q)


def test_decode_query_beyond_half_precision(kv8):
    """A rotated q beyond fp16's range (60000 sqrt(2)): the cached keys are scaled down so that
    the scores stay ordinary."""
    lengths = [70, 33]
    c = R.filled_cache(kv8, "e4m3", lengths, 2, seed=18, spare=4)
    c.scales[..., 0] *= 2.0 ** -15
    q = torch.full((2, 16, 128), 60000.0, device="cuda").half()
    kv = torch.zeros((2, 2, 128), device="cuda").half()
    c.tails.zero_()
    cos, sin = R.rope_tables(100)
    ref = R.Ref(c, "e4m3")
    ws = kv8.Workspace(c, 2, 16)
    out = kv8.decode(c, 0, q, kv, kv, torch.from_numpy(cos).cuda(), torch.from_numpy(sin).cuda(),
                     None, ws).cpu().numpy()
    hq, hkv = q.cpu().numpy(), kv.cpu().numpy()
    for b in range(2):
        want, tol = ref.decode(0, b, hq[b], hkv[b], hkv[b], cos, sin, lengths[b])
        assert np.isfinite(out[b]).all() and (np.abs(out[b] - want) <= tol).all()
    assert ws.errors() == 0


@pytest.mark.parametrize("code", CODES)
def test_decode_scales_far_apart(kv8, code):
    """Pages whose value (and key) scales differ by 2^14, and a page of zeros."""
    lengths = [320, 75]
    c = R.filled_cache(kv8, code, lengths, 2, seed=11, spare=6)
    for i in range(0, c.pages, 3):
        c.scales[0, i, :, 1] *= 2.0 ** -14
        c.scales[0, (i + 1) % c.pages, :, 0] *= 2.0 ** -10
    c.codes.view(torch.uint8)[0, int(c.table[0, 4])] = 0
    c.scales[0, int(c.table[0, 4])] = 1.0
    decode_case(kv8, code, lengths, 2, 8, seed=11, cache=c)


def test_decode_nan_block_reads_nan(kv8):
    """A block that was stored with a NaN gives NaN to its sequence and head alone."""
    lengths = [90, 90]
    c = R.filled_cache(kv8, "e4m3", lengths, 2, seed=12)
    c.scales[0, int(c.table[1, 1]), 1, 0] = float("nan")
    q = torch.randn((2, 16, 128), device="cuda").half()
    kv = torch.randn((2, 2, 128), device="cuda").half()
    cos, sin = (torch.from_numpy(x).cuda() for x in R.rope_tables(100))
    ws = kv8.Workspace(c, 2, 16)
    out = kv8.decode(c, 0, q, kv, kv, cos, sin, None, ws)
    nan = torch.isnan(out)
    assert nan[1, 8:].all() and not nan[1, :8].any() and not nan[0].any()
    assert ws.errors() == 0


def test_decode_flags(kv8):
    """Slots, row counts, rope rows and pages out of range: flagged, the output zero (NaN for
    a page), nothing of theirs written; a good neighbour is served."""
    lengths = [50, 50, 50, 50, 63, 63, 50]
    c = R.filled_cache(kv8, "e4m3", lengths, 2, seed=13, room=1)
    R.give_pages(c, [5])
    c.tokens[1] = -1
    c.tokens[2] = 2 * 32 + 31 if c.max_pages == 2 else 10 ** 6
    c.table[3, 0] = c.pages
    c.table[4, 1] = -1                                     # the block that closes has no page
    ref = R.Ref(c, "e4m3")
    B = 8
    slot = [0, 1, 2, 3, 4, 5, 6, 7]                        # 7: no such slot
    rows = [50, 50, 50, 50, 63, 63, 60, 50]                # 60 of 60: no such row
    cos, sin = R.rope_tables(64)
    cos, sin = cos[:, :64].copy(), sin[:, :64].copy()
    rows[6] = 64
    q = torch.randn((B, 16, 128), device="cuda").half()
    kv = torch.randn((B, 2, 128), device="cuda").half()
    ws = kv8.Workspace(c, B, 16)
    out = kv8.decode(c, 0, q, kv, kv, torch.from_numpy(cos).cuda(), torch.from_numpy(sin).cuda(),
                     ints(slot), ws, rope_row=ints(rows)).float().cpu().numpy()
    assert ws.errors() == (kv8.FLAG_ROWS_HELD | kv8.FLAG_PAGE | kv8.FLAG_ROPE_ROW | kv8.FLAG_SLOT)
    for b in (1, 2, 6, 7):
        assert (out[b] == 0).all()
    assert np.isnan(out[3]).all()
    hq, hkv = q.cpu().numpy(), kv.cpu().numpy()
    for b in (0, 4, 5):
        if b == 4:
            ref.close = lambda *a: None
        want, tol = ref.decode(0, b, hq[b], hkv[b], hkv[b], cos, sin, rows[b])
        if b == 4:
            del ref.close
        assert (np.abs(out[b] - want) <= tol).all()
    ref.tails[0, 3, 0, :, 50 % 32] = R.rotate(hkv[3], cos, sin, 50)
    ref.tails[0, 3, 1, :, 50 % 32] = hkv[3]
    ref.same(c)


def test_decode_grow_steps(kv8):
    """70 steps of grow and decode from an empty and a part-filled sequence, block ends among
    them, checked at every step against the growing reference."""
    rng = np.random.default_rng(14)
    c = kv8.Cache.empty(1, 8, 2, 4, 2)
    c.codes.view(torch.uint8).zero_()
    c.scales.zero_()
    c.tails.zero_()
    ws, slot = kv8.Workspace(c, 2, 16), ints([0, 1])
    first = rng.standard_normal((45, 2, 2, 128)).astype(np.float16)
    t = torch.from_numpy(first).cuda()
    kv8.grow(c, slot, ws, ahead=ints([0, 45]))
    ref = R.Ref(c, "e4m3")
    kv8.store(c, 0, t[:, 0], t[:, 1], ints([0, 0]), ints([0, 45]), slot, 45, ws)
    ref.store(0, 1, first[:, 0], first[:, 1])
    kv8.grow(c, slot, ws, advance=ints([0, 45]), ahead=1)
    ref.grow([0, 1], [0, 45], [1, 1])
    cos, sin = R.rope_tables(130)
    tc, ts = torch.from_numpy(cos).cuda(), torch.from_numpy(sin).cuda()
    for step in range(70):
        q = rng.standard_normal((2, 16, 128)).astype(np.float16)
        k, v = rng.standard_normal((2, 2, 2, 128)).astype(np.float16)
        out = kv8.decode(c, 0, *(torch.from_numpy(x).cuda() for x in (q, k, v)), tc, ts, slot, ws)
        got = out.cpu().numpy().astype(np.float64)
        for b in range(2):
            want, tol = ref.decode(0, b, q[b], k[b], v[b], cos, sin, int(ref.tokens[b]))
            assert (np.abs(got[b] - want) <= tol).all(), (step, b)
        kv8.grow(c, slot, ws, advance=1, ahead=1)
        ref.grow([0, 1], [1, 1], [1, 1])
    ref.same(c)
    assert ws.errors() == 0


def test_decode_repeats_bit_for_bit(kv8):
    """The same call again, on the same workspace: the same bits (no order of arrival shows)."""
    _, ws, run, out = decode_case(kv8, "e4m3", [4000, 31, 900, 3, 2500, 64] * 5, 2, 8, seed=15)
    first = out.clone()
    for _ in range(20):
        out.zero_()
        run()
        assert torch.equal(out, first)
    assert ws.errors() == 0


def test_decode_captured_and_on_two_streams(kv8):
    """A captured step replays with the values then in its buffers; two workspaces serve two
    streams at once."""
    lengths = [300, 31, 1000]
    made = [R.filled_cache(kv8, "e4m3", lengths, 2, seed=s, spare=9) for s in (16, 17)]
    cos, sin = (torch.from_numpy(x).cuda() for x in R.rope_tables(1100))
    gen = torch.Generator(device="cuda")
    gen.manual_seed(1)
    qkv = [torch.randn((3, 20, 128), generator=gen, device="cuda").half() for _ in range(2)]
    for c in made:
        R.give_pages(c, range(3))
    saved = [[x.clone() for x in (c.codes.view(torch.uint8), c.scales, c.tails)] for c in made]

    def step(c, x, ws):
        return kv8.decode(c, 0, x[:, :16], x[:, 16:18], x[:, 18:], cos, sin, None, ws)
    ws = [kv8.Workspace(c, 3, 16) for c in made]
    plain = [[step(c, x, w).clone() for x in qkv] for c, w in zip(made, ws)]
    x = qkv[0].clone()
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=side):
        got = step(made[0], x, ws[0])
    for i in (0, 1, 0):
        x.copy_(qkv[i])
        graph.replay()
        assert torch.equal(got, plain[0][i])
    streams = [torch.cuda.Stream() for _ in made]
    torch.cuda.synchronize()
    outs = [[], []]
    for _ in range(10):
        for j in range(2):
            with torch.cuda.stream(streams[j]):
                outs[j].append(step(made[j], qkv[1], ws[j]))
    torch.cuda.synchronize()
    for j in range(2):
        assert all(torch.equal(o, plain[j][1]) for o in outs[j])
        assert ws[j].errors() == 0
    del saved


# ------------------------------------------------------------------- pages
def test_grow(kv8):
    rng = np.random.default_rng(20)
    lengths = [0, 31, 32, 200, 63, 5, 95]
    c = R.filled_cache(kv8, "e4m3", lengths, 1, seed=20, spare=40, room=9)
    ref, ws = R.Ref(c, "e4m3"), kv8.Workspace(c, 8)
    slot = [3, -1, 0, 6, 1, 5]
    for adv, ahead in ((0, 1), (1, 1), (0, 1), (0, 0), ([0, 4, 5, 1, 0, 27], [40, 0, 33, 1, 2, 100]),
                       (3, [1, 1, 1, 64, 1, 1])):
        a = adv if isinstance(adv, list) else [adv] * 6
        h = ahead if isinstance(ahead, list) else [ahead] * 6
        kv8.grow(c, ints(slot), ws, advance=ints(adv) if isinstance(adv, list) else adv,
                 ahead=ints(ahead) if isinstance(ahead, list) else ahead)
        assert not ref.grow(slot, a, h)
        ref.same(c)
    assert ws.errors() == 0
    del rng


def test_grow_many_sequences_and_pages(kv8):
    """More sequences than a block has threads, free pages scattered over many passes."""
    rng = np.random.default_rng(21)
    S = 1500
    lengths = [int(x) for x in rng.integers(0, 80, S)]
    c = R.filled_cache(kv8, "int8", lengths, 1, seed=21, spare=9000, room=4)
    ref, ws = R.Ref(c, "int8"), kv8.Workspace(c, S)
    slot = rng.permutation(S)
    adv, ahead = rng.integers(0, 20, S), rng.integers(0, 60, S)
    kv8.grow(c, ints(slot), ws, advance=ints(adv), ahead=ints(ahead))
    # the reference gives pages one by one: the k-th need takes the k-th lowest free page
    for s, a in zip(slot, adv):
        ref.tokens[s] += a
    free = iter(np.flatnonzero(ref.refs == 0))
    for s, a in zip(slot, ahead):
        for j in range(ref.tokens[s] // 32, (ref.tokens[s] + a) // 32):
            ref.table[s, j] = next(free)
            ref.refs[ref.table[s, j]] = 1
    ref.same(c, pages=False)
    assert ws.errors() == 0


def test_grow_out_of_pages_and_refused(kv8):
    c = R.filled_cache(kv8, "e4m3", [31, 63, 0, 31], 1, seed=22, spare=2, room=4)
    ref, ws = R.Ref(c, "e4m3"), kv8.Workspace(c, 4)
    for slot, kw in (([0, 1, 0], {}), ([0, 4], {}), ([0, -2], {}),
                     ([0, 1], dict(advance=5 * 32 + 31)), ([2, 0], dict(advance=ints([0, -1])))):
        kv8.grow(c, ints(slot), ws, **{**dict(ahead=1), **kw})
        assert ws.errors() in (kv8.FLAG_SLOT, kv8.FLAG_ROWS_HELD)
        ref.same(c)
    kv8.grow(c, ints([3, 0, 2, 1]), ws, ahead=1)           # two pages for three
    assert ws.errors() == kv8.FLAG_EXHAUSTED
    assert ref.grow([3, 0, 2, 1], [0] * 4, [1] * 4)
    ref.same(c)


@pytest.mark.parametrize("code,layers,heads", [("e4m3", 3, 2), ("int8", 1, 5)])
def test_fork_random_steps(kv8, code, layers, heads):
    """Beam-like histories: reorder, duplicate, drop, idle, advance, with pages given between."""
    rng = np.random.default_rng(23)
    B, S = 12, 14
    lengths = [40, 95, 0, 31, 64, 7, 200, 33, 1, 32, 63, 5, 0, 0]
    c = R.filled_cache(kv8, code, lengths, heads, layers, seed=23, spare=60, room=4, poison=False)
    ref, ws = R.Ref(c, code), kv8.Workspace(c, B)
    slot = [int(x) for x in rng.permutation(12)]
    for step in range(25):
        kind = step % 4
        parent = rng.integers(0, B, B) if kind == 0 else \
            (np.arange(B) // 4 * 4 + rng.integers(0, 4, B)) if kind == 1 else \
            rng.permutation(B) if kind == 2 else rng.integers(-1, B, B)
        adv = int(rng.integers(0, 3))
        got = kv8.fork(c, ints(slot), ints(parent), ws, advance=adv).cpu().tolist()
        slot = ref.fork(slot, parent.tolist(), adv)
        assert got == slot
        ref.same(c, pages=False)
        kv8.grow(c, ints(slot), ws, ahead=3)
        ref.grow(slot, [0] * B, [3] * B)
        ref.same(c, pages=False)
        if kind == 3 and max(slot) >= 0:              # refill the dropped ones
            live = [b for b in range(B) if slot[b] >= 0]
            parent = [b if slot[b] >= 0 else live[0] for b in range(B)]
            got = kv8.fork(c, ints(slot), ints(parent), ws).cpu().tolist()
            slot = ref.fork(slot, parent)
            assert got == slot
    assert ws.errors() == 0


def test_fork_refused_and_out_of_slots(kv8):
    c = R.filled_cache(kv8, "e4m3", [40, 10, 70], 2, seed=24)
    ref, ws = R.Ref(c, "e4m3"), kv8.Workspace(c, 8)
    for slot, parent in (([0, 1, 1], [0, 1, 2]), ([0, 1, 3], [0, 1, 2]), ([0, 1, 2], [0, 1, 3]),
                         ([0, 1, -3], [0, 1, 2]), ([0, 1, 2], [-2, 1, 2])):
        assert kv8.fork(c, ints(slot), ints(parent), ws, advance=1).cpu().tolist() == slot
        assert ws.errors() == kv8.FLAG_SLOT
        ref.same(c)
    # four children of one, three slots: the last child finds none
    got = kv8.fork(c, ints([2, 0, 1, -1]), ints([0, 0, 0, 0]), ws).cpu().tolist()
    assert ws.errors() == kv8.FLAG_EXHAUSTED
    assert got == ref.fork([2, 0, 1, -1], [0, 0, 0, 0]) == [2, 0, 1, -1]
    ref.same(c)
    # everything dropped: every page is free again
    got = kv8.fork(c, ints([2, 0, 1]), ints([-1, -1, -1]), ws).cpu().tolist()
    assert got == [-1, -1, -1] and int(c.refs.abs().sum()) == 0 and int(c.tokens.sum()) == 0
    assert (c.table == -1).all() and ws.errors() == 0


@pytest.mark.parametrize("code,layers,pages", [("e4m3", 3, 0), ("int8", 1, 5000)])
def test_compact(kv8, code, layers, pages):
    lengths = [40, 0, 200, 31, 64, 95]
    c = R.filled_cache(kv8, code, lengths, 2, layers, seed=25, spare=11 + pages, room=2)
    ws = kv8.Workspace(c, 6)
    live = sum(n // 32 for n in lengths)
    into = R.filled_cache(kv8, code, [3] * 8, 2, layers, seed=26, spare=live + 2, room=9,
                          poison=False)
    ref, want = R.Ref(c, code), R.Ref(into, code)
    n = torch.zeros(1, dtype=torch.int32, device="cuda")
    kv8.compact(c, into, ws, live=n)
    order = np.flatnonzero(ref.refs > 0)
    back = {p: i for i, p in enumerate(order)}
    want.codes[:, :live], want.scales[:, :live] = ref.codes[:, order], ref.scales[:, order]
    want.refs[:] = 0
    want.refs[:live] = ref.refs[order]
    want.table[:] = -1
    want.tokens[:] = 0
    want.tokens[:6] = ref.tokens
    for s in range(6):
        for j, p in enumerate(ref.table[s]):
            if p >= 0:
                want.table[s, j] = back[p]
        want.tails[:, s, :, :, :lengths[s] % 32] = ref.tails[:, s, :, :, :lengths[s] % 32]
    assert int(n) == live and ws.errors() == 0
    want.same(into)
    ref.same(c)


def test_compact_that_does_not_fit(kv8):
    c = R.filled_cache(kv8, "e4m3", [40, 200], 2, seed=27, spare=4)   # 2 + 2 pages for 60 rows
    ws = kv8.Workspace(c, 2)
    n = torch.zeros(1, dtype=torch.int32, device="cuda")
    for spare, room, flag in ((6, 9, kv8.FLAG_EXHAUSTED), (9, 5, kv8.FLAG_ROWS_HELD)):
        into = R.filled_cache(kv8, "e4m3", [3] * 2, 2, seed=28, spare=spare, room=room,
                              poison=False)
        ref = R.Ref(into, "e4m3")
        kv8.compact(c, into, ws, live=n)
        assert int(n) == -1 and ws.errors() == flag
        ref.same(into)
    # a page given for later rows that the narrower table has no room for
    into = R.filled_cache(kv8, "e4m3", [3] * 2, 2, seed=28, spare=20, room=7, poison=False)
    ref = R.Ref(into, "e4m3")
    kv8.grow(c, ints([0, 1]), ws, ahead=60)
    kv8.compact(c, into, ws, live=n)
    assert int(n) == -1 and ws.errors() == kv8.FLAG_ROWS_HELD
    ref.same(into)


# --------------------------------------------------------------- wrappers
def test_wrapper_refusals(kv8):
    c = kv8.Cache.empty(1, 4, 2, 4, 2)
    ws = kv8.Workspace(c, 2, 16)
    ok = dict(q=torch.zeros((2, 16, 128), device="cuda").half(),
              k=torch.zeros((2, 2, 128), device="cuda").half())
    cos = torch.zeros((3, 9, 128), device="cuda")
    slot = ints([0, 1])

    def call(q=ok["q"], k=ok["k"], v=ok["k"], cos=cos, sin=cos, slot=slot, layer=0, w=ws, **kw):
        return kv8.decode(c, layer, q, k, v, cos, sin, slot, w, **kw)
    for bad in (dict(q=ok["q"].float()), dict(q=ok["q"].cpu()), dict(w=None)):
        with pytest.raises(TypeError):
            call(**bad)
    for bad in (dict(q=ok["q"][:1]), dict(k=ok["k"][:, :1]), dict(layer=1), dict(layer=-1),
                dict(slot=slot[:1]), dict(rope_row=slot[:1]), dict(out=ok["q"][:1]),
                dict(q=ok["q"].transpose(0, 1).contiguous().transpose(0, 1)),
                dict(sin=cos[:, :8].contiguous())):
        with pytest.raises(ValueError):
            call(**bad)
    with pytest.raises(TypeError):
        call(slot=slot.long())
    with pytest.raises(ValueError):
        kv8.grow(c, slot, ws, advance=-1)
    with pytest.raises(TypeError):
        kv8.grow(c, slot, ws, ahead=slot.long())
    with pytest.raises(ValueError):
        kv8.fork(c, slot, slot[:1], ws)
    from pvlc_b200 import abi
    with pytest.raises(abi.PvlcError):
        kv8.fork(c, slot, slot, ws, out=slot)
    with pytest.raises(abi.PvlcError):
        kv8.Workspace(c, 4000, 16)
    with pytest.raises(ValueError):
        kv8.Cache(c.codes, c.scales, c.tails[:, :1], c.table, c.tokens, c.refs)
    with pytest.raises(TypeError):
        kv8.Cache(c.codes.view(torch.uint8), c.scales, c.tails, c.table, c.tokens, c.refs)
    small = kv8.Workspace(c, 2, 16)
    small.nbytes = 4096
    with pytest.raises(abi.PvlcError):
        kv8.grow(c, slot, small, ahead=1)
