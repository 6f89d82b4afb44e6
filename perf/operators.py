"""Measured cases of the 8-bit paged KV cache and of beam search.

Four operators that a beam-searching OCR decoder calls next to one another:

  store   rows of prompts into 8-bit pages (kv8_store)
  decode  one token of every sequence against the pages (kv8_decode)
  pages   reordering, growing (kv8_fork, kv8_grow) and compacting (kv8_compact) sequences
  beam    the best continuations of every request (beam_topk)

A cache is `codes` [layers, pages, 2, heads, 32, 128] (8 bits; K and V), `scales` [layers, pages,
heads, 2] (f32 powers of two), `tails` [layers, slots, 2, heads, 32, 128] (fp16 rows of each
sequence's open block), `table` [slots, max_pages], `tokens` [slots] and `refs` [pages] (int32).
"""
import math

import torch

own = False

PAGE, HD = 32, 128
CODES = {"e4m3": (torch.float8_e4m3fn, 448.0), "int8": (torch.int8, 127.0)}
THETA = 500000.0


# ------------------------------------------------------------------ cases
def listed():
    return [
        # the second half of a page's prompt, continued in the middle of a block, one layer
        dict(name="store one prompt int8", op="store", code="int8", heads=2, batch=1, low=1564,
             high=1564, held=23, seed=1),
        # a batch of 256 page prompts, one layer
        dict(name="store 256 prompts e4m3", op="store", code="e4m3", heads=2, batch=256, low=1238,
             high=1238, held=0, seed=2),
        # one page being read, one layer: latency
        dict(name="decode 1 x 1023 e4m3", op="decode", code="e4m3", heads=2, group=8, batch=1,
             low=1023, high=1023, beams=1, seed=3),
        # the serving batch of the decode benchmark: ragged, long
        dict(name="decode 64 ragged e4m3", op="decode", code="e4m3", heads=2, group=8, batch=64,
             low=512, high=8192, beams=1, seed=4),
        # 64 pages with four beams each, the prompt's pages shared by the four
        dict(name="decode 64 x 4 beams int8", op="decode", code="int8", heads=2, group=8,
             batch=256, low=1238, high=1500, beams=4, seed=5),
        # a decoder with more key heads and fewer queries for each
        dict(name="decode 8 heads e4m3", op="decode", code="e4m3", heads=8, group=4, batch=16,
             low=4096, high=8192, beams=1, seed=6),
        # the beams of two requests after a step, every layer
        dict(name="fork 2 x 4 beams", op="fork", code="e4m3", heads=2, layers=18, batch=8, beams=4,
             low=1238, high=1300, seed=7),
        # the beams of a serving batch after a step, every layer
        dict(name="fork 64 x 4 beams", op="fork", code="int8", heads=2, layers=18, batch=256,
             beams=4, low=1238, high=1500, seed=8),
        # a small cache, half of it free, into one that fits
        dict(name="compact 65 pages", op="compact", code="int8", heads=2, layers=3, slots=5,
             low=200, high=447, spare=2.0, seed=9),
        # a decoder's cache after most of its requests have ended
        dict(name="compact 32 sequences", op="compact", code="e4m3", heads=2, layers=18, slots=32,
             low=512, high=2500, spare=3.0, seed=10),
        # one request, half-precision logits: latency
        dict(name="beam 1 x 4 f16", op="beam", dtype="f16", batch=1, beams=4, vocab=103424, topk=8,
             seed=11),
        # a serving batch's logits
        dict(name="beam 64 x 4 f32", op="beam", dtype="f32", batch=64, beams=4, vocab=103424,
             topk=8, seed=12),
    ]


def _spread(rng, low, high):
    return int(round(math.exp(rng.uniform(math.log(low), math.log(high)))))


def draw(rng):
    """Another case: an operator, then its sizes over the ranges above (no dearer than the
    largest listed case of the operator)."""
    op = rng.choice(["store", "decode", "fork", "compact", "beam"])
    seed = rng.randrange(1 << 20)
    code = rng.choice(["e4m3", "int8"])
    if op == "store":
        heads = rng.choice([1, 2, 2, 4, 8])
        batch = _spread(rng, 1, 256)
        high = _spread(rng, 1, max(2, min(8192, 256 * 1238 * 2 // (batch * heads))))
        return dict(op=op, code=code, heads=heads, batch=batch, low=rng.randint(1, high),
                    high=high, held=rng.randint(0, 100), seed=seed)
    if op == "decode":
        heads = rng.choice([1, 2, 2, 4, 8])
        group = rng.choice([1, 2, 4, 7, 8, 8, 16])
        beams = rng.choice([1, 1, 4])
        batch = beams * _spread(rng, 1, 64 if beams == 4 else 200)
        high = _spread(rng, 1, max(2, min(8192, 64 * 8192 * 2 // (batch * heads))))
        return dict(op=op, code=code, heads=heads, group=group, batch=batch,
                    low=rng.randint(0, high), high=high, beams=beams, seed=seed)
    if op == "fork":
        beams = rng.randint(1, 8)
        return dict(op=op, code=code, heads=rng.choice([1, 2, 4]), layers=rng.choice([1, 3, 18]),
                    batch=beams * _spread(rng, 1, 32), beams=beams, low=1, high=_spread(rng, 2, 1500),
                    seed=seed)
    if op == "compact":
        slots = _spread(rng, 1, 32)
        return dict(op=op, code=code, heads=rng.choice([1, 2]), layers=rng.choice([1, 3, 18]),
                    slots=slots, low=rng.randint(0, 300), high=_spread(rng, 300, 2500),
                    spare=rng.choice([1.25, 2.0, 3.0]), seed=seed)
    return dict(op=op, dtype=rng.choice(["f16", "f32", "f32"]), batch=_spread(rng, 1, 64),
                beams=rng.randint(1, 4), vocab=_spread(rng, 100, 103424), topk=rng.randint(1, 16),
                seed=seed)


# ----------------------------------------------------------------- inputs
def _gen(seed):
    g = torch.Generator(device="cuda")
    g.manual_seed(seed)
    return g


def _lengths(case):
    """The case's lengths: of the case alone, so that work() knows them."""
    g = torch.Generator()
    g.manual_seed(case["seed"])
    n = case.get("batch") or case["slots"]
    n //= case.get("beams", 1)
    got = torch.randint(case["low"], case["high"] + 1, (n,), generator=g)
    return got.repeat_interleave(case.get("beams", 1)).tolist()


def _codes(g, layers, pages, heads, code):
    """Pages of N(0, 1) rows: codes around scales of 2^-7 .. 2^-4."""
    kind, most = CODES[code]
    e = torch.randint(-1, 2, (layers, pages, heads, 2), generator=g, device="cuda")
    base = -6.0 if code == "e4m3" else -5.0
    scales = torch.exp2(base + e.float())
    codes = torch.empty((layers, pages, 2, heads, PAGE, HD), dtype=kind, device="cuda")
    step = max(1, (1 << 26) // (pages * 2 * heads * PAGE * HD))
    for i in range(0, layers, step):
        x = torch.randn(codes[i:i + step].shape, generator=g, device="cuda")
        x /= scales[i:i + step].transpose(2, 3)[..., None, None]
        x.clamp_(-most, most)
        codes[i:i + step] = x.round_().to(kind) if code == "int8" else x.to(kind)
    return codes, scales


def _cache(g, case, layers, rows, shared, pages_more, max_more=2):
    """A cache whose sequence s holds rows[s] rows in slot s, its pages in no order; every
    `shared` neighbours share all but their last full page."""
    full = [n // PAGE for n in rows]
    host = torch.Generator()
    host.manual_seed(int(torch.randint(0, 1 << 30, (1,), generator=g, device="cuda")))
    slots, need = len(rows), 0
    width = max(full + [0]) + max_more
    table = torch.full((slots, width), -1, dtype=torch.int32)
    for s, n in enumerate(full):
        common = max(0, n - 1) if s % shared else 0
        if common:
            table[s, :common] = table[s - s % shared, :common]
        table[s, common:n] = torch.arange(need, need + n - common, dtype=torch.int32)
        need += n - common
    pages = need + pages_more(need)
    order = torch.randperm(pages, generator=host).to(torch.int32)
    table = torch.where(table >= 0, order[table.clamp(min=0).long()], table)
    refs = torch.bincount(table[table >= 0].long(), minlength=pages).to(torch.int32)
    codes, scales = _codes(g, layers, pages, case["heads"], case["code"])
    tails = torch.randn((layers, slots, 2, case["heads"], PAGE, HD), generator=g,
                        device="cuda").half()
    return dict(codes=codes, scales=scales, tails=tails, table=table.cuda(),
                tokens=torch.tensor(rows, dtype=torch.int32, device="cuda"), refs=refs.cuda())


def _rope(rows):
    """Axis-major M-RoPE tables [3, rows, 128] of text positions (all axes alike)."""
    freq = THETA ** (-torch.arange(0, HD, 2, dtype=torch.float64, device="cuda") / HD)
    ang = torch.arange(rows, dtype=torch.float64, device="cuda")[:, None] * freq
    ang = torch.cat([ang, ang], 1).expand(3, rows, HD)
    return ang.cos().float().contiguous(), ang.sin().float().contiguous()


def prepare(case, seed):
    g = _gen(seed)
    randn = lambda *s: torch.randn(s, generator=g, device="cuda")  # noqa: E731
    ints = lambda x: torch.tensor(x, dtype=torch.int32, device="cuda")  # noqa: E731
    if case["op"] == "beam":
        B, W, V = case["batch"], case["beams"], case["vocab"]
        logits = randn(B * W, V) * 3
        logits[:, ::97] = -math.inf                     # suppressed tokens
        scores = -5 * torch.rand((B, W), generator=g, device="cuda")
        return dict(case=case, scores=scores,
                    logits=logits.half() if case["dtype"] == "f16" else logits)
    if case["op"] == "store":
        count, held = _lengths(case), case["held"]
        B, H = case["batch"], case["heads"]
        cache = _cache(g, case, 1, [held] * B, 1, lambda n: sum(held // PAGE + c // PAGE + 2 for c in count),
                       max(count) // PAGE + 2)
        # the pages that the new rows will fill
        free = (cache["refs"] == 0).nonzero().flatten().int().tolist()
        table, at = cache["table"].cpu(), 0
        for b, c in enumerate(count):
            a, z = held // PAGE, (held + c) // PAGE
            table[b, a:z] = torch.tensor(free[at:at + z - a], dtype=torch.int32)
            at += z - a
        used = table[table >= 0].long()
        cache["refs"] = torch.bincount(used, minlength=cache["refs"].numel()).int().cuda()
        cache["table"] = table.cuda()
        rows = sum(count)
        kv = randn(rows, 2, H, HD).half()               # K and V side by side, as projected
        begin = [sum(count[:b]) for b in range(B)]
        return dict(case=case, cache=cache, k=kv[:, 0], v=kv[:, 1], begin=ints(begin),
                    count=ints(count), slot=ints(list(range(B))), rows=max(count))
    if case["op"] == "decode":
        rows, H, G, B = _lengths(case), case["heads"], case["group"], case["batch"]
        cache = _cache(g, case, 1, rows, case["beams"], lambda n: n // 8 + B)
        # a page for the blocks that this token fills
        full = [s for s, n in enumerate(rows) if n % PAGE == PAGE - 1]
        free = (cache["refs"] == 0).nonzero().flatten()[:len(full)]
        cache["table"][full, [rows[s] // PAGE for s in full]] = free.int()
        cache["refs"][free] = 1
        qkv = randn(B, (G + 2) * H * HD).half()         # one projection's rows
        q = qkv[:, :G * H * HD].view(B, G * H, HD)
        k = qkv[:, G * H * HD:(G + 1) * H * HD].view(B, H, HD)
        v = qkv[:, (G + 1) * H * HD:].view(B, H, HD)
        cos, sin = _rope(max(rows) + 8)
        return dict(case=case, cache=cache, q=q, k=k, v=v, cos=cos, sin=sin,
                    slot=ints(list(range(B))), rope_row=ints([n + 3 for n in rows]))
    if case["op"] == "fork":
        rows, B, W = _lengths(case), case["batch"], case["beams"]
        cache = _cache(g, case, case["layers"], rows, W, lambda n: n // 8 + 2 * B)
        pick = torch.randint(0, W, (B,), generator=g, device="cuda").int()
        parent = torch.arange(B, device="cuda", dtype=torch.int32) // W * W + pick
        return dict(case=case, cache=cache, slot=ints(list(range(B))), parent=parent)
    rows = _lengths(case)
    cache = _cache(g, case, case["layers"], rows, 1, lambda n: int((case["spare"] - 1) * n) + 1)
    live = sum(n // PAGE for n in rows)
    into = {n: torch.zeros_like(t) for n, t in cache.items()}
    for n, dim in (("codes", 1), ("scales", 1), ("refs", 0)):
        into[n] = into[n].narrow(dim, 0, live + 1).clone()
    return dict(case=case, cache=cache, into=into)


# ------------------------------------------------------------- plain forms
def _quantise(x, code):
    """[..., 32, 128] f32 -> codes and their scales [...]: the smallest power of two that
    brings the block's largest magnitude into the code's range."""
    kind, most = CODES[code]
    top = x.abs().amax((-1, -2))
    m, e = torch.frexp(top)                    # top = m 2^e, 0.5 <= m < 1
    qm, qe = math.frexp(most)
    scale = torch.ldexp(torch.ones_like(top), e - qe + (m > qm).int())
    scale = torch.where(top > 0, scale, torch.ones_like(scale))
    y = x / scale[..., None, None]
    return (y.round() if code == "int8" else y).to(kind), scale


def _plain_store(s):
    c, case = s["cache"], s["case"]
    codes, scales, tails = c["codes"][0], c["scales"][0], c["tails"][0]
    slot, H = s["slot"].long(), case["heads"]
    held, count = c["tokens"][slot].long(), s["count"].long()
    old = held % PAGE                            # rows already in the open block
    blocks = (PAGE - 1 + s["rows"]) // PAGE + 1
    at = torch.arange(blocks * PAGE, device="cuda")
    src = (s["begin"].long()[:, None] + at - old[:, None]).clamp(0, s["k"].shape[0] - 1)
    first = torch.arange(PAGE, device="cuda") < old[:, None]
    done, last = (old + count) // PAGE, (old + count) % PAGE
    fills = torch.arange(blocks, device="cuda") < done[:, None]
    page = c["table"][slot].long().gather(
        1, (held // PAGE)[:, None].add(torch.arange(blocks, device="cuda"))
        .clamp(max=c["table"].shape[1] - 1))
    keep = torch.arange(PAGE, device="cuda") < last[:, None]
    keep &= ~((done == 0)[:, None] & first)       # rows that the tail holds already

    def half(j, x):
        rows = x[src].view(-1, blocks, PAGE, H, HD).transpose(2, 3)
        rows[:, 0] = torch.where(first[:, None, :, None], tails[slot, j], rows[:, 0])
        y, sc = _quantise(rows[fills].float(), case["code"])
        codes[:, j].view(torch.uint8)[page[fills]] = y.view(torch.uint8)
        scales[:, :, j][page[fills]] = sc
        end = rows.gather(1, done.clamp(max=blocks - 1)[:, None, None, None, None]
                          .expand(-1, 1, H, PAGE, HD))[:, 0]
        tails[slot, j] = torch.where(keep[:, None, :, None], end, tails[slot, j])

    half(0, s["k"])
    half(1, s["v"])
    return dict(codes=codes, scales=scales, tails=tails)


def _rotate(x, cos, sin):
    d = torch.arange(HD, device="cuda") % 64
    axis = (d >= 16).long() + (d >= 40).long()
    c = cos.gather(1, axis.expand(1, 1, HD).expand(cos.shape[0], 1, HD))
    n = sin.gather(1, axis.expand(1, 1, HD).expand(sin.shape[0], 1, HD))
    turned = torch.cat([-x[..., 64:], x[..., :64]], -1)
    return x * c + turned * n


def _plain_decode(s):
    c, case = s["cache"], s["case"]
    codes, scales, tails = c["codes"][0], c["scales"][0], c["tails"][0]
    slot, H, G = s["slot"].long(), case["heads"], case["group"]
    B = slot.shape[0]
    n = c["tokens"][slot].long()
    cos, sin = (t[:, s["rope_row"].long()].transpose(0, 1) for t in (s["cos"], s["sin"]))
    q = _rotate(s["q"].float(), cos, sin).view(B, H, G, HD)
    b = torch.arange(B, device="cuda")
    tails[slot, 0, :, n % PAGE] = _rotate(s["k"].float(), cos, sin).half()
    tails[slot, 1, :, n % PAGE] = s["v"]
    wide = c["table"].shape[1]
    page = c["table"][slot].clamp(min=0).long()
    open_ = tails[slot].float()

    def rows(j):
        x = codes[:, j][page.view(-1)].float()
        x *= scales[:, :, j][page.view(-1)][..., None, None]
        x = x.view(B, wide, H, PAGE, HD).transpose(1, 2).reshape(B, H, wide * PAGE, HD)
        return torch.cat([x, open_[:, j]], 2)

    at = torch.arange((wide + 1) * PAGE, device="cuda")
    live = (at < (n // PAGE * PAGE)[:, None]) | ((at >= wide * PAGE)
                                                 & (at - wide * PAGE <= (n % PAGE)[:, None]))
    w = torch.matmul(q, rows(0).transpose(2, 3)) / math.sqrt(HD)
    w = w.masked_fill(~live[:, None, None], -math.inf)
    w = torch.exp(w - w.amax(-1, keepdim=True))
    w = w / w.sum(-1, keepdim=True)
    v = rows(1).masked_fill(~live[:, None, :, None], 0.0)
    out = torch.matmul(w, v).view(B, H * G, HD).half()
    closed = n % PAGE == PAGE - 1
    y, sc = _quantise(open_[closed], case["code"])
    into = page[b, (n // PAGE).clamp(max=wide - 1)][closed]
    codes.view(torch.uint8)[into] = y.view(torch.uint8)
    scales[into] = sc.transpose(1, 2)
    return dict(out=out, codes=codes, scales=scales, tails=tails)


def _plain_fork(s):
    c = s["cache"]
    slot, parent = s["slot"].long(), s["parent"].long()
    table, tokens, refs, tails = c["table"], c["tokens"], c["refs"], c["tails"]
    B, S = slot.shape[0], tokens.shape[0]
    b = torch.arange(B, device="cuda")
    eldest = torch.full((B,), B, device="cuda").scatter_reduce(0, parent, b, "amin")
    keeps = eldest[parent] == b                   # the first child stays in its parent's slot
    kept = torch.zeros(S, dtype=torch.bool, device="cuda").index_fill(0, slot[parent], True)
    gone = torch.zeros(S, dtype=torch.bool, device="cuda").index_fill(0, slot, True) & ~kept
    free = (gone | (~kept & (tokens == 0))).nonzero().flatten()
    free = torch.cat([free, free.new_zeros(1)])    # never empty; the last is not taken
    new = torch.where(keeps, slot[parent], free[((~keeps).long().cumsum(0) - 1).clamp(min=0)])
    # dropped sequences give their pages back
    held = table[gone]
    refs -= torch.bincount(held[held >= 0].long(), minlength=refs.shape[0]).int()
    table[gone] = -1
    tokens[gone] = 0
    # the other children share the full pages and copy the open block
    src, dst = slot[parent][~keeps], new[~keeps]
    full = torch.arange(table.shape[1], device="cuda") < (tokens[src] // PAGE)[:, None]
    row = torch.where(full, table[src], -1)
    refs += torch.bincount(row[full].long(), minlength=refs.shape[0]).int()
    table[dst] = row
    tokens[dst] = tokens[src]
    open_ = torch.arange(PAGE, device="cuda") < (tokens[src] % PAGE)[:, None]
    tails[:, dst] = torch.where(open_[None, :, None, None, :, None], tails[:, src], tails[:, dst])
    # a page for every block that the next row fills, the lowest free ones
    n = tokens[new].long()
    needs = (n % PAGE == PAGE - 1) & (table[new].gather(1, (n // PAGE)[:, None])[:, 0] < 0)
    given = (refs == 0).nonzero().flatten()[:int(needs.sum())]
    table[new[needs], (n // PAGE)[needs]] = given.int()
    refs[given] = 1
    s["slot"] = new.int()
    return dict(slot=s["slot"], table=table, tokens=tokens, refs=refs, tails=tails)


def _plain_compact(s):
    c, d = s["cache"], s["into"]
    live = (c["refs"] > 0).nonzero().flatten()
    to = torch.full_like(c["refs"], -1)
    to[live] = torch.arange(live.shape[0], device="cuda", dtype=torch.int32)
    n = live.shape[0]
    d["codes"].view(torch.uint8)[:, :n] = c["codes"].view(torch.uint8)[:, live]
    d["scales"][:, :n] = c["scales"][:, live]
    d["refs"].zero_()
    d["refs"][:n] = c["refs"][live]
    d["table"].copy_(torch.where(c["table"] >= 0, to[c["table"].clamp(min=0).long()], -1))
    d["tokens"].copy_(c["tokens"])
    open_ = torch.arange(PAGE, device="cuda") < (c["tokens"] % PAGE)[:, None]
    d["tails"].copy_(torch.where(open_[None, :, None, None, :, None], c["tails"], d["tails"]))
    return dict(d)


def _plain_beam(s):
    case = s["case"]
    B, W, K = case["batch"], case["beams"], case["topk"]
    x = s["logits"].double()
    top = x.amax(1, keepdim=True)
    lse = top + torch.exp(x - top).sum(1, keepdim=True).log()
    best, token = torch.sort(s["logits"], dim=1, descending=True, stable=True)
    best, token = best[:, :K].double(), token[:, :K]
    k = best.shape[1]
    score = (s["scores"].double().view(B * W, 1) - lse + best).view(B, W * k)
    score, at = torch.sort(score, dim=1, descending=True, stable=True)
    at = at[:, :K]
    return dict(score=score[:, :K].float(), beam=(at // k).int(),
                token=token.reshape(B, W * k).gather(1, at).int())


def _plain(s):
    return {"store": _plain_store, "decode": _plain_decode, "fork": _plain_fork,
            "compact": _plain_compact, "beam": _plain_beam}[s["case"]["op"]](s)


# ------------------------------------------------------ the framework's calls
def _handles(s):
    """What a program makes once for its cache and keeps: the cache objects and a workspace."""
    import os
    import sys
    package = os.path.join(os.getcwd(), "paddleocr-vl-webgpu_b200")
    if package not in sys.path:
        sys.path.insert(0, package)
    from pvlc_b200 import kv8, ops
    case, got = s["case"], {"kv8": kv8, "ops": ops}
    if case["op"] == "beam":
        got["ws"] = ops.BeamWorkspace(case["batch"], case["beams"], case["vocab"], case["topk"])
    else:
        got["cache"] = kv8.Cache(**s["cache"])
        if "into" in s:
            got["into"] = kv8.Cache(**s["into"])
        got["ws"] = kv8.Workspace(got["cache"], case.get("batch", 1),
                                  case["heads"] * case.get("group", 1))
    return got


def _ours(s):
    if "handles" not in s:
        s["handles"] = _handles(s)
    h, op, c = s["handles"], s["case"]["op"], s.get("cache")
    kv8 = h["kv8"]
    if op == "store":
        kv8.store(h["cache"], 0, s["k"], s["v"], s["begin"], s["count"], s["slot"], s["rows"], h["ws"])
        return dict(codes=c["codes"][0], scales=c["scales"][0], tails=c["tails"][0])
    if op == "decode":
        out = kv8.decode(h["cache"], 0, s["q"], s["k"], s["v"], s["cos"], s["sin"], s["slot"],
                         h["ws"], rope_row=s["rope_row"])
        return dict(out=out, codes=c["codes"][0], scales=c["scales"][0], tails=c["tails"][0])
    if op == "fork":
        s["slot"] = kv8.fork(h["cache"], s["slot"], s["parent"], h["ws"])
        kv8.grow(h["cache"], s["slot"], h["ws"], ahead=1)
        return dict(slot=s["slot"], table=c["table"], tokens=c["tokens"], refs=c["refs"],
                    tails=c["tails"])
    if op == "compact":
        kv8.compact(h["cache"], h["into"], h["ws"])
        return dict(s["into"])
    score, beam, token = h["ops"].beam_topk(s["logits"], s["scores"], s["case"]["topk"], h["ws"])
    return dict(score=score, beam=beam, token=token)


def run(state):
    return _ours(state) if own else _plain(state)


# ------------------------------------------------------------------- work
def work(case):
    """Bytes that a pass cannot do without, and its operations."""
    op = case["op"]
    if op == "beam":
        n = case["batch"] * case["beams"] * case["vocab"]
        return dict(bytes=n * (2 if case["dtype"] == "f16" else 4) + case["batch"] * (case["beams"] * 4
                    + case["topk"] * 12), flops=3 * n)
    rows, H = _lengths(case), case["heads"]
    row8, row16 = 2 * H * HD, 4 * H * HD          # a row's K and V in 8 and in 16 bits
    if op == "store":
        held = case["held"]
        old, total = held % PAGE, 0
        for c in rows:
            filled = (old + c) // PAGE * PAGE
            total += c * row16 + filled * row8 + filled // PAGE * H * 8
            total += (old if filled else 0) * row16 + ((old + c - filled) if filled else c) * row16
        return dict(bytes=total, flops=3 * sum(rows) * 2 * H * HD)
    if op == "decode":
        G, W, total, flops = case["group"], case["beams"], 0, 0
        for b, n in enumerate(rows):
            full = n // PAGE
            mine = full if b % W == 0 else min(full, 1)      # beams share all but the last page
            total += mine * (PAGE * row8 + H * 8) + (n % PAGE + 2) * row16 + full * 4
            total += 2 * G * H * HD * 2 + HD * 8
            if n % PAGE == PAGE - 1:
                total += PAGE * row8 + H * 8
            flops += 4 * G * H * HD * (n + 1)
        return dict(bytes=total, flops=flops)
    if op == "fork":
        # about (1 - 1/W)^W of a request's beams end, and as many are copied
        W, L = case["beams"], case["layers"]
        part = (1 - 1 / W) ** W
        total = sum(part * (2 * L * (n % PAGE) * row16 + 3 * (n // PAGE) * 4) for n in rows)
        return dict(bytes=int(total) + 16 * case["batch"], flops=0)
    L, total = case["layers"], 0
    for n in rows:
        total += 2 * L * (n // PAGE * (PAGE * row8 + H * 8) + n % PAGE * row16) + 2 * (n // PAGE) * 4
    return dict(bytes=total, flops=0)


# ------------------------------------------------------- 64-bit definitions
def _exact_codes(x, code):
    """Codes (as numbers) and the scale of one [32, 128] block of doubles."""
    most = CODES[code][1]
    top = float(x.abs().max())
    scale = 1.0
    if top > 0:
        scale = 2.0 ** math.floor(math.log2(top / most))
        while top > most * scale:
            scale *= 2
        while top <= most * scale / 2:
            scale /= 2
    y = x / scale
    if code == "int8":
        return torch.round(y), scale
    step = torch.exp2(torch.floor(torch.log2(y.abs().clamp(min=2.0 ** -6))) - 3)
    return torch.round(y / step) * step, scale


def _exact_rotated(x, angle_cos, angle_sin, row):
    y = x.clone()
    for d in range(64):
        axis = 0 if d < 16 else 1 if d < 40 else 2
        for e, p, sign in ((d, d + 64, -1.0), (d + 64, d, 1.0)):
            y[:, e] = x[:, e] * angle_cos[axis, row, e] + sign * x[:, p] * angle_sin[axis, row, e]
    return y


def exact(case, seed):
    op = case["op"]
    if op in ("fork", "compact"):
        return None                                # whole numbers and copies
    s = prepare(case, seed)
    if op == "beam":
        B, W, K = case["batch"], case["beams"], case["topk"]
        got = []
        for r in range(B):
            x = s["logits"][r * W:(r + 1) * W].double()
            p = x - torch.logsumexp(x, 1, keepdim=True) + s["scores"][r].double()[:, None]
            got.append(p.flatten().topk(K).values)
        return dict(score=torch.stack(got), beam=None, token=None)
    c = s["cache"]
    codes, scales = c["codes"][0].double(), c["scales"][0].double()
    tails = c["tails"][0].double()
    table, tokens = c["table"].cpu(), c["tokens"].cpu().tolist()
    H = case["heads"]
    if op == "store":
        count = _lengths(case)
        if sum(count) * H > 20000:
            return None
        at = 0
        for b, n in enumerate(count):
            held = tokens[b]
            for j, x in ((0, s["k"]), (1, s["v"])):
                for h in range(H):
                    rows = torch.cat([tails[b, j, h, :held % PAGE], x[at:at + n, h].double()])
                    full = rows.shape[0] // PAGE
                    for f in range(full):
                        page = int(table[b, held // PAGE + f])
                        y, sc = _exact_codes(rows[f * PAGE:(f + 1) * PAGE], case["code"])
                        codes[page, j, h], scales[page, h, j] = y, sc
                    left = rows[full * PAGE:]
                    tails[b, j, h, :left.shape[0]] = left
            at += n
        return dict(codes=codes if case["code"] == "e4m3" else None, scales=scales, tails=tails)
    rows, G = _lengths(case), case["group"]
    if case["batch"] * H > 600:
        return None
    out = torch.empty(s["q"].shape, dtype=torch.float64, device="cuda")
    q, k, v = s["q"].double(), s["k"].double(), s["v"].double()
    cos, sin, at = s["cos"].double(), s["sin"].double(), s["rope_row"].tolist()
    closed = []
    for b, n in enumerate(rows):
        new = _exact_rotated(torch.cat([k[b], q[b]]), cos, sin, at[b])
        tails[b, 0, :, n % PAGE] = new[:H].half().double()     # the cache holds fp16 rows
        tails[b, 1, :, n % PAGE] = v[b]
        page = table[b, :n // PAGE].long().cuda()
        for h in range(H):
            keys, values = (torch.cat([(codes[page, j, h] * scales[page, h, j, None, None]).view(-1, HD),
                                       tails[b, j, h, :n % PAGE + 1]]) for j in (0, 1))
            w = torch.softmax(new[H + h * G:H + (h + 1) * G] @ keys.T / math.sqrt(HD), -1)
            out[b, h * G:(h + 1) * G] = w @ values
        if n % PAGE == PAGE - 1:
            closed.append((b, int(table[b, n // PAGE])))
    for b, page in closed:
        for j in (0, 1):
            for h in range(H):
                codes[page, j, h], scales[page, h, j] = _exact_codes(tails[b, j, h], case["code"])
    return dict(out=out, codes=codes if case["code"] == "e4m3" else None, scales=scales,
                tails=tails)
