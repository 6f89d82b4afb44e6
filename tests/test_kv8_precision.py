"""Scores of the 8-bit decode where they are small differences of large products: queries with
a common part, queries beyond fp16's range.

The rotated q goes to the tensor cores as its fp16 rounding and the rest of it, the codes as
the numbers they are, so what is left of an error is f32 arithmetic's, and the bound below counts
that and nothing else.  The host tests run the same bound over numpy emulations of the scores:
the kernel's own way is within it; q rounded to fp16 alone, and int8 codes that carry a bias
through the sums, are not."""
import math

import numpy as np
import pytest
import torch

import kv8_ref as R

PAGE, HD = 32, 128
H = 2
LENGTHS = [200, 70, 33, 0, 95 + 3]

# q: `mean` in every dim, and what fp16 leaves of N(0, 1) beside it; cos, sin: the rotation (the
# same for every dim and axis); keys: N(0, 1) times `keys`, with `paired` dim 2 i + 1 the negative
# of dim 2 i, so that the common part of q adds up to nothing.
CASES = {
    "common part 512": dict(mean=512.0, cos=0.70710678, sin=0.0, keys=4.0, paired=True),
    "common part 32": dict(mean=32.0, cos=0.70710678, sin=0.0, keys=4.0, paired=True),
    "beyond fp16": dict(mean=60000.0, cos=1.0, sin=-0.4, keys=2.0 ** -15, paired=False),
}


class Case:
    """Sequences of LENGTHS rows and one token of each, on the host."""

    def __init__(self, code, group, name, seed=1):
        c = CASES[name]
        rng = np.random.default_rng(seed)
        self.code, self.G, self.QH = code, group, H * group
        self.cos, self.sin = np.float32(c["cos"]), np.float32(c["sin"])
        n = lambda *s: rng.standard_normal(s)  # noqa: E731

        def paired(x):
            x = (x * c["keys"]).astype(np.float16)
            if c["paired"]:
                x[..., 1::2] = -x[..., ::2]
            return x
        B = len(LENGTHS)
        self.q = (c["mean"] + n(B, self.QH, HD)).astype(np.float16)
        self.k, self.v = paired(n(B, H, HD)), n(B, H, HD).astype(np.float16)
        # rows as they went in: every page quantised, the open block fp16
        self.seqs = []
        for b, rows in enumerate(LENGTHS):
            kv = np.stack([paired(n(rows, H, HD)), n(rows, H, HD).astype(np.float16)])
            pages = []
            for p in range(rows // PAGE):
                blk = kv[:, p * PAGE:(p + 1) * PAGE]
                # pages of different sizes: their scales differ
                blk = (blk * np.float16(2.0 ** -(p % 3))).astype(np.float16)
                pages.append([[R.quantise(blk[j, :, h], code) for h in range(H)] for j in (0, 1)])
            self.seqs.append((pages, kv[:, rows // PAGE * PAGE:]))
        y = self.k.astype(np.float32)
        self.k_rot = (y * self.cos + np.concatenate([-y[..., 64:], y[..., :64]], -1) * self.sin
                      ).astype(np.float16)

    def rows(self, b, h, j):
        """Codes [n + 1, 128] (the open block's rows as they are) and their scales, K or V."""
        pages, tail = self.seqs[b]
        codes = [p[j][h][0] for p in pages] + [tail[j, :, h].astype(np.float64),
                                               (self.k_rot, self.v)[j][b, h:h + 1].astype(np.float64)]
        scale = [np.full(PAGE, p[j][h][1]) for p in pages] + [np.ones(len(tail[j]) + 1)]
        return np.concatenate(codes), np.concatenate(scale)

    def want(self, b, i, scores=None):
        """Output of head i of sequence b in 64 bits, and how far a kernel may be from it; or
        the output that these scores give."""
        h = i // self.G
        (kc, ks), (vc, vs) = self.rows(b, h, 0), self.rows(b, h, 1)
        V = vc * vs[:, None]
        x = self.q[b, i].astype(np.float64)
        y = np.concatenate([-x[64:], x[:64]])
        c, s = float(self.cos), float(self.sin)
        q = x * c + y * s
        unit = ks / math.sqrt(HD)
        w = (kc @ q) * unit if scores is None else scores
        p = np.exp(w - w.max())
        p /= p.sum()
        out = p @ V
        # The rotation: two f32 products and their sum, 2^-24 each.  q as an fp16 number (cut off
        # at 65504) and the rest as another: the rest's rounding, 2^-11 of it, or 2^-25.
        rest = q - half(q)
        dq = 2.0 ** -23 * (np.abs(x * c) + np.abs(y * s)) + 2.0 ** -11 * np.abs(rest) + 2.0 ** -25
        # A matrix instruction adds 16 products to its accumulator, each with 23 bits or more behind
        # the largest of the 17.  A lane brings four neighbouring dims at a time, so no sum is
        # above the groups of four's and no product above the largest.  A page's row takes 8
        # instructions with q, 8 with the rest in an accumulator of its own, and their sum; a row
        # of the open block all 16 in one.
        prod = kc * q
        largest = np.abs(prod.reshape(len(kc), 32, 4).sum(2)).sum(1) + np.abs(prod).max(1)
        low = np.abs(kc) @ np.abs(rest)
        steps = np.where(np.arange(len(kc)) < len(self.seqs[b][0]) * PAGE, 8 * 17, 16 * 17) + 1
        # f32 scaling of the score and of the exponent, in powers of two: 2^-22 of what it is
        e = (np.abs(kc) @ dq + steps * 2.0 ** -23 * (largest + low)) * unit \
            + 2.0 ** -22 * (np.abs(w).max() + 24)
        # With scores off by at most e_r, out moves by sum p_r (exp(+-e_r) - 1) (V_r - out) over a
        # sum of weights that is within exp(+-max e) of 1.
        spread = p @ np.abs(V) + 2.0 ** -39 * np.abs(V).sum(0)
        moved = math.exp(e.max()) * ((p * np.expm1(e)) @ np.abs(V - out))
        # A weight's fp16 rounding is 2^-11 (weights below 2^-39 of the largest may go), f32 sums
        # over the rows are within 2^-13; the result is rounded to fp16.
        tol = moved + (2.0 ** -11 + 2.0 ** -13) * (spread + moved) * 1.01 + 2.0 ** -11 * np.abs(out) \
            + 2.0 ** -25
        return out, tol

    def emulated(self, b, i, how):
        """The scores of head i as f32 sums of 16 products at a time make them."""
        kc, ks = self.rows(b, i // self.G, 0)
        full = len(self.seqs[b][0]) * PAGE
        x = self.q[b, i].astype(np.float32)
        y = np.concatenate([-x[64:], x[:64]])
        q = (x * self.cos + y * self.sin).astype(np.float32)
        hi = half(q)
        parts = [hi] if how == "half q" else [hi, (q - hi).astype(np.float16).astype(np.float64)]
        bias = np.zeros(len(kc))
        if how == "biased":
            bias[:full] = 1152.0
        s = np.zeros(len(kc), np.float32)
        for part in parts:
            acc = np.zeros(len(kc), np.float32)
            for k in range(0, HD, 16):
                acc = (acc + (kc[:, k:k + 16] + bias[:, None]) @ part[k:k + 16]).astype(np.float32)
            s += acc
        s = s - np.float32(q.sum(dtype=np.float32)) * bias.astype(np.float32)
        return s.astype(np.float64) * ks / math.sqrt(HD)


def half(q):
    return np.clip(np.clip(q, -65504, 65504).astype(np.float16).astype(np.float64), -65504, 65504)


def worst(case, how):
    """The largest error over its bound, of outputs from emulated scores."""
    top = 0.0
    for b in range(len(LENGTHS)):
        for i in range(case.QH):
            want, tol = case.want(b, i)
            got, _ = case.want(b, i, case.emulated(b, i, how))
            top = max(top, float((np.abs(got - want) / tol).max()))
    return top


@pytest.mark.parametrize("name", CASES)
@pytest.mark.parametrize("code", ["e4m3", "int8"])
def test_the_bound_holds_for_split_queries(code, name):
    assert worst(Case(code, 8, name), "split") < 1


@pytest.mark.parametrize("code", ["e4m3", "int8"])
@pytest.mark.parametrize("name", ["common part 512", "beyond fp16"])
def test_the_bound_shows_a_lost_rest(code, name):
    assert worst(Case(code, 8, name), "half q") > 2


def test_the_bound_shows_biased_codes():
    assert worst(Case("int8", 8, "common part 512"), "biased") > 2


@pytest.mark.gpu
@pytest.mark.parametrize("name", CASES)
@pytest.mark.parametrize("group", [8, 16, 3])
@pytest.mark.parametrize("code", ["e4m3", "int8"])
def test_decode(cuda_lib, code, group, name):
    from pvlc_b200 import kv8
    case = Case(code, group, name)
    B, most = len(LENGTHS), max(LENGTHS) // PAGE + 1
    total = sum(n // PAGE for n in LENGTHS) + 1
    c = kv8.Cache.empty(1, total, B, most, H, R.DTYPE[code])
    codes, scales = np.zeros((total, 2, H, PAGE, HD)), np.ones((total, H, 2), np.float32)
    tails = np.full((B, 2, H, PAGE, HD), np.nan, np.float16)
    table, at = np.full((B, most), -1, np.int32), 0
    for b, (pages, tail) in enumerate(case.seqs):
        for p, page in enumerate(pages):
            table[b, p] = at
            for j in (0, 1):
                for h in range(H):
                    codes[at, j, h], scales[at, h, j] = page[j][h]
            at += 1
        tails[b, :, :, :tail.shape[1]] = tail.transpose(0, 2, 1, 3)
    c.codes[0].view(torch.uint8).copy_(torch.from_numpy(codes).float().to(c.codes.dtype)
                                       .view(torch.uint8))
    c.scales[0].copy_(torch.from_numpy(scales))
    c.tails[0].copy_(torch.from_numpy(tails))
    c.table.copy_(torch.from_numpy(table))
    c.tokens.copy_(torch.tensor(LENGTHS, dtype=torch.int32))
    c.refs[:at] = 1
    ws = kv8.Workspace(c, B, case.QH)
    q, k, v = (torch.from_numpy(x).cuda() for x in (case.q, case.k, case.v))
    cos, sin = (torch.full((3, 1, HD), float(x), device="cuda") for x in (case.cos, case.sin))
    row = torch.zeros(B, dtype=torch.int32, device="cuda")
    out = kv8.decode(c, 0, q, k, v, cos, sin, None, ws, rope_row=row).cpu().numpy()
    assert ws.errors() == 0
    for b in range(B):
        for i in range(case.QH):
            want, tol = case.want(b, i)
            off = np.abs(out[b, i].astype(np.float64) - want)
            assert (off <= tol).all(), (LENGTHS[b], i, float((off / tol).max()))
