"""Plain 64-bit restatement of the 8-bit paged KV cache, for the tests: numpy arrays, one
sequence, block and head at a time."""
import math

import numpy as np
import torch

PAGE, HD = 32, 128
MOST = {"e4m3": 448.0, "int8": 127.0}
DTYPE = {"e4m3": torch.float8_e4m3fn, "int8": torch.int8}


def quantise(x, code):
    """[32, 128] block -> (code values, scale)."""
    x = np.asarray(x, np.float64)
    if not np.isfinite(x).all():
        return np.zeros_like(x), math.nan
    top, scale = np.abs(x).max(), 1.0
    if top > 0:
        e = -60
        while top > MOST[code] * 2.0 ** e:
            e += 1
        scale = 2.0 ** e
    y = x / scale
    if code == "int8":
        return np.rint(y), scale
    # e4m3: three fraction bits, exponents -6 .. 8, spacing 2^-9 below 2^-6
    mag = np.maximum(np.abs(y), 2.0 ** -6)
    step = 2.0 ** (np.floor(np.log2(mag)) - 3)
    return np.rint(y / step) * step, scale


def rotate(x, cos, sin, row):
    """[heads, 128] fp16 values rotated as the cache keeps them: f32 products and one f32 sum,
    rounded to fp16."""
    x = x.astype(np.float32)
    d = np.arange(HD) % 64
    axis = (d >= 16).astype(int) + (d >= 40)
    c, s = cos[axis, row, np.arange(HD)], sin[axis, row, np.arange(HD)]
    y = np.concatenate([-x[:, 64:], x[:, :64]], 1)
    return (x * c + y * s).astype(np.float16)


class Ref:
    """Cache state on the host: codes as their values."""

    def __init__(self, cache, code):
        self.code = code
        self.codes = cache.codes.float().cpu().numpy().astype(np.float64)
        self.scales = cache.scales.cpu().numpy().astype(np.float64)
        self.tails = cache.tails.cpu().numpy()
        self.table = cache.table.cpu().numpy().copy()
        self.tokens = cache.tokens.cpu().numpy().copy()
        self.refs = cache.refs.cpu().numpy().copy()
        self.H = self.codes.shape[3]

    def same(self, cache, pages=True):
        np.testing.assert_array_equal(cache.table.cpu().numpy(), self.table)
        np.testing.assert_array_equal(cache.tokens.cpu().numpy(), self.tokens)
        np.testing.assert_array_equal(cache.refs.cpu().numpy(), self.refs)
        np.testing.assert_array_equal(cache.tails.cpu().numpy().view(np.uint16),
                                      self.tails.view(np.uint16))
        if pages:
            np.testing.assert_array_equal(cache.scales.cpu().numpy(), self.scales)
            np.testing.assert_array_equal(cache.codes.float().cpu().numpy(), self.codes)

    def close(self, layer, slot, block, rows):
        """rows [2, H, 32, 128] become the slot's page of that block."""
        page = self.table[slot, block]
        for j in range(2):
            for h in range(self.H):
                y, s = quantise(rows[j, h], self.code)
                self.codes[layer, page, j, h] = y
                self.scales[layer, page, h, j] = s

    def store(self, layer, slot, k, v):
        """k, v [n, H, 128] fp16 behind the slot's rows (tokens is left)."""
        n = int(self.tokens[slot])
        tail = self.tails[layer, slot]                        # [2, H, 32, 128]
        block = tail.copy()
        for i in range(len(k)):
            r = (n + i) % PAGE
            block[0, :, r], block[1, :, r] = k[i], v[i]
            if r == PAGE - 1:
                self.close(layer, slot, (n + i) // PAGE, block)
        left = (n + len(k)) % PAGE
        keep = n % PAGE if n // PAGE == (n + len(k)) // PAGE else 0
        tail[:, :, keep:left] = block[:, :, keep:left]

    def rows(self, layer, slot, h, n):
        """The n rows of a head as the cache holds them: K, V [n, 128] doubles."""
        out = []
        for j in range(2):
            pages = self.table[slot, :n // PAGE]
            full = (self.codes[layer, pages, j, h] *
                    self.scales[layer, pages, h, j][:, None, None]).reshape(-1, HD)
            out.append(np.concatenate([full, self.tails[layer, slot, j, h, :n % PAGE]
                                       .astype(np.float64)]))
        return out

    def decode(self, layer, slot, q, k, v, cos, sin, row):
        """Append and attend: (out [QH, 128], elementwise error bound of an fp16 kernel)."""
        n = int(self.tokens[slot])
        tail = self.tails[layer, slot]
        tail[0, :, n % PAGE] = rotate(k, cos, sin, row)
        tail[1, :, n % PAGE] = v
        G = q.shape[0] // self.H
        q32 = q.astype(np.float64)
        d = np.arange(HD) % 64
        axis = (d >= 16).astype(int) + (d >= 40)
        c = cos[axis, row, np.arange(HD)].astype(np.float64)
        s = sin[axis, row, np.arange(HD)].astype(np.float64)
        q64 = q32 * c + np.concatenate([-q32[:, 64:], q32[:, :64]], 1) * s
        out, tol = np.empty((len(q), HD)), np.empty((len(q), HD))
        for h in range(self.H):
            pages = self.table[slot, :n // PAGE]
            keys, vals = [], []
            for j, got in ((0, keys), (1, vals)):
                full = (self.codes[layer, pages, j, h] *
                        self.scales[layer, pages, h, j][:, None, None]).reshape(-1, HD)
                got.append(np.concatenate([full, tail[j, h, :n % PAGE + 1].astype(np.float64)]))
            K, V = keys[0], vals[0]
            for i in range(h * G, (h + 1) * G):
                w = K @ q64[i] / math.sqrt(HD)
                p = np.exp(w - w.max())
                p /= p.sum()
                out[i] = p @ V
                # The kernel rounds the rotated q to fp16 (2^-11 of each value), which moves
                # every score by at most e = 2^-11 max_r sum|q||k_r| / sqrt(128); f32 products,
                # sums and exponents move it by less than e / 64 + 2^-18.  A weight moves by a
                # factor within exp(+-2 e) of 1, its fp16 rounding by 2^-11; weights are kept
                # to 2^-39 of the largest.  The result is rounded to fp16 (2^-11, or 2^-25).
                e = (2.0 ** -11 * (1 + 1 / 64)
                     * (np.abs(K) @ np.abs(q64[i])).max() / math.sqrt(HD) + 2.0 ** -18)
                spread = p @ np.abs(V) + 2.0 ** -39 * np.abs(V).sum(0)
                tol[i] = (np.expm1(2 * e) + 2.0 ** -11) * spread * 1.01 + \
                    2.0 ** -11 * np.abs(out[i]) + 2.0 ** -25
        if n % PAGE == PAGE - 1:
            self.close(layer, slot, n // PAGE, tail)
        return out, tol

    def grow(self, slots, advance, ahead):
        for s, a in zip(slots, advance):
            if s >= 0:
                self.tokens[s] += a
        short = False
        for s, a in zip(slots, ahead):
            if s < 0:
                continue
            for j in range(self.tokens[s] // PAGE, (self.tokens[s] + a) // PAGE):
                if self.table[s, j] < 0:
                    free = np.flatnonzero(self.refs == 0)
                    if len(free) == 0:
                        short = True
                        continue
                    self.table[s, j] = free[0]
                    self.refs[free[0]] = 1
        return short

    def fork(self, slots, parent, advance=0):
        for s in slots:
            if s >= 0:
                self.tokens[s] += advance
        src = [slots[m] if m >= 0 else -1 for m in parent]
        kept = set(x for x in src if x >= 0)
        named = set(s for s in slots if s >= 0)
        free = [s for s in range(len(self.tokens))
                if s not in kept and (s in named or self.tokens[s] == 0)]
        new, taken, moves = [], set(), []
        for x in src:
            if x < 0:
                new.append(-1)
            elif x not in taken:
                taken.add(x)
                new.append(x)
            elif free:
                new.append(free.pop(0))
                moves.append((new[-1], x))
            else:
                new.append(-1)
        def drop(s):
            for p in self.table[s][self.table[s] >= 0]:
                self.refs[p] -= 1
            self.table[s] = -1
            self.tokens[s] = 0
        for s in named - kept:
            drop(s)
        for to, x in moves:
            drop(to)
            n = self.tokens[x]
            self.tokens[to] = n
            self.table[to, :n // PAGE] = self.table[x, :n // PAGE]
            for p in self.table[to, :n // PAGE]:
                self.refs[p] += 1
            self.tails[:, to, :, :, :n % PAGE] = self.tails[:, x, :, :, :n % PAGE]
        return new


def rope_tables(rows, seed=0):
    """[3, rows, 128] f32 tables with three different axes."""
    rng = np.random.default_rng(seed)
    freq = 500000.0 ** (-np.arange(0, HD, 2) / HD)
    pos = np.stack([np.arange(rows) * f + rng.integers(0, 9) for f in (1.0, 0.5, 0.25)])
    ang = pos[:, :, None] * freq
    ang = np.concatenate([ang, ang], 2)
    return np.cos(ang).astype(np.float32), np.sin(ang).astype(np.float32)


def filled_cache(kv8, code, lengths, H=2, layers=1, seed=0, spare=3, poison=True, room=3,
                 share=1):
    """A cache whose slot s holds lengths[s] random rows, its pages in random order, rows
    that are no sequence's NaN (codes 0x7f / -128 with scale NaN in free pages)."""
    rng = np.random.default_rng(seed)
    S = len(lengths)
    M = max([n // PAGE for n in lengths]) + room
    full = sum(n // PAGE for n in lengths)
    P = full + spare
    c = kv8.Cache.empty(layers, P, S, M, H, DTYPE[code])
    order = rng.permutation(P)
    table, at = np.full((S, M), -1, np.int32), 0
    for s, n in enumerate(lengths):
        table[s, :n // PAGE] = order[at:at + n // PAGE]
        at += n // PAGE
    scale = 2.0 ** rng.integers(-8, -4, (layers, P, H, 2))
    vals = rng.standard_normal((layers, P, 2, H, PAGE, HD))
    y = vals / scale.transpose(0, 1, 3, 2)[..., None, None]
    if code == "int8":
        codes = torch.from_numpy(np.clip(np.rint(y), -127, 127)).to(torch.int8)
    else:
        codes = torch.from_numpy(np.clip(y, -448, 448)).float().to(torch.float8_e4m3fn)
    tails = rng.standard_normal((layers, S, 2, H, PAGE, HD)).astype(np.float16)
    if poison:
        free = order[at:]
        scale[:, free] = np.nan
        codes.view(torch.uint8)[:, free] = 0x7f
        for s, n in enumerate(lengths):
            tails[:, s, :, :, n % PAGE:] = np.nan
    c.codes.view(torch.uint8).copy_(codes.view(torch.uint8))
    c.scales.copy_(torch.from_numpy(scale))
    c.tails.copy_(torch.from_numpy(tails))
    c.table.copy_(torch.from_numpy(table))
    c.tokens.copy_(torch.tensor(lengths, dtype=torch.int32))
    refs = np.bincount(table[table >= 0], minlength=P).astype(np.int32)
    c.refs.copy_(torch.from_numpy(refs))
    return c


def give_pages(c, slots, rows=1):
    """Pages for the blocks that the next `rows` rows of the slots fill."""
    table, refs, tokens = c.table.cpu(), c.refs.cpu(), c.tokens.cpu()
    free = iter((refs == 0).nonzero().flatten().tolist())
    for s in slots:
        for j in range(int(tokens[s]) // PAGE, (int(tokens[s]) + rows) // PAGE):
            if table[s, j] < 0:
                p = next(free)
                table[s, j] = p
                refs[p] = 1
    c.table.copy_(table)
    c.refs.copy_(refs)
