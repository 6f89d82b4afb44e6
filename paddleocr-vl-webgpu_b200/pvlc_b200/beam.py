"""Beam search over the 8-bit paged KV cache: OcrEngine.generate_beam.

All of a step runs on the device, captured in one CUDA graph: the decoder layers with
kv8.decode, the LM head, ops.beam_topk over each request's beams, the bookkeeping of ended and
live hypotheses (a few elementwise operations on [requests, 2 * beams]), kv8.fork to give every
surviving beam its cache, and kv8.grow for the next row's page.  The beams of a request share
its prompt's pages and whatever full pages of their history they have in common.  The host
reads the chosen tokens once a chunk and traces the hypotheses back at the end.

A step takes the 2 * beams best continuations of a request.  Those of the first `beams` that
end (EOS) become hypotheses, scored by log-probability over length ** length_penalty (the
length counts the EOS); the best `beams` hypotheses are kept.  The first `beams` that do not
end go on.  A request is done when it has `beams` hypotheses and its best live beam, scored at
its present length, is no better than the worst of them; its sequences then leave the cache.
At max_new_tokens the live beams of the others become hypotheses too.
"""
from __future__ import annotations

import math

import numpy as np
import torch
import torch.nn.functional as F

from . import abi, greedy, kv8, ops, positions


class BeamDecoder:
    """The buffers and the step graph of a batch shape: `requests` x `beams` sequences of up
    to `rows` cache rows."""

    def __init__(self, eng, requests: int, beams: int, rows: int, pages: int, cache_dtype,
                 length_penalty: float):
        c, dev = eng.cfg, eng.device
        self.eng, self.B, self.W, self.rows = eng, requests, beams, rows
        self.N = N = requests * beams
        self.penalty = float(length_penalty)
        self.cache = kv8.Cache.empty(c.decoder_layers, pages, N, rows // kv8.PAGE + 1,
                                     c.kv_heads, cache_dtype, dev)
        self.ws = kv8.Workspace(self.cache, N, c.query_heads)
        self.topk = 2 * beams
        self.bws = ops.BeamWorkspace(requests, beams, c.vocab, self.topk, dev)
        ints = dict(dtype=torch.int32, device=dev)
        # decode M-RoPE tables of linear positions; the graph reads them in place
        rc, rs = positions.linear_rope_tables(rows + 1, c.decoder_theta, c.head_dim)
        self.rcos, self.rsin = torch.from_numpy(rc).to(dev), torch.from_numpy(rs).to(dev)
        self.tok = torch.zeros(N, dtype=torch.int64, device=dev)
        self.slot = torch.full((N,), -1, **ints)
        self.slot_new = torch.full((N,), -1, **ints)
        self.parent = torch.full((N,), -1, **ints)
        self.rope_row = torch.zeros(N, **ints)
        self.scores = torch.zeros((requests, beams), dtype=torch.float32, device=dev)
        self.picked = (torch.empty((requests, self.topk), dtype=torch.float32, device=dev),
                       torch.empty((requests, self.topk), **ints),
                       torch.empty((requests, self.topk), **ints))
        self.first_row = (torch.arange(requests, device=dev) * beams).unsqueeze(1)
        self.rank = torch.arange(self.topk, device=dev)
        # generated tokens so far; what the last step chose; ended hypotheses, best first
        self.made = torch.zeros((), dtype=torch.int64, device=dev)
        self.step_tok = torch.zeros((requests, beams), **ints)
        self.step_beam = torch.zeros((requests, beams), **ints)
        self.done = torch.zeros(requests, dtype=torch.bool, device=dev)
        self.end_score = torch.zeros((requests, beams), dtype=torch.float32, device=dev)
        self.end_step = torch.zeros((requests, beams), dtype=torch.int64, device=dev)
        self.end_beam = torch.zeros((requests, beams), dtype=torch.int64, device=dev)
        QW, KW = c.query_heads * c.head_dim, c.kv_heads * c.head_dim
        self.qkv = torch.empty((N, QW + 2 * KW), dtype=torch.float16, device=dev)
        self.q = self.qkv[:, :QW].view(N, c.query_heads, c.head_dim)
        self.k = self.qkv[:, QW:QW + KW].view(N, c.kv_heads, c.head_dim)
        self.v = self.qkv[:, QW + KW:].view(N, c.kv_heads, c.head_dim)
        # decode leaves an idle sequence's rows as they are: zero, or the last ones of a request that
        # is done.  They go through the layers with the others; nothing reads what becomes of them.
        self.ctx = torch.zeros((N, c.query_heads, c.head_dim), dtype=torch.float16, device=dev)
        self.logits = None
        self.graph = None

    # ---------------------------------------------------------------- a step
    def _select(self):
        """Ended and live hypotheses of the picked continuations (at the prompt, all of beam 0).
        Sets tok, scores and parent."""
        B, W = self.B, self.W
        score, beam, token = self.picked
        self.made += 1
        length = self.made.to(torch.float32) ** self.penalty
        ends = token == self.eng.cfg.eos_token_id
        # ended hypotheses: the kept ones first, so that equal scores stay in order
        new = torch.where(ends & (self.rank < W) & ~self.done.unsqueeze(1), score / length,
                          -math.inf)
        both, order = torch.sort(torch.cat([self.end_score, new], 1), dim=1, descending=True,
                                 stable=True)
        order = order[:, :W]
        self.end_score.copy_(both[:, :W])
        self.end_step.copy_(torch.cat([self.end_step, self.made.expand(B, self.topk)], 1)
                            .gather(1, order))
        self.end_beam.copy_(torch.cat([self.end_beam, beam.long()], 1).gather(1, order))
        # live beams: the first W continuations that do not end
        live = torch.sort(ends.to(torch.int32), dim=1, stable=True).indices[:, :W]
        self.scores.copy_(score.gather(1, live))
        self.step_tok.copy_(token.gather(1, live))
        self.step_beam.copy_(beam.gather(1, live))
        beaten = self.scores[:, 0] / length <= self.end_score[:, -1]
        self.done |= beaten & (self.end_score[:, -1] > -math.inf)
        self.tok.copy_(self.step_tok.view(-1))
        self.parent.copy_(torch.where(self.done.unsqueeze(1), -1, self.first_row + self.step_beam)
                          .view(-1))

    def _step(self):
        eng, c = self.eng, self.eng.cfg
        h32 = eng.embed.index_select(0, self.tok).float()
        pending = None
        for l, L in enumerate(eng.dlayers):
            n1 = ops.add_norm(h32, L["n1"], c.rms_eps, delta=pending)
            torch.mm(n1, L["qkv"].t(), out=self.qkv)
            kv8.decode(self.cache, l, self.q, self.k, self.v, self.rcos, self.rsin, self.slot,
                       self.ws, rope_row=self.rope_row, out=self.ctx)
            pending = eng._layer_mlp(L, h32, F.linear(self.ctx.view(self.N, -1), L["o"]))
        fn = ops.add_norm(h32, eng.final_norm, c.rms_eps, delta=pending)
        self.logits = eng._logits(fn)
        ops.beam_topk(self.logits, self.scores, self.topk, self.bws, out=self.picked)
        self._select()
        self._move(1)
        self.rope_row += 1

    def _move(self, advance: int):
        """The surviving beams' caches, and pages for their next row."""
        kv8.fork(self.cache, self.slot, self.parent, self.ws, advance=advance, out=self.slot_new)
        self.slot.copy_(self.slot_new)
        kv8.grow(self.cache, self.slot, self.ws, ahead=1)

    def _capture(self):
        """Capture the step.  Every sequence is idle meanwhile (slot -1), so neither the warm-up
        nor the capture touches the cache."""
        self.slot.fill_(-1)
        s = torch.cuda.Stream()
        s.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(s):
            self._step()                 # cuBLAS handles and workspaces
        torch.cuda.current_stream().wait_stream(s)
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            self._step()
        self.graph = graph               # a capture that failed is not replayed

    # ----------------------------------------------------------------- a batch
    def prompts(self, lengths):
        """Pages for the prompts (slot r * beams for request r); returns their int32 slots and
        the function that stores layer l's rows from fp16 caches."""
        if self.graph is None:
            self._capture()
        dev = self.eng.device
        self.cache.reset()
        B, most = self.B, max(lengths)
        slots = (self.first_row.view(-1)).to(torch.int32)
        count = torch.tensor(lengths, dtype=torch.int32).to(dev, non_blocking=True)
        kv8.grow(self.cache, slots, self.ws, ahead=count)

        def store(l, k, v):              # [B, rows, kv_heads, 128], prompt b at [b, :lengths[b]]
            rows = k.shape[1]
            begin = torch.arange(B, dtype=torch.int32, device=dev) * rows
            kv8.store(self.cache, l, k.view(-1, *k.shape[2:]), v.view(-1, *v.shape[2:]), begin,
                      count, slots, most, self.ws)

        def stored():
            kv8.grow(self.cache, slots, self.ws, advance=count)
            self.slot.fill_(-1)
            self.slot[:: self.W] = slots
        return store, stored

    def start(self, logits, lengths, deltas):
        """The first tokens, from the prompts' logits [B, vocab]."""
        B, W = self.B, self.W
        pos = np.asarray(lengths, dtype=np.int64) + np.asarray(deltas, dtype=np.int64)
        if pos.min() < 0:
            raise positions.PositionError("decode position is negative")
        if pos.max() > max(lengths):
            raise ValueError("decode positions do not fit the tables")
        self.rope_row.copy_(torch.from_numpy(np.repeat(pos, W).astype(np.int32)))
        self.made.zero_()
        self.done.zero_()
        self.end_score.fill_(-math.inf)
        # more continuations than the vocabulary has do not exist: they stay -infinity
        k = min(self.topk, logits.shape[1])
        zero = torch.zeros((B, 1), dtype=torch.float32, device=logits.device)
        got = ops.beam_topk(logits, zero, k)
        self.picked[0].fill_(-math.inf)
        for to, x in zip(self.picked, got):
            to[:, :k].copy_(x)
        for to in self.picked[1:]:
            to[:, k:].zero_()
        self._select()
        self._move(0)

    def run(self, steps: int, record: bool):
        """Queue `steps` steps; returns what they chose: tokens, beams [steps, B, W], and with
        record their logits [steps, N, vocab] and scores [steps, B, W] (device).  Does not
        wait."""
        tok = torch.empty((steps,) + self.step_tok.shape, dtype=torch.int32, device=self.tok.device)
        beam = torch.empty_like(tok)
        logits, scores = [], []
        for i in range(steps):
            self.graph.replay()
            tok[i].copy_(self.step_tok)
            beam[i].copy_(self.step_beam)
            if record:
                logits.append(self.logits.clone())
                scores.append(self.scores.clone())
        return tok, beam, (torch.stack(logits), torch.stack(scores)) if record else None


def hypotheses(tok, beam, end_score, end_step, end_beam, done, scores, penalty):
    """One request's hypotheses, best first: (score, token list, reason).  tok, beam [S, W]:
    what each step chose; end_*: the ended ones (made at token number end_step from beam
    end_beam of the step before); scores [W]: the live beams' at the end."""
    def path(step, w):
        out = []
        while step >= 0:
            out.append(int(tok[step, w]))
            w = int(beam[step, w])
            step -= 1
        return out[::-1]

    found = []
    for s, n, w in zip(end_score, end_step, end_beam):
        if s > -math.inf:
            found.append((float(s), path(int(n) - 2, int(w)), int(n), greedy.EOS_TOKEN))
    if not done:
        n = len(tok)
        for w, s in enumerate(scores):
            if s > -math.inf:
                found.append((float(np.float32(s) / np.float32(n) ** np.float32(penalty)),
                              path(n - 1, w), n, greedy.MAX_NEW_TOKENS))
    found.sort(key=lambda h: -h[0])          # stable: ended ones first among equals
    return [(s, p, why) for s, p, _, why in found[:len(scores)]]


def run_chunks(left, chunk, status, queue):
    """Queue up to `left` steps, a chunk at a time, until all requests are done.  status: (done
    flags on the host, the event after which they are there) as the prompts left them;
    queue(steps) queues steps and returns the status behind them.  One chunk is queued ahead of
    the status that is being looked at."""
    ahead = None
    while True:
        if left > 0:
            ahead = queue(min(chunk, left))
            left -= chunk
        done, event = status
        event.synchronize()
        if ahead is None or bool(done.all()):
            return
        status, ahead = ahead, None


def _decoder(eng, requests, beams, rows, pages, cache_dtype, length_penalty) -> BeamDecoder:
    """The engine's decoder of the last batch when it is for as many requests and beams and has
    room for these rows and pages (what it computes does not depend on how much it has), else
    a new one, with room for that batch too where only room is missing."""
    key = (requests, beams, cache_dtype, float(length_penalty))
    if eng._beam is not None and eng._beam[0] == key:
        dec = eng._beam[1]
        if rows <= dec.rows and pages <= dec.cache.pages:
            return dec
        rows, pages = max(rows, dec.rows), max(pages, dec.cache.pages)
        del dec
    eng._beam = None
    torch.cuda.empty_cache()
    eng._beam = (key, BeamDecoder(eng, requests, beams, rows, pages, cache_dtype, length_penalty))
    return eng._beam[1]


def generate(eng, images_patches, grids, max_new_tokens, beams, length_penalty, cache_dtype,
             chunk, timings, prepare, record):
    """OcrEngine.generate_beam."""
    from .model import _download
    c, B = eng.cfg, len(grids)
    if not 1 <= beams <= 32:
        raise ValueError("beams must be 1 to 32")
    if max_new_tokens < 1 or chunk < 1:
        raise ValueError("max_new_tokens and chunk must be positive")
    if cache_dtype not in kv8.CODE_TYPES:
        raise TypeError("cache_dtype must be float8_e4m3fn or int8")
    ev = None
    if timings is not None:
        ev = [torch.cuda.Event(enable_timing=True) for _ in range(4)]
        ev[0].record()
    plan = eng._plan_prompts(grids)
    T = max(plan.lengths)
    img = eng.encode_images(images_patches, grids, prepare)
    if ev:
        ev[1].record()
    # pages: every prompt's full ones once, and for each beam those that its new rows can fill
    pages = sum(n // kv8.PAGE for n in plan.lengths) + B * beams * (max_new_tokens // kv8.PAGE + 1)
    dec = _decoder(eng, B, beams, T + max_new_tokens, pages, cache_dtype, length_penalty)
    # one layer's fp16 rows at a time: the prefill writes them, the store reads them
    kc = torch.empty((B, T, c.kv_heads, c.head_dim), dtype=torch.float16, device=eng.device)
    vc = torch.empty_like(kc)
    store, stored = dec.prompts(plan.lengths)
    fn = eng._prefill(plan, img, lambda l: (kc, vc), lambda l: store(l, kc, vc))
    stored()
    logits0 = eng._logits(fn.index_select(0, plan.last))
    dec.start(logits0, plan.lengths, plan.deltas)
    if ev:
        ev[2].record()
    parts = [(_download(dec.step_tok.unsqueeze(0)), _download(dec.step_beam.unsqueeze(0)), None)]
    first_scores = dec.scores.clone() if record else None

    def queue(steps):
        tok, beam, rec = dec.run(steps, record)
        parts.append((_download(tok), _download(beam), rec))
        return _download(dec.done)
    run_chunks(max_new_tokens - 1, chunk, _download(dec.done), queue)
    ends = [_download(t) for t in (dec.end_score, dec.end_step, dec.end_beam, dec.done, dec.scores)]
    if ev:
        ev[3].record()
    for _, event in ends:
        event.synchronize()
    flags = dec.ws.errors()
    if flags:
        raise abi.PvlcError(abi.DEVICE_FAULT_FLAG, f"kv8 fault flags {flags:#x}")
    flags = ops.fault_flags()
    if flags:
        raise abi.PvlcError(abi.DEVICE_FAULT_FLAG, f"vision / prefill fault flags {flags:#x}")
    tok = np.concatenate([p[0][0].numpy() for p in parts])
    beam = np.concatenate([p[1][0].numpy() for p in parts])
    es, en, eb, done, live = (h.numpy() for h, _ in ends)
    found = [hypotheses(tok[:, r], beam[:, r], es[r], en[r], eb[r], bool(done[r]), live[r],
                        length_penalty) for r in range(B)]
    if not all(found):                      # every logit of some request NaN or -infinity
        raise greedy.GreedyError(greedy.NON_FINITE_INPUT, "no hypothesis has a finite score")
    found = [[(s, p + [c.eos_token_id] if why == greedy.EOS_TOKEN else p, why)
              for s, p, why in f] for f in found]
    if ev:
        ev[3].synchronize()
        timings.update(encode_ms=ev[0].elapsed_time(ev[1]), prefill_ms=ev[1].elapsed_time(ev[2]),
                       decode_ms=ev[2].elapsed_time(ev[3]), decode_steps=len(tok) - 1)
    out = dict(tokens=[f[0][1] for f in found], stop=[f[0][2] for f in found], hypotheses=found)
    if record:
        rec = [p[2] for p in parts[1:]]
        out["steps"] = dict(
            tokens=tok, beams=beam, first_logits=logits0.cpu(),
            logits=torch.cat([x for x, _ in rec]).cpu() if rec else None,
            scores=torch.cat([first_scores.unsqueeze(0)] + [x for _, x in rec]).cpu())
    return out
