"""Beam search through the engine (OcrEngine.generate_beam): the run of the 8-bit cache's
operators together.

The search's choices are held to a plain replay in 64 bits on the logits that the run recorded;
the logits are held to a single sequence decoded without beams, forks or a batch, on a cache of
its own, along every returned hypothesis: same arithmetic, other summation orders, so within
the engine's parity rule for logits (1e-2 of the largest).  A wrong parent, page or open block
would make them other sequences' logits."""
import dataclasses
import math

import numpy as np
import pytest
import torch
import torch.nn.functional as F

from pvlc_b200 import greedy
from pvlc_b200 import model as M

pytestmark = pytest.mark.gpu

CFG = M.ModelConfig(vision_layers=1, decoder_layers=3)
GRIDS = [(1, 4, 6), (1, 8, 8), (1, 6, 4)]           # prompts of 19, 29 and 19 rows


@pytest.fixture(scope="module")
def setup(cuda_lib):
    w = M.init_weights(CFG, seed=3, device="cuda")
    # sharper logits than random weights give, so that beams live and die
    w.decoder[-1].mul_(4.0)
    g = torch.Generator(device="cuda")
    g.manual_seed(5)
    patches = [torch.randn((t * h * x, CFG.patch_input), generator=g, device="cuda")
               for t, h, x in GRIDS]
    return w, patches


def replay(first, logits, scores, W, eos, penalty, steps):
    """The search on recorded logits: first [V], logits[s] [W, V] of what were then the live
    beams, whose f32 scores after step s are scores[s] [W]; each is checked before the next
    step starts from it, so no error adds up.  Returns the choices of every step and the
    hypotheses.

    A step's candidates are f64 sums whose log-sums are within 1e-6: two that are 2e-6 apart
    are in order.  Scores over lengths are f32 quotients (and powers, 2^-22): 2^-20 of their
    size apart is in order."""
    def logp(x):
        x = x.astype(np.float64)
        m = x.max(-1, keepdims=True)
        return x - m - np.log(np.exp(x - m).sum(-1, keepdims=True))

    def apart(a, b):
        assert abs(a - b) > 2.0 ** -20 * abs(b), "the inputs leave the order open"
    live, hist, ended = np.array([0.0]), [], []
    done = False
    for s in range(steps):
        lp = logp(first[None] if s == 0 else logits[s - 1]) + live[:, None]
        flat = lp.ravel()
        order = np.argsort(-flat, kind="stable")[:2 * W + 1]
        assert np.abs(np.diff(flat[order])).min() > 2e-6, "the inputs leave the order open"
        order = order[:2 * W]
        beam, token = np.divmod(order, lp.shape[1])
        n = s + 1
        for rank, (b, t, i) in enumerate(zip(beam, token, order)):
            if t == eos and rank < W:
                ended.append((flat[i] / n ** penalty, s, int(b)))
        ended.sort(key=lambda e: -e[0])
        for a, b in zip(ended, ended[1:]):
            apart(a[0], b[0])
        ended = ended[:W]
        go = [(b, t, flat[i]) for b, t, i in zip(beam, token, order) if t != eos][:W]
        hist.append(([int(t) for _, t, _ in go], [int(b) for b, _, _ in go]))
        live = scores[s].astype(np.float64)
        np.testing.assert_allclose(live, [x for _, _, x in go], rtol=2.0 ** -24, atol=1e-6)
        if len(ended) == W:
            apart(live[0] / n ** penalty, ended[-1][0])
            if live[0] / n ** penalty <= ended[-1][0]:
                done = True
                break

    def path(s, w):
        out = []
        while s >= 0:
            out.append(hist[s][0][w])
            w = hist[s][1][w]
            s -= 1
        return out[::-1]
    hyps = [(sc, path(s - 1, b) + [eos], greedy.EOS_TOKEN) for sc, s, b in ended]
    if not done:
        n = len(hist)
        hyps += [(x / n ** penalty, path(n - 1, w), greedy.MAX_NEW_TOKENS)
                 for w, x in enumerate(live)]
        hyps.sort(key=lambda h: -h[0])
        for a, b in zip(hyps, hyps[1:]):
            apart(a[0], b[0])
        hyps = hyps[:W]
    return hist, hyps


def run(setup, W, steps, eos=2, penalty=1.0, dtype=torch.float8_e4m3fn, chunk=5):
    w, patches = setup
    eng = M.OcrEngine(dataclasses.replace(CFG, eos_token_id=eos), w)
    res = eng.generate_beam(patches, GRIDS, steps, beams=W, length_penalty=penalty,
                            cache_dtype=dtype, chunk=chunk, record=True)
    return eng, res


def check_replay(res, W, eos, penalty, steps):
    rec = res["steps"]
    for r in range(len(GRIDS)):
        lg = rec["logits"].numpy()[:, r * W:(r + 1) * W] if rec["logits"] is not None else None
        hist, hyps = replay(rec["first_logits"].numpy()[r], lg, rec["scores"].numpy()[:, r], W,
                            eos, penalty, steps)
        for s, (tok, beam) in enumerate(hist):
            assert rec["tokens"][s, r].tolist() == tok, (r, s)
            assert rec["beams"][s, r].tolist() == beam, (r, s)
        got = res["hypotheses"][r]
        assert [(t, why) for _, t, why in got] == [(t, why) for _, t, why in hyps], r
        np.testing.assert_allclose([s for s, _, _ in got], [s for s, _, _ in hyps],
                                   rtol=2.0 ** -21, atol=1e-6)
        assert res["tokens"][r] == got[0][1] and res["stop"][r] == got[0][2]


@pytest.mark.parametrize("W,steps,dtype", [(4, 40, torch.float8_e4m3fn), (3, 13, torch.int8),
                                           (1, 6, torch.int8), (8, 3, torch.float8_e4m3fn),
                                           (2, 1, torch.float8_e4m3fn)])
def test_choices_follow_the_recorded_logits(setup, W, steps, dtype):
    eng, res = run(setup, W, steps, dtype=dtype)
    check_replay(res, W, 2, 1.0, steps)
    # every page's count is the number of table entries that name it
    c = eng._beam[1].cache
    t = c.table[c.table >= 0].long()
    assert torch.equal(torch.bincount(t, minlength=c.pages), c.refs.long())


@pytest.mark.parametrize("penalty", [0.0, 1.0, 2.0])
def test_hypotheses_that_end(setup, penalty):
    """A token that the search picks becomes the end token: hypotheses end, requests are done
    early, their sequences leave the cache."""
    W, steps = 3, 24
    _, free = run(setup, W, steps)
    tok = free["steps"]["tokens"]
    ids, count = np.unique(tok[2:12], return_counts=True)
    for eos in ids[np.argsort(-count)][:2]:
        eng, res = run(setup, W, steps, eos=int(eos), penalty=penalty)
        check_replay(res, W, int(eos), penalty, steps)
        dec = eng._beam[1]
        # some ended (at a penalty of 2, score / length^2, longer ones may still outrank them)
        assert (dec.end_score > -math.inf).any()
        if penalty < 2:
            assert any(why == greedy.EOS_TOKEN for h in res["hypotheses"] for _, _, why in h)
        done = dec.done.cpu().numpy()
        slot = dec.slot.view(len(GRIDS), W).cpu().numpy()
        assert ((slot == -1).all(1) == done).all()
        t = dec.cache.table[dec.cache.table >= 0].long()
        assert torch.equal(torch.bincount(t, minlength=dec.cache.pages), dec.cache.refs.long())


def alone(eng, prompt_kv, length, delta, tokens, dtype):
    """Logits after each of `tokens`, one sequence on a cache of its own, step by step."""
    from pvlc_b200 import kv8, ops, positions
    c = eng.cfg
    n = length + len(tokens)
    cache = kv8.Cache.empty(c.decoder_layers, n // 32 + 1, 1, n // 32 + 1, c.kv_heads, dtype)
    ws = kv8.Workspace(cache, 1, c.query_heads)
    slot = torch.zeros(1, dtype=torch.int32, device="cuda")
    kv8.grow(cache, slot, ws, ahead=length)
    zero, count = slot.clone(), slot + length
    for l, (k, v) in enumerate(prompt_kv):
        kv8.store(cache, l, k, v, zero, count, slot, length, ws)
    kv8.grow(cache, slot, ws, advance=length, ahead=1)
    rc, rs = (torch.from_numpy(x).cuda() for x in
              positions.linear_rope_tables(n + 1, c.decoder_theta, c.head_dim))
    out = []
    QH, KH = c.query_heads, c.kv_heads
    for i, t in enumerate(tokens):
        h32 = eng.embed[t:t + 1].float()
        pending = None
        row = torch.tensor([length + delta + i], dtype=torch.int32, device="cuda")
        for l, L in enumerate(eng.dlayers):
            n1 = ops.add_norm(h32, L["n1"], c.rms_eps, delta=pending)
            qkv = F.linear(n1, L["qkv"]).view(1, QH + 2 * KH, 128)
            ctx = kv8.decode(cache, l, qkv[:, :QH], qkv[:, QH:QH + KH], qkv[:, QH + KH:], rc, rs,
                             slot, ws, rope_row=row)
            pending = eng._layer_mlp(L, h32, F.linear(ctx.view(1, -1), L["o"]))
        fn = ops.add_norm(h32, eng.final_norm, c.rms_eps, delta=pending)
        out.append(eng._logits(fn)[0].cpu().numpy())
        kv8.grow(cache, slot, ws, advance=1, ahead=1)
    assert ws.errors() == 0
    return out


@pytest.mark.parametrize("dtype", [torch.float8_e4m3fn, torch.int8])
def test_every_hypothesis_has_its_own_history(setup, dtype):
    W, steps = 4, 40                       # past a page's end for every prompt
    eng, res = run(setup, W, steps, dtype=dtype)
    w, patches = setup
    plan = eng._plan_prompts(GRIDS)
    T = max(plan.lengths)
    kept = []
    shape = (len(GRIDS), T, CFG.kv_heads, CFG.head_dim)
    caches = [(torch.zeros(shape, dtype=torch.float16, device="cuda"),
               torch.zeros(shape, dtype=torch.float16, device="cuda"))
              for _ in range(CFG.decoder_layers)]
    eng._prefill(plan, eng.encode_images(patches, GRIDS), lambda l: caches[l], kept.append)
    assert kept == list(range(CFG.decoder_layers))
    rec = res["steps"]
    for r in range(len(GRIDS)):
        kv = [(k[r], v[r]) for k, v in caches]
        for w_end in (0, W - 1):
            # the path of a live beam: its token and number at every step
            path, b = [], w_end
            for s in range(steps - 1, -1, -1):
                path.append((int(rec["tokens"][s, r, b]), b))
                b = int(rec["beams"][s, r, b])
            path.reverse()
            got = alone(eng, kv, plan.lengths[r], plan.deltas[r], [t for t, _ in path[:-1]], dtype)
            for s, x in enumerate(got):
                want = rec["logits"][s, r * W + path[s][1]].numpy()
                assert np.abs(want - x).max() <= 1e-2 * np.abs(x).max(), (r, w_end, s)


def test_recognize_with_beams(setup):
    """Host pages in, hypotheses out; the greedy call beside it is what it was."""
    from pvlc_b200 import preprocess as P
    w, _ = setup
    eng = M.OcrEngine(CFG, w)
    rng = np.random.default_rng(1)
    pages = [rng.integers(0, 256, (56, 84, 3), dtype=np.uint8) for _ in range(2)]
    cfg = P.VisionPreprocessConfig(min_pixels=56 * 84, max_pixels=56 * 84)
    before = eng.recognize(pages, 6, preprocess_config=cfg)
    timings = {}
    got = eng.recognize(pages, 6, preprocess_config=cfg, beams=3, timings=timings)
    assert timings["decode_ms"] > 0 and timings["decode_steps"] == 5
    for h in got["hypotheses"]:
        assert len(h) == 3 and h[0][0] >= h[1][0] >= h[2][0]
        assert all(1 <= len(t) <= 6 for _, t, _ in h)
    again = eng.recognize(pages, 6, preprocess_config=cfg)
    assert again["tokens"] == before["tokens"]
    second = eng.recognize(pages, 6, preprocess_config=cfg, beams=3)
    assert second["tokens"] == got["tokens"] and second["hypotheses"] == got["hypotheses"]


def test_refusals(setup):
    w, patches = setup
    eng = M.OcrEngine(CFG, w)
    for kw in (dict(beams=0), dict(beams=33), dict(chunk=0)):
        with pytest.raises(ValueError):
            eng.generate_beam(patches, GRIDS, 4, **kw)
    with pytest.raises(ValueError):
        eng.generate_beam(patches, GRIDS, 0)
    with pytest.raises(TypeError):
        eng.generate_beam(patches, GRIDS, 4, cache_dtype=torch.float16)


def test_non_finite_logits_are_an_error(setup):
    """As in the greedy search; the engine is of use again afterwards."""
    w, patches = setup
    eng = M.OcrEngine(CFG, w)
    good = eng.generate_beam(patches, GRIDS, 4, beams=2)
    head, eng.lm_head = eng.lm_head, torch.full_like(eng.lm_head, math.nan)
    eng._beam = None                     # the captured step reads the head that it was captured with
    with pytest.raises(greedy.GreedyError):
        eng.generate_beam(patches, GRIDS, 4, beams=2)
    eng.lm_head, eng._beam = head, None
    assert eng.generate_beam(patches, GRIDS, 4, beams=2) == good
