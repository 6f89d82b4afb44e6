"""Beam selection (pvlc_lm_head_beam_topk) against a plain 64-bit sort of all candidates.

Order: larger score, then lower beam, larger logit, lower token; NaN counts as -infinity.  The
kernel's log-sum-exp differs from the 64-bit one by less than 1e-6 (f32 exponentials, each
within 2^-22, of chunk maxima; f64 sums of chunks), so scores have to be within 1e-6 + 2^-24
of their size, and the order has to be equal wherever two candidates of different beams are
further apart than 2e-6; the inputs below are checked to be."""
import numpy as np
import pytest
import torch

pytestmark = pytest.mark.gpu


def plain(logits, scores, K):
    """[B * W, V], [B, W] -> (score, beam, token) [B, K] and the smallest gap between the
    neighbouring picked candidates of different beams."""
    B, W = scores.shape
    x = logits.astype(np.float64)
    x[np.isnan(x)] = -np.inf
    V = x.shape[1]
    out = [np.zeros((B, K)), np.zeros((B, K), int), np.zeros((B, K), int)]
    gap = np.inf
    for r in range(B):
        y = x[r * W:(r + 1) * W]
        with np.errstate(all="ignore"):
            top = y.max(1, keepdims=True)
            lse = top + np.log(np.exp(y - top).sum(1, keepdims=True))
            c = scores[r].astype(np.float64)[:, None] - lse + y
        c[np.isnan(c)] = -np.inf
        beam, token = np.divmod(np.arange(W * V), V)
        order = np.lexsort((token, -y.ravel() + 0.0, beam, -c.ravel()))
        picked = order[:K + 1]
        s = c.ravel()[picked]
        b = beam[picked]
        with np.errstate(all="ignore"):
            d = np.abs(np.diff(s))[(np.diff(b) != 0)]
        d = d[np.isfinite(d)]
        gap = min(gap, d.min() if d.size else np.inf)
        out[0][r], out[1][r], out[2][r] = s[:K], b[:K], token[order[:K]]
    return out, gap


def check(logits, scores, K, dtype=torch.float32, gap=2e-6, view=None):
    from pvlc_b200 import ops
    t = torch.from_numpy(logits).to(dtype).cuda()
    if view is not None:
        t = view(t)
    got = ops.beam_topk(t, torch.from_numpy(scores).cuda(), K)
    want, d = plain(t.float().cpu().numpy(), scores, K)
    assert d > gap or gap is None
    np.testing.assert_array_equal(got[1].cpu().numpy(), want[1])
    np.testing.assert_array_equal(got[2].cpu().numpy(), want[2])
    a, b = got[0].cpu().numpy().astype(np.float64), want[0]
    fin = np.isfinite(b)
    np.testing.assert_array_equal(np.isfinite(a), fin)
    np.testing.assert_array_equal(a[~fin], b[~fin])
    assert (np.abs(a - b)[fin] <= 1e-6 + 2.0 ** -24 * np.abs(b[fin])).all()


@pytest.mark.parametrize("dtype", [torch.float32, torch.float16])
@pytest.mark.parametrize("B,W,V,K", [(1, 1, 1, 1), (1, 1, 5, 5), (2, 3, 4, 9), (1, 4, 1000, 8),
                                     (3, 2, 8191, 4), (2, 1, 8193, 16), (2, 5, 16385, 10),
                                     (1, 32, 700, 64), (5, 4, 103424, 8), (1, 1, 103424, 1)])
def test_random(cuda_lib, B, W, V, K, dtype):
    rng = np.random.default_rng(B * 1000 + V + K)
    check((rng.standard_normal((B * W, V)) * 3).astype(np.float32),
          (-5 * rng.random((B, W))).astype(np.float32), K, dtype, gap=0.0 if V < 6 else 2e-6)


@pytest.mark.parametrize("K", [1, 8, 33, 64])
def test_ties_within_a_row(cuda_lib, K):
    """Few distinct logits: hundreds of equal ones, which go to the lower token."""
    rng = np.random.default_rng(K)
    x = rng.integers(-2, 3, (6, 20000)).astype(np.float32)
    x[:, ::7] = -0.0
    check(x, np.array([[-1.0, -2.25], [-3.5, -1.0], [0.0, -9.0]], np.float32), K)


def test_equal_rows_tie_across_beams(cuda_lib):
    """Beams with the same row and score: the lower beam first."""
    rng = np.random.default_rng(1)
    x = np.repeat(rng.standard_normal((1, 9000)).astype(np.float32), 4, 0)
    check(x, np.full((1, 4), -2.0, np.float32), 16, gap=-1)


def test_all_equal(cuda_lib):
    check(np.zeros((4, 30000), np.float32), np.array([[-1.0, -1.0, -3.0, -0.5]], np.float32), 64,
          gap=-1)


def test_masked_rows_and_beams(cuda_lib):
    """Suppressed tokens, rows with fewer than K tokens left or none, dead beams, NaN, +inf."""
    rng = np.random.default_rng(2)
    x = rng.standard_normal((12, 17000)).astype(np.float32)
    x[:, ::3] = -np.inf
    x[1] = -np.inf
    x[2, 5:] = -np.inf
    x[3] = -np.inf
    x[3, 16999] = 2.0
    x[5, ::2] = np.nan
    x[6, 77] = np.inf
    x[8:12] = -np.inf
    s = np.array([[0.0, -1.0, -2.0, -3.0], [0.0, -1.0, -np.inf, -np.inf],
                  [-1.0, -2.0, -np.inf, -4.0]], np.float32)
    check(x, s, 16)


def test_first_step_of_a_search(cuda_lib):
    """One live beam: every candidate is its own."""
    rng = np.random.default_rng(3)
    x = rng.standard_normal((4, 5000)).astype(np.float32)
    check(x, np.array([[0.0] + [-np.inf] * 3], np.float32), 8)


@pytest.mark.parametrize("dtype", [torch.float32, torch.float16])
def test_pitched_and_odd_rows(cuda_lib, dtype):
    rng = np.random.default_rng(4)
    x = rng.standard_normal((6, 9011)).astype(np.float32)
    s = (-rng.random((2, 3))).astype(np.float32)
    check(x, s, 8, dtype, view=lambda t: t[:, 3:9004])
    check(x, s, 8, dtype, view=lambda t: t[:, 1:9002])


def test_large_and_small_values(cuda_lib):
    rng = np.random.default_rng(5)
    x = rng.standard_normal((4, 9000)).astype(np.float32)
    x[0] *= 1e4
    x[1] *= 1e-6
    x[2] += 8e4
    x[3] = -3e38
    x[3, 8] = 3e38
    # the f32 logits of rows 0 and 2 are exact in f64, their log-sum is the largest logit's
    # size times 2^-52: the same bounds hold
    check(x, np.array([[-1.0, -2.0], [-0.5, -7.0]], np.float32), 12)


def test_captured_and_reused_workspace(cuda_lib):
    from pvlc_b200 import ops
    rng = np.random.default_rng(6)
    xs = [torch.from_numpy(rng.standard_normal((8, 20000)).astype(np.float32)).cuda()
          for _ in range(3)]
    s = torch.from_numpy((-rng.random((2, 4))).astype(np.float32)).cuda()
    ws = ops.BeamWorkspace(2, 4, 20000, 8)
    want = [ops.beam_topk(x, s, 8) for x in xs]
    x = xs[0].clone()
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=side):
        got = ops.beam_topk(x, s, 8, ws)
    for i in (2, 0, 1):
        x.copy_(xs[i])
        graph.replay()
        for a, b in zip(got, want[i]):
            assert torch.equal(a, b)


def test_workspace_serves_smaller_calls(cuda_lib):
    from pvlc_b200 import ops
    rng = np.random.default_rng(7)
    ws = ops.BeamWorkspace(25, 1, 103424, 8)
    for B, W, V in ((25, 1, 103424), (22, 1, 103424), (3, 4, 60000), (1, 1, 40), (5, 5, 8192)):
        x = rng.standard_normal((B * W, V)).astype(np.float32)
        s = (-rng.random((B, W))).astype(np.float32)
        got = ops.beam_topk(torch.from_numpy(x).cuda(), torch.from_numpy(s).cuda(), 8, ws)
        want, gap = plain(x, s, 8)
        assert gap > 2e-6
        np.testing.assert_array_equal(got[2].cpu().numpy(), want[2])


def test_many_reach_the_bound(cuda_lib):
    """Chunks where more elements reach the selection's bound than are ranked at once, next
    to ordinary ones, and more chunks than a join bounds by."""
    rng = np.random.default_rng(8)
    x = rng.standard_normal((8, 60000)).astype(np.float32)
    x[:, 9000:11000] = 6.5
    x[3, 30000:30700] = 7.0
    check(x, (-rng.random((2, 4))).astype(np.float32), 24)
    big = rng.standard_normal((2, 4_300_000)).astype(np.float32)
    check(big, np.array([[-0.5, -0.25]], np.float32), 5)


def test_wrapper_refusals(cuda_lib):
    from pvlc_b200 import abi, ops
    x, s = torch.zeros((8, 100), device="cuda"), torch.zeros((2, 4), device="cuda")
    with pytest.raises(TypeError):
        ops.beam_topk(x.double(), s, 4)
    with pytest.raises(TypeError):
        ops.beam_topk(x, s.cpu(), 4)
    with pytest.raises(ValueError):
        ops.beam_topk(x[:7], s, 4)
    with pytest.raises(ValueError):
        ops.beam_topk(x.t().contiguous().t(), s, 4)
    with pytest.raises(abi.PvlcError):
        ops.beam_topk(x, s, 65)
    with pytest.raises(abi.PvlcError):
        ops.beam_topk(x, s, 8, ops.BeamWorkspace(1, 1, 100, 1))
    with pytest.raises(ValueError):
        ops.beam_topk(x, s, 4, out=(s, s.int(), s.int()[:1]))


@pytest.mark.parametrize("B,W,V,K", [(1, 1, 40, 16), (2, 4, 150, 16), (2, 2, 4097, 24), (1, 3, 8193, 64),
                                     (40, 4, 9000, 12)])
@pytest.mark.parametrize("left", [0, 1, 5, 12, 30])
def test_few_tokens_allowed(cuda_lib, B, W, V, K, left):
    """A mask that leaves `left` tokens of a row, first and last ones among them, and other rows
    with a NaN for each masked one: fewer than K continuations are finite, or just as many."""
    rng = np.random.default_rng(left * 7 + V)
    x = np.full((B * W, V), -np.inf, np.float32)
    for r in range(B * W):
        at = rng.choice(V, left, replace=False)
        if left > 1:
            at[:2] = 0, V - 1
        if r % 3 == 1:
            x[r] = np.nan
        x[r, at] = rng.standard_normal(left) * 3
    check(x, (-5 * rng.random((B, W))).astype(np.float32), K)


@pytest.mark.parametrize("B,W,V,K", [(3, 1, 5000, 64), (2, 2, 300, 33), (1, 8, 70, 48), (7, 5, 2000, 17)])
def test_more_wanted_than_there_are_chunks(cuda_lib, B, W, V, K):
    rng = np.random.default_rng(K)
    check((rng.standard_normal((B * W, V)) * 3).astype(np.float32),
          (-2 * rng.random((B, W))).astype(np.float32), K)
