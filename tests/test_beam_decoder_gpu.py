"""The decoder that an engine keeps between beam searches."""
import pytest
import torch

from pvlc_b200 import model as M

pytestmark = pytest.mark.gpu
CFG = M.ModelConfig(vision_layers=1, decoder_layers=3)
LONG = [(1, 12, 12), (1, 10, 12)]            # the longer prompt is the same in the first two
MIXED = [(1, 12, 12), (1, 4, 6)]
SHORT = [(1, 6, 4), (1, 8, 8)]


@pytest.fixture(scope="module")
def weights(cuda_lib):
    return M.init_weights(CFG, seed=3, device="cuda")


def patches(grids):
    g = torch.Generator(device="cuda").manual_seed(7)
    return [torch.randn((h * w, CFG.patch_input), generator=g, device="cuda") for _, h, w in grids]


def search(eng, grids, steps, **kw):
    return eng.generate_beam(patches(grids), grids, steps, beams=3, **kw)


def test_a_batch_that_fits_keeps_the_decoder(weights):
    """And finds what a decoder of its own finds, bit for bit."""
    eng = M.OcrEngine(CFG, weights)
    first = search(eng, LONG, 40)
    dec = eng._beam[1]
    for grids, steps in ((MIXED, 40), (SHORT, 40), (SHORT, 7), (LONG, 40)):
        got = search(eng, grids, steps)
        assert eng._beam[1] is dec, (grids, steps)
        assert got == search(M.OcrEngine(CFG, weights), grids, steps)
    assert got == first


def test_a_batch_that_does_not_fit_gets_another(weights):
    eng = M.OcrEngine(CFG, weights)
    search(eng, SHORT, 7)
    small = eng._beam[1]
    got = search(eng, LONG, 7)
    dec = eng._beam[1]
    assert dec is not small and got == search(M.OcrEngine(CFG, weights), LONG, 7)
    pages = dec.cache.pages
    search(eng, SHORT, 7)
    assert eng._beam[1] is dec
    # more pages, fewer rows: room for both
    search(eng, SHORT, 64)
    assert eng._beam[1].cache.pages > pages and eng._beam[1].rows >= dec.rows
    # another penalty, code type or number of requests is another decoder
    for kw in (dict(length_penalty=2.0), dict(cache_dtype=torch.int8)):
        old = eng._beam[1]
        search(eng, SHORT, 7, **kw)
        assert eng._beam[1] is not old
    old = eng._beam[1]
    search(eng, SHORT + SHORT[:1], 7)
    assert eng._beam[1] is not old


def test_a_capture_that_failed_is_not_replayed(weights, monkeypatch):
    """The call raises (out of memory, say); the next one captures the step again."""
    from pvlc_b200 import beam
    eng, real, calls = M.OcrEngine(CFG, weights), beam.ops.beam_topk, []

    def second_fails(*args, **kw):
        calls.append(1)
        if len(calls) == 2:                  # the warm-up's, then the capture's
            raise RuntimeError("not this time")
        return real(*args, **kw)
    monkeypatch.setattr(beam.ops, "beam_topk", second_fails)
    with pytest.raises(RuntimeError, match="not this time"):
        search(eng, SHORT, 9)
    monkeypatch.undo()
    assert search(eng, SHORT, 9) == search(M.OcrEngine(CFG, weights), SHORT, 9)
