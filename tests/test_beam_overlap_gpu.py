"""Outputs of a beam selection in the gaps between pitched logits are taken; on them refused."""
import pytest
import torch

pytestmark = pytest.mark.gpu


def test_outputs_beside_the_logits(cuda_lib):
    from pvlc_b200 import abi, ops
    g = torch.Generator(device="cuda").manual_seed(1)
    x = torch.randn((6, 160), generator=g, device="cuda")
    scores = torch.randn((3, 2), generator=g, device="cuda")
    logits = x[:, :100]
    want = ops.beam_topk(logits, scores, 5, ops.BeamWorkspace(3, 2, 100, 5))

    def place(row, col, dtype):
        return x.view(-1)[row * 160 + col:row * 160 + col + 15].view(dtype).view(3, 5)
    outs = lambda *at: tuple(place(r, c, d) for (r, c), d in  # noqa: E731
                             zip(at, (torch.float32, torch.int32, torch.int32)))
    for at in ([(0, 100), (1, 110), (5, 145)], [(2, 100), (2, 115), (2, 130)], [(4, 145), (0, 101), (3, 120)]):
        got = outs(*at)
        ops.beam_topk(logits, scores, 5, out=got)
        for a, b in zip(got, want):
            assert torch.equal(a, b)
    for at in ([(0, 99), (1, 110), (5, 145)], [(2, 100), (2, 114), (2, 130)], [(4, 146), (0, 101), (3, 120)],
               [(0, 110), (1, 110), (1, 96)]):
        with pytest.raises(abi.PvlcError):
            ops.beam_topk(logits, scores, 5, out=outs(*at))
