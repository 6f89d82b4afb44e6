"""What a reported fault leaves behind.  The faults are words written from the host: nothing here
hangs or faults."""
import pytest
import torch

import kv8_ref as R

pytestmark = pytest.mark.gpu
TICKETS = slice(64, 64 + 2048 * 16)           # of a workspace's 32-bit words


@pytest.fixture(scope="module")
def kv8(cuda_lib):
    from pvlc_b200 import kv8
    return kv8


def time_out(ws, tickets=1):
    """As after a wait that ran out: the flag, and tickets of split units."""
    words = ws.buffer.view(torch.int32)
    words[0] = 8
    words[TICKETS] = tickets


def test_a_reported_timeout_leaves_no_tickets(kv8):
    lengths = [4000, 31, 900, 3, 2500, 64] * 5
    c = R.filled_cache(kv8, "e4m3", lengths, 2, seed=15, spare=40)
    R.give_pages(c, range(len(lengths)))
    g = torch.Generator(device="cuda").manual_seed(1)
    x = torch.randn((len(lengths), 20, 128), generator=g, device="cuda").half()
    cos, sin = (torch.from_numpy(t).cuda() for t in R.rope_tables(4100))
    ws = kv8.Workspace(c, len(lengths), 16)

    def step():
        return kv8.decode(c, 0, x[:, :16], x[:, 16:18], x[:, 18:], cos, sin, None, ws).clone()
    good = step()
    assert ws.errors() == 0
    time_out(ws)
    assert ws.errors() == kv8.FLAG_TIMEOUT
    assert not ws.buffer.view(torch.int32)[TICKETS].any()
    for _ in range(3):
        assert torch.equal(step(), good)
    # the other flags leave the tickets, which calls in flight may be using, alone
    ws.buffer.view(torch.int32)[0] = kv8.FLAG_PAGE
    ws.buffer.view(torch.int32)[TICKETS.stop - 1] = 5
    assert ws.errors() == kv8.FLAG_PAGE
    assert int(ws.buffer.view(torch.int32)[TICKETS.stop - 1]) == 5
    ws.buffer.view(torch.int32)[TICKETS.stop - 1] = 0


def test_a_search_after_a_reported_timeout(cuda_lib):
    """The call that met the fault raises; the next one finds what the one before it found."""
    from pvlc_b200 import abi
    from pvlc_b200 import model as M
    cfg = M.ModelConfig(vision_layers=1, decoder_layers=2)
    eng = M.OcrEngine(cfg, M.init_weights(cfg, seed=3, device="cuda"))
    g = torch.Generator(device="cuda").manual_seed(5)
    grids = [(1, 8, 8), (1, 6, 4)]
    patches = [torch.randn((h * w, cfg.patch_input), generator=g, device="cuda") for _, h, w in grids]
    good = eng.generate_beam(patches, grids, 40, beams=3)
    dec = eng._beam[1]
    time_out(dec.ws)
    with pytest.raises(abi.PvlcError):
        eng.generate_beam(patches, grids, 40, beams=3)
    assert not dec.ws.buffer.view(torch.int32)[TICKETS].any()
    assert eng.generate_beam(patches, grids, 40, beams=3) == good
