"""Outputs right beside what a call reads, in one allocation, are taken; on it they are refused."""
import pytest
import torch

import kv8_ref as R

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def kv8(cuda_lib):
    from pvlc_b200 import kv8
    return kv8


@pytest.mark.parametrize("batch", [1, 3])
def test_decode_beside_its_inputs(kv8, batch):
    from pvlc_b200 import abi
    lengths = [100, 31, 7][:batch]
    c = R.filled_cache(kv8, "e4m3", lengths, 2, seed=40, spare=9)
    R.give_pages(c, range(batch))
    g = torch.Generator(device="cuda").manual_seed(1)
    qkv, n = 20 * 128, 16 * 128 * batch
    # out, the projection's rows, each with a gap behind it that holds another out, and out
    buf = torch.randn(2 * n + batch * (qkv + n), generator=g, device="cuda").half()
    rows = buf[n:n + batch * (qkv + n)].view(batch, qkv + n)
    q, k, v = (x.unflatten(1, (-1, 128)) for x in rows[:, :qkv].split([2048, 256, 256], 1))
    outs = [buf[:n], buf[-n:], rows[0, qkv:], rows[-1, qkv:]]
    cos, sin = (torch.from_numpy(t).cuda() for t in R.rope_tables(200))
    ws = kv8.Workspace(c, batch, 16)

    def step(out):
        return kv8.decode(c, 0, q, k, v, cos, sin, None, ws, out=out)
    want = step(None)
    for o in outs:
        o = o.view(batch, 16, 128)
        assert torch.equal(step(o), want)
    for at in (16, n - 16, n + qkv - 256 - 16, n + 512):
        with pytest.raises(abi.PvlcError):
            step(buf[at:at + n].view(batch, 16, 128))
    assert torch.equal(step(None), want) and ws.errors() == 0
