"""Calls on a workspace of another device than the current one (fakes: no GPU needed)."""
import ctypes
import types

import pytest
import torch

from pvlc_b200 import abi, kv8


@pytest.mark.parametrize("status,flags", [(abi.OK, 0), (abi.DEVICE_FAULT_FLAG, 16)])
def test_errors_are_read_on_the_workspaces_device(monkeypatch, status, flags):
    """The default stream's handle is 0 on every device, so the device has to be current."""
    current, calls = [0], []

    class Device:
        def __init__(self, device):
            self.index = torch.device(device).index

        def __enter__(self):
            self.before, current[0] = current[0], self.index

        def __exit__(self, *e):
            current[0] = self.before

    def errors(ws, out, stream):
        calls.append((current[0], ws, stream))
        ctypes.cast(out, ctypes.POINTER(ctypes.c_uint32))[0] = flags
        return status
    monkeypatch.setattr(torch.cuda, "device", Device)
    monkeypatch.setattr(kv8, "_raw_stream", lambda index: 0)
    monkeypatch.setattr(abi, "lib", lambda: types.SimpleNamespace(pvlc_attn_kv8_errors=errors))
    ws = kv8.Workspace.__new__(kv8.Workspace)
    ws.device, ws.index, ws._p = torch.device("cuda:1"), 1, 4096
    assert ws.errors() == flags
    assert calls == [(1, 4096, 0)] and current == [0]
