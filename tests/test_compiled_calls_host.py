"""What the compiled argument checks were built for, and what building them takes (no GPU needed)."""
import os
import subprocess
import sys
import types

import pytest
import torch

import pvlc_b200
from pvlc_b200 import abi

PACKAGE = os.path.dirname(os.path.dirname(abi.__file__))


def test_built_for_this_torch_and_python():
    abi.lib()
    assert abi.calls is not None
    assert abi.calls.built_for == f"{torch.__version__} {sys.implementation.cache_tag}"


@pytest.mark.parametrize("built_for", [None, "2.10.0+cu128 cpython-312", torch.__version__,
                                       f"{torch.__version__} cpython-39", ""])
def test_a_module_built_for_another_is_not_called(monkeypatch, built_for):
    """Its functions would read tensors by another layout: no compiled checks, then."""
    handle = abi.lib()
    bound = []
    other = types.SimpleNamespace(bind=lambda *a: bound.append(a))
    if built_for is not None:
        other.built_for = built_for
    monkeypatch.setattr(pvlc_b200, "_calls", other, raising=False)
    monkeypatch.setitem(sys.modules, "pvlc_b200._calls", other)
    assert abi._bind_calls(handle) is None and not bound
    other.built_for = f"{torch.__version__} {sys.implementation.cache_tag}"
    assert abi._bind_calls(handle) is other and len(bound) == 1


def make(*args):
    return subprocess.run(["make", "-C", PACKAGE, *args], capture_output=True, text=True)


def test_the_library_is_built_without_python_or_torch():
    got = make("-n", "-W", "csrc/py_calls.cpp", "lib", "PYTHON=/nonexistent")
    assert got.returncode == 0 and "py_calls" not in got.stdout, got.stdout + got.stderr
    got = make("calls", "PYTHON=/nonexistent")
    assert got.returncode == 0 and "is not built" in got.stdout, got.stdout + got.stderr


def test_the_library_loads_without_torch():
    """A program that uses the C ABI through abi.lib() alone does not wait for torch to load."""
    code = f"import sys; sys.path.insert(0, {PACKAGE!r}); from pvlc_b200 import abi; abi.lib(); " \
           "assert 'torch' not in sys.modules; assert abi.calls is not None"
    got = subprocess.run([sys.executable, "-c", code], capture_output=True, text=True)
    assert got.returncode == 0, got.stderr
    with pytest.raises(AttributeError):
        abi.no_such_name
