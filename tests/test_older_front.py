"""A native front left from a build before some of today's calls: same C ABI version, same torch, fewer functions."""

import types

import pytest
import torch

import m5kernels_amd as m5
from m5kernels_amd import _lib, hip


@pytest.fixture
def older_front(monkeypatch):
    """What load_fast() finds: a front of the projections alone."""
    module = types.SimpleNamespace(abi_version=_lib.load().m5k_abi_version(), torch_version=torch.__version__)
    for name in ("bind", "quantize", "gemm", "qk", "qkv"):
        setattr(module, name, lambda *args: None)
    spec = types.SimpleNamespace(loader=types.SimpleNamespace(exec_module=lambda m: None))
    monkeypatch.setattr(_lib.importlib.util, "spec_from_file_location", lambda *args: spec)
    monkeypatch.setattr(_lib.importlib.util, "module_from_spec", lambda s: module)
    return module


def test_it_is_refused(older_front):
    with pytest.warns(RuntimeWarning, match="paged_attention"):
        assert _lib.load_fast() is None


def test_the_python_front_takes_the_call(older_front, monkeypatch):
    monkeypatch.setattr(hip, "_fast", hip._NativeFront())
    x = torch.zeros(2, 5, 64)
    with pytest.warns(RuntimeWarning, match="build the package again"):
        with pytest.raises(ValueError, match="ROCm device tensor"):
            m5.rope(x, torch.zeros(5, dtype=torch.int32), torch.ones(32, dtype=torch.float64))


def test_every_call_is_looked_for(older_front):
    calls = {n for n in vars(hip._NativeFront) if not n.startswith("_")}
    assert calls | {"bind"} == set(_lib.FRONT_CALLS)
