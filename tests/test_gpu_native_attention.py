"""The native front of the attention step: it takes plain calls, gives the bits of the Python front, and leaves every
other call to it."""

from __future__ import annotations

import pytest
import torch

import m5kernels_amd as m5
from m5kernels_amd import _lib, hip

pytestmark = pytest.mark.gpu

BF16 = torch.bfloat16


@pytest.fixture(scope="module")
def front():
    module = _lib.load_fast()
    if module is None:
        pytest.skip("the native front is not built")
    module.bind(_lib._current_raw_stream, hip._native_splits, hip._native_staged)
    return module


def _r(device, *shape, dtype=BF16, seed=0):
    g = torch.Generator().manual_seed(seed)
    return torch.randn(*shape, generator=g).to(dtype).to(device)


def _i(device, *values):
    return torch.tensor(values, dtype=torch.int32, device=device)


def _calls(device):
    """name -> (arguments of the native function, the public call)."""
    f, _ = m5.rope_frequencies(64, device=device)
    x, p = _r(device, 4, 9, 64), torch.arange(9, dtype=torch.int32, device=device)
    k, v = _r(device, 2, 9, 64, seed=1), _r(device, 2, 9, 64, seed=2)
    kc, vc = _r(device, 6, 2, 16, 64, seed=3), _r(device, 6, 2, 16, 64, seed=4)
    table = torch.tensor([[0, 3, 1], [2, 5, 4]], dtype=torch.int32, device=device)
    starts, context, slopes = _i(device, 0, 5, 9), _i(device, 40, 44), torch.rand(4, device=device)
    y = _r(device, 9, 8 * 64, seed=5).view(9, 8, 64).transpose(0, 1)  # heads of one projection, read in place
    return {
        "rope": ((x, p, f, "half", 1.0), lambda: m5.rope(x, p, f)),
        "paged_append": ((k, v, kc, vc, table, starts, context, x, f, "interleaved", 1.25),
                         lambda: m5.paged_append(k, v, kc, vc, table, starts, context, q=x, frequencies=f,
                                                 layout="interleaved", magnitude=1.25)),
        "paged_attention": ((x, kc, vc, table, starts, context, None, 30, 20.0, slopes, None),
                            lambda: m5.paged_attention(x, kc, vc, table, starts, context, window=30, softcap=20.0,
                                                       slopes=slopes)),
        "attention": ((y[:4], y[4:6], y[6:], True, None, starts, _i(device, 2, 3), None, None, 0.2),
                      lambda: m5.attention(y[:4], y[4:6], y[6:], causal=True, document_starts=starts,
                                           prefix_lengths=_i(device, 2, 3), scale=0.2)),
    }


@pytest.mark.parametrize("name", ["rope", "paged_append", "paged_attention", "attention"])
def test_takes_plain_calls_with_the_same_bits(name, front, device, monkeypatch):
    native, public = _calls(device)[name]
    got = getattr(front, name)(*native)
    assert isinstance(got, torch.Tensor)
    monkeypatch.setattr(hip, "_fast", None)
    assert torch.equal(got, public())


def test_append_without_queries(front, device, monkeypatch):
    native, _ = _calls(device)["paged_append"]
    k, v, kc, vc = native[:4]
    kc2, vc2 = kc.clone(), vc.clone()
    assert front.paged_append(*native[:7], None, None, "half", 1.0) is True
    monkeypatch.setattr(hip, "_fast", None)
    assert m5.paged_append(k, v, kc2, vc2, *native[4:7]) is None
    assert torch.equal(kc, kc2) and torch.equal(vc, vc2)


def test_key_splits_have_their_workspace(front, device, monkeypatch):
    q, k = _r(device, 8, 1, 128), _r(device, 2, 7000, 128, seed=1)
    got = front.attention(q, k, k, False, None, None, None, None, None, None)
    monkeypatch.setattr(hip, "_fast", None)
    assert torch.equal(got, m5.attention(q, k, k))


@pytest.mark.parametrize("name,at,value", [
    ("rope", 0, lambda t: t[:, :, ::2]), ("rope", 0, lambda t: t.cpu()), ("rope", 1, lambda t: t.long()),
    ("rope", 2, lambda t: t.float()), ("rope", 3, lambda t: "third"), ("rope", 4, lambda t: -1.0),
    ("rope", 4, lambda t: 1), ("rope", 4, lambda t: float("nan")), ("rope", 0, lambda t: t[:, :0]),
    ("paged_append", 1, lambda t: t[:1]), ("paged_append", 2, lambda t: t[:1].expand(6, 2, 16, 64)),
    ("paged_append", 4, lambda t: t.long()), ("paged_append", 7, lambda t: t[:, :4]),
    ("paged_append", 8, lambda t: None),
    ("paged_attention", 0, lambda t: t[:3]), ("paged_attention", 0, lambda t: t.half()),
    ("paged_attention", 5, lambda t: t[:1]), ("paged_attention", 6, lambda t: 0.0),
    ("paged_attention", 7, lambda t: 0), ("paged_attention", 7, lambda t: True),
    ("paged_attention", 7, lambda t: 1 << 70),
    ("paged_attention", 10, lambda t: torch.zeros(2, dtype=torch.int32).cuda()),
    ("attention", 3, lambda t: 1), ("attention", 1, lambda t: t[:, :5]), ("attention", 0, lambda t: t.float()),
    ("attention", 4, lambda t: 5), ("attention", 6, lambda t: t[:1]), ("attention", 9, lambda t: float("inf")),
])
def test_leaves_other_calls(name, at, value, front, device):
    native = list(_calls(device)[name][0])
    native[at] = value(native[at])
    assert getattr(front, name)(*native) is None
