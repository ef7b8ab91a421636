"""Refusals of the attention operators, on the CPU: every check that comes before a launch."""

from __future__ import annotations

import ctypes
import math

import pytest
import torch

import m5kernels_amd as m5
from m5kernels_amd import _lib
from m5kernels_amd import attention_ops as module

BF16 = torch.bfloat16


def _t(*shape, dtype=BF16):
    return torch.zeros(*shape, dtype=dtype)


def test_rope_frequencies():
    f, mag = m5.rope_frequencies(8, 100.0, device="cpu")
    assert mag == 1.0 and torch.allclose(f, torch.tensor([1.0, 100 ** -0.25, 0.1, 100 ** -0.75], dtype=torch.float64))
    assert torch.allclose(m5.rope_frequencies(8, scaling="linear", factor=4.0, device="cpu")[0],
                          m5.rope_frequencies(8, device="cpu")[0] / 4)
    ntk = m5.rope_frequencies(8, scaling="ntk", factor=4.0, device="cpu")[0] / m5.rope_frequencies(8, device="cpu")[0]
    assert ntk[0] == 1 and math.isclose(float(ntk[-1]), 0.25, rel_tol=1e-12)
    f, mag = m5.rope_frequencies(128, scaling="yarn", factor=8.0, original_length=4096, device="cpu")
    plain = m5.rope_frequencies(128, device="cpu")[0]
    turns = 4096 * plain / (2 * math.pi)
    assert torch.equal(f[turns >= 32], plain[turns >= 32])
    assert torch.allclose(f[turns <= 1], plain[turns <= 1] / 8, rtol=1e-15)
    assert ((f <= plain) & (f >= plain / 8 * (1 - 1e-15))).all()
    assert math.isclose(mag, 0.1 * math.log(8) + 1)


@pytest.mark.parametrize("args,kw,error", [
    ((7,), {}, ValueError), ((0,), {}, ValueError), ((8, -1.0), {}, ValueError), ((8, float("inf")), {}, ValueError),
    ((8,), dict(scaling="cubic"), NotImplementedError), ((8,), dict(factor=2.0), ValueError),
    ((8,), dict(scaling="linear", factor=0.5), ValueError), ((2,), dict(scaling="ntk", factor=2.0), ValueError),
    ((8,), dict(scaling="yarn", factor=2.0), ValueError),
    ((8,), dict(scaling="yarn", factor=2.0, original_length=64, fast=1.0, slow=1.0), ValueError),
])
def test_rope_frequencies_refusals(args, kw, error):
    with pytest.raises(error):
        m5.rope_frequencies(*args, device="cpu", **kw)


def _rope(**change):
    a = dict(x=_t(2, 5, 64), positions=torch.zeros(5, dtype=torch.int32),
             frequencies=torch.ones(32, dtype=torch.float64))
    kw = {k: change.pop(k) for k in ("layout", "magnitude") if k in change}
    a.update(change)
    return m5.rope(a["x"], a["positions"], a["frequencies"], **kw)


@pytest.mark.parametrize("change", [
    dict(x=_t(5, 64)), dict(x=_t(2, 5, 64, dtype=torch.int8)), dict(x=_t(0, 5, 64)),
    dict(positions=torch.zeros(4, dtype=torch.int32)), dict(positions=torch.zeros(5, dtype=torch.int64)),
    dict(frequencies=torch.ones(33, dtype=torch.float64)), dict(frequencies=torch.ones(32)),
    dict(frequencies=torch.ones(0, dtype=torch.float64)), dict(layout="third"), dict(magnitude=0.0),
    dict(magnitude=float("nan")), {},
])
def test_rope_refusals(change):
    with pytest.raises(ValueError):  # the last one for tensors that are not on the device
        _rope(**change)


def _attention(**change):
    a = dict(q=_t(4, 5, 64), k=_t(2, 5, 64), v=_t(2, 5, 64))
    a.update({k: change.pop(k) for k in ("q", "k", "v") if k in change})
    return m5.attention(a["q"], a["k"], a["v"], **change)


@pytest.mark.parametrize("change,error", [
    (dict(q=_t(3, 5, 64)), ValueError), (dict(q=_t(4, 5, 128)), ValueError), (dict(v=_t(2, 6, 64)), ValueError),
    (dict(q=_t(4, 5, 64, dtype=torch.float32), k=_t(2, 5, 64, dtype=torch.float32)), ValueError),
    (dict(q=_t(4, 5, 64, dtype=torch.float16)), ValueError), (dict(k=_t(2, 64)), ValueError),
    (dict(q=_t(4, 5, 96), k=_t(2, 5, 96), v=_t(2, 5, 96)), NotImplementedError),
    (dict(causal=1), ValueError), (dict(window=0), ValueError), (dict(window=True), ValueError),
    (dict(softcap=0.0), ValueError), (dict(softcap=-1.0), ValueError), (dict(scale=0.0), ValueError),
    (dict(scale=float("inf")), ValueError), (dict(slopes=torch.zeros(3)), ValueError),
    (dict(slopes=torch.zeros(4, dtype=torch.float64)), ValueError),
    (dict(prefix_lengths=torch.zeros(1, dtype=torch.int32)), ValueError),
    (dict(causal=True, window=3, prefix_lengths=torch.zeros(1, dtype=torch.int32)), NotImplementedError),
    (dict(document_starts=torch.zeros(1, dtype=torch.int32)), ValueError),
    (dict(q=_t(4, 6, 64), document_starts=torch.zeros(2, dtype=torch.int32)), ValueError),
    (dict(document_starts=torch.zeros(2, dtype=torch.int64)), ValueError), ({}, ValueError),
])
def test_attention_refusals(change, error):
    with pytest.raises(error):
        _attention(**change)


I32 = torch.int32


def _paged_args(**change):
    a = dict(q=_t(4, 3, 64), kc=_t(5, 2, 16, 64), vc=_t(5, 2, 16, 64), table=torch.zeros(2, 3, dtype=I32),
             starts=torch.zeros(3, dtype=I32), context=torch.zeros(2, dtype=I32))
    a.update({k: change.pop(k) for k in tuple(a) if k in change})
    return list(a.values()), change


PAGED = [
    (dict(kc=_t(5, 2, 16)), ValueError), (dict(vc=_t(5, 2, 8, 64)), ValueError),
    (dict(kc=_t(0, 2, 16, 64)), ValueError), (dict(table=torch.zeros(2, 3, dtype=torch.int64)), ValueError),
    (dict(table=torch.zeros(0, 3, dtype=I32)), ValueError), (dict(starts=torch.zeros(2, dtype=I32)), ValueError),
    (dict(context=torch.zeros(3, dtype=I32)), ValueError), ({}, ValueError),
]


@pytest.mark.parametrize("change,error", PAGED + [
    (dict(q=_t(3, 3, 64)), ValueError), (dict(window=-1), ValueError), (dict(slopes=torch.zeros(2)), ValueError),
    (dict(window=4, prefix_lengths=torch.zeros(2, dtype=I32)), NotImplementedError),
])
def test_paged_attention_refusals(change, error):
    args, kw = _paged_args(**dict(change))
    with pytest.raises(error):
        m5.paged_attention(*args, **kw)


@pytest.mark.parametrize("change,error", PAGED + [
    (dict(k=_t(2, 3, 32)), ValueError), (dict(v=_t(2, 4, 64)), ValueError),
    (dict(q=_t(4, 3, 64), f=None), ValueError), (dict(layout="third"), ValueError),
    (dict(k=_t(2, 3, 64, dtype=torch.float16)), ValueError),
])
def test_paged_append_refusals(change, error):
    change = dict(change)
    k, v, f = change.pop("k", _t(2, 3, 64)), change.pop("v", _t(2, 3, 64)), change.pop("f", None)
    q = change.pop("q", None)
    args, kw = _paged_args(**change)
    with pytest.raises(error):
        m5.paged_append(k, v, *args[1:], q=q, frequencies=f, **kw)


def test_written_caches_are_no_expanded_views():
    with pytest.raises(ValueError, match="expanded|ROCm"):
        kc = _t(1, 2, 16, 64).expand(5, 2, 16, 64)
        args, _ = _paged_args(kc=kc)
        m5.paged_append(_t(2, 3, 64), _t(2, 3, 64), *args[1:])


def test_c_entries_refuse_without_launching():
    lib = _lib.load()
    p, s, n = ctypes.c_void_p(64), ctypes.c_float(1.0), ctypes.c_int(0)

    def attention(q=p, dtype=_lib.BF16, tokens=4, heads=4, d=64, qt=64, keys=4, kvh=2, scale=1.0, causal=0, window=0,
                  cap=0.0, starts=None, docs=0, prefix=None, splits=1, ws=None, n=0):
        return lib.m5k_attention(q, dtype, tokens, heads, d, 256, qt, p, 256, 64, p, 256, 64, keys, kvh, scale, causal,
                                 window, cap, None, starts, docs, prefix, p, splits, ws, n, None)

    for bad, text in ((dict(q=None), b"null"), (dict(dtype=_lib.F32), b"dtype"), (dict(d=96), b"head_dim"),
                      (dict(heads=3), b"multiple"), (dict(tokens=0), b"positive"), (dict(qt=63), b"aligned"),
                      (dict(q=ctypes.c_void_p(68)), b"aligned"), (dict(scale=0.0), b"scale"),
                      (dict(cap=-1.0), b"softcap"), (dict(scale=float("nan")), b"scale"),
                      (dict(window=-1), b"window"), (dict(splits=0), b"splits"),
                      (dict(splits=2), b"workspace"), (dict(splits=2, ws=p, n=100), b"workspace"),
                      (dict(keys=-1), b"keys"), (dict(starts=p, docs=1, keys=5), b"documents"),
                      (dict(prefix=p), b"causal"), (dict(prefix=p, causal=1, window=2), b"combined")):
        assert attention(**bad) == 1 and text in lib.m5k_last_error(), (bad, lib.m5k_last_error())
    assert lib.m5k_attention_plan(0, 4, 3, 2, 0, 4, 256, ctypes.byref(n), None) == 1

    def rope(pairs=2, d=8, x=p, heads=2):
        return lib.m5k_rope(x, _lib.F32, 4, heads, d, 8, 8, p, p, pairs, 0, s, p, None)

    for bad in (dict(pairs=5), dict(pairs=0), dict(x=None), dict(heads=0), dict(d=0)):
        assert rope(**bad) == 1 and b"rope" in lib.m5k_last_error()


def test_plan():
    """Enough rows: tiles of 128, no split.  Few rows: waves share them, and as many workgroups as run at once split the
    keys, over 256 at least each."""
    plan = lambda *a: module._plan(*a, 256)  # noqa: E731
    assert plan(0, 4096, 56, 56, 0, 4096) == (1, False)
    assert plan(0, 1, 8, 8, 0, 255) == (1, True)
    assert plan(1, 1, 64, 8, 1, 131072) == (64, True)
    assert plan(1, 64, 64, 8, 64, 8192) == (1, False) and plan(1, 32, 64, 8, 32, 2048) == (2, True)
    splits, few = plan(1, 8, 64, 8, 8, 8192)
    assert 1 < splits <= 32 and few
    assert plan(0, 5000, 4, 1, 0, 5000) == (3, False) and plan(0, 2000, 4, 1, 0, 2000) == (1, True)
    assert plan(0, 300, 56, 56, 0, 300) == (1, False) and plan(0, 128, 56, 56, 0, 128) == (1, True)
