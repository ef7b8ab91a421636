"""Caches in 8 bits and windows with first keys, on the CPU: the reference, and every refusal before a launch."""

from __future__ import annotations

import ctypes

import pytest
import torch

import cache_codes_reference as codes
import m5kernels_amd as m5
from m5kernels_amd import _lib
from m5kernels_amd import attention_ops as module

BF16, U8, I8 = torch.bfloat16, torch.uint8, torch.int8


def test_reference_codes():
    """Every code stands for itself, ties go to the even one, E4M3 as torch has it."""
    every = torch.arange(256).to(U8)
    finite = (every & 127) != 127
    assert torch.equal(codes.values(every)[finite], every.view(torch.float8_e4m3fn).double()[finite])
    assert torch.equal(codes.encode(codes.values(every)[finite], U8), every[finite])
    x = torch.randn(5000, dtype=torch.float64, generator=torch.Generator().manual_seed(0)).float() * 30
    assert torch.equal(codes.encode(x.double(), U8), x.to(torch.float8_e4m3fn).view(U8))
    half = torch.tensor([0.5, 1.5, -2.5, 126.5], dtype=torch.float64)
    assert codes.encode(half, I8).tolist() == [0, 2, -2, 126]


@pytest.mark.parametrize("top,dtype,byte", [
    (0.0, U8, 0), (448.0, U8, 127), (448.5, U8, 128), (1.75, U8, 119), (1.76, U8, 120), (127.0, I8, 127),
    (127.01, I8, 128), (1.0, I8, 121), (3.4e38, U8, 247), (3.4e38, I8, 249), (float("inf"), I8, 255),
    (float("nan"), U8, 255), (1e-45, U8, 0)])
def test_reference_exponents(top, dtype, byte):
    assert codes.exponent(top, dtype) == byte


def _t(*shape, dtype=BF16):
    return torch.zeros(*shape, dtype=dtype)


def _vectors(sequences=3, width=4):
    return (torch.zeros(sequences, width, dtype=torch.int32), torch.zeros(sequences + 1, dtype=torch.int32),
            torch.zeros(sequences, dtype=torch.int32))


def _call(op, **change):
    a = dict(k=_t(2, 5, 64), v=_t(2, 5, 64), q=_t(4, 5, 64), k_cache=_t(6, 2, 32, 64, dtype=U8),
             v_cache=_t(6, 2, 32, 64, dtype=U8), k_scales=_t(6, 2, 2, dtype=U8), v_scales=_t(6, 2, 2, dtype=U8))
    kw = {n: change.pop(n) for n in list(change) if n not in a}
    a.update(change)
    scales = dict(k_scales=a["k_scales"], v_scales=a["v_scales"])
    if op == "append":
        return m5.paged_append(a["k"], a["v"], a["k_cache"], a["v_cache"], *_vectors(), **scales, **kw)
    if op == "read":
        return m5.paged_read(a["k_cache"], a["v_cache"], *_vectors(), kw.pop("tokens", 5), **scales, **kw)
    return m5.paged_attention(a["q"], a["k_cache"], a["v_cache"], *_vectors(), **scales, **kw)


BOTH = ("k_cache", "v_cache")


@pytest.mark.parametrize("op", ["append", "read", "attend"])
@pytest.mark.parametrize("change,error", [
    (dict(v_scales=None), ValueError), (dict(k_scales=_t(6, 2, 2)), ValueError),
    (dict(k_scales=_t(6, 2, dtype=U8)), ValueError), (dict(k_scales=_t(6, 2, 1, dtype=U8)), ValueError),
    (dict(k_scales=_t(5, 2, 2, dtype=U8), v_scales=_t(5, 2, 2, dtype=U8)), ValueError),
    (dict(k_scales=_t(6, 2, 0, dtype=U8), v_scales=_t(6, 2, 0, dtype=U8)), ValueError),
    (dict(k_scales=_t(6, 2, 3, dtype=U8), v_scales=_t(6, 2, 3, dtype=U8)), ValueError),  # blocks that do not divide
    (dict(k_scales=_t(6, 2, 4, dtype=U8), v_scales=_t(6, 2, 4, dtype=U8)), NotImplementedError),  # of 8 tokens
    (dict(k_cache=_t(6, 2, 32, 64), v_cache=_t(6, 2, 32, 64)), ValueError),  # no codes
    (dict(v_cache=_t(6, 2, 32, 64, dtype=I8)), ValueError),  # of two kinds
    (dict(k_cache=_t(6, 2, 32, 96, dtype=U8), v_cache=_t(6, 2, 32, 96, dtype=U8)), NotImplementedError),
    ({}, ValueError),  # CPU tensors
])
def test_refusals(op, change, error):
    with pytest.raises(error):
        _call(op, **change)


def test_blocks_are_limited():
    scales = _t(6, 2, 1, dtype=U8)
    wide = dict(k_cache=_t(6, 2, 256, 64, dtype=U8), v_cache=_t(6, 2, 256, 64, dtype=U8))
    with pytest.raises(NotImplementedError, match="16 to 128"):
        _call("read", k_scales=scales, v_scales=scales, **wide)


def test_read_needs_scales():
    with pytest.raises(ValueError, match="needs k_scales"):
        _call("read", k_scales=None, v_scales=None)


@pytest.mark.parametrize("options", [
    dict(sinks=4), dict(sinks=0, window=8), dict(sinks=-1, window=8), dict(sinks=True, window=8),
    dict(sinks=2.0, window=8)])
def test_sinks_refusals(options):
    q, k = _t(4, 5, 64), _t(2, 5, 64)
    with pytest.raises(ValueError):
        m5.attention(q, k, k, causal=True, **options)
    with pytest.raises(ValueError, match="sinks" if options["sinks"] != 4 else "ROCm|sinks"):
        module._first_keys(options["sinks"], options.get("window"))


def test_reach():
    assert module._reach(1000, 10, 0, True) == 1000  # without first keys the plan is as it was
    assert module._reach(1000, 10, 4, True) == 78 and module._reach(1000, 10, 4, False) == 88
    assert module._reach(70, 10, 4, True) == 70


@pytest.mark.parametrize("kind", [-1, 3, 5, 6, 7, 8, 16, 24, 34])
def test_plans_of_no_such_cache(kind):
    n = ctypes.c_int()
    lib = _lib.load()
    assert lib.m5k_attention_plan(kind, 5, 8, 2, 3, 1000, 256, ctypes.byref(n), None) == 1
    assert b"paged" in lib.m5k_last_error()


def test_plans_by_what_the_cache_holds():
    """(key splits, whether waves share rows): codes take few rows a sequence in that form whatever their number."""
    few = lambda *a: module._plan(*a, 256)[1]  # noqa: E731
    for mode, capped in ((_lib.QUANT_FP8, False), (_lib.QUANT_INT8, True)):
        assert few(module._coded_plan(mode, 128, capped), 1024, 32, 8, 64, 2048)
        assert few(module._coded_plan(mode, 64, capped), 300, 8, 8, 300, 8192)
    assert few(module._coded_plan(_lib.QUANT_FP8, 128, True), 8192, 32, 8, 1, 8192)
    assert not few(module._coded_plan(_lib.QUANT_FP8, 128, False), 8192, 32, 8, 1, 8192)
    assert not few(module._coded_plan(_lib.QUANT_INT8, 128, True), 8192, 32, 8, 1, 8192)
    assert not few(1, 300, 8, 8, 300, 8192)


def test_c_entries_check_before_launching():
    lib = _lib.load()
    p = ctypes.c_void_p(256)  # never dereferenced
    rows = (4096, 2048, 64)

    def attend(mode=0, block=16, slot=64, exps=p, sinks=0, window=0):
        row = (4096, 2048, slot)
        return lib.m5k_paged_attention_codes(
            p, _lib.BF16, 5, 4, 64, 320, 64, mode, p, *row, exps, 4, 2, p, *row, p, 4, 2, block, 6, 32, 2, p, 4, 3, p,
            p, ctypes.c_float(0.1), window, sinks, ctypes.c_float(0), None, None, p, 1, None, 0, None)

    for kw, word in ((dict(mode=7), b"codes"), (dict(block=8), b"block"), (dict(block=24), b"block"),
                     (dict(slot=32), b"apart"), (dict(slot=72), b"aligned"), (dict(exps=None), b"null"),
                     (dict(sinks=4), b"window")):
        assert attend(**kw) == 1
        assert word in lib.m5k_last_error(), (kw, lib.m5k_last_error())

    def append(mode=0, block=16, dim=64, pairs=0, q=None, k_token=64):
        return lib.m5k_paged_append_codes(
            p, 320, k_token, p, 320, 64, _lib.BF16, 5, 2, dim, mode, p, *rows, p, 4, 2, p, *rows, p, 4, 2, block, 6, 32,
            p, 4, 3, p, p, q, 0, 0, 0, None, None, pairs, 0, ctypes.c_float(1), None)

    for kw, word in ((dict(mode=3), b"codes"), (dict(block=144), b"block"), (dict(dim=96), b"head_dim"),
                     (dict(pairs=3), b"pairs"), (dict(q=p), b"q_out"), (dict(k_token=65), b"aligned")):
        assert append(**kw) == 1
        assert word in lib.m5k_last_error(), (kw, lib.m5k_last_error())

    def read(dtype=_lib.BF16, tokens=5, out=p):
        return lib.m5k_paged_read(0, p, *rows, p, 4, 2, p, *rows, p, 4, 2, 16, 6, 32, 2, 64, p, 4, 3, p, p, tokens, out,
                                  p, dtype, None)

    for kw, word in ((dict(dtype=9), b"dtype"), (dict(tokens=0), b"tokens"),
                     (dict(out=ctypes.c_void_p(8)), b"aligned")):
        assert read(**kw) == 1
        assert word in lib.m5k_last_error(), (kw, lib.m5k_last_error())
