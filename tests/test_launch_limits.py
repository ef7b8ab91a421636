"""Calls whose launch would have more threads along an axis than 32 bits count are refused by the C entries, on the
CPU."""

from __future__ import annotations

import ctypes

import pytest

from m5kernels_amd import _lib

P = ctypes.c_void_p(256)  # never dereferenced
ROWS = (4096, 2048, 128)


def _read(lib, tokens, dim):
    return lib.m5k_paged_read(_lib.QUANT_FP8, P, *ROWS, P, 4, 2, P, *ROWS, P, 4, 2, 16, 6, 32, 1, dim, P, 4, 3, P, P,
                              tokens, P, P, _lib.BF16, None)


def _append(lib, tokens, dim):
    return lib.m5k_paged_append_codes64(
        P, 320, 64, P, 320, 64, _lib.BF16, tokens, 8, dim, _lib.QUANT_FP8, P, *ROWS, P, 4, 2, P, *ROWS, P, 4, 2, 16, 6,
        32, P, 4, 3, P, P, None, 0, 0, 0, None, None, 0, 0, 1.0, None)


def _paged(lib, tokens, heads):
    return lib.m5k_paged_attention(P, _lib.BF16, tokens, heads, 64, 64, 64 * heads, P, *ROWS, P, *ROWS, 6, 32, heads, P,
                                   4, tokens, P, P, 0.1, 0, 0.0, None, None, P, 1, None, 0, None)


def _rope(lib, tokens, dim):
    return lib.m5k_rope(P, _lib.BF16, tokens, 1, dim, dim, dim, P, P, 1, 0, 1.0, P, None)


@pytest.mark.parametrize("call,sizes", [(_read, (1 << 28, 128)), (_read, ((1 << 28) - 15, 128)),
                                        (_append, (1 << 28, 64)), (_paged, (1 << 24, 63)),
                                        (_rope, (1 << 28, 254))])
def test_refused_before_the_launch(call, sizes):
    lib = _lib.load()
    assert call(lib, *sizes) == 1
    assert b"launch" in lib.m5k_last_error()


def test_reads_of_just_as_many_threads():
    """The limit that paged_read's Python layer checks is the launch's: 8 values a thread, workgroups of 256."""
    from m5kernels_amd.attention_ops import _READ_MAX

    for width in (64, 128):
        tokens = _READ_MAX // width
        assert -(-tokens * width // 2048) * 256 < 1 << 32 <= -(-(tokens + 1) * width // 2048) * 256
