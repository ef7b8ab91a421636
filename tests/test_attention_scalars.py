"""Scales and caps that FP32, in which the kernels take them, has no normal number for, on the CPU: a cap that became 0
would be no cap, and a scale over a cap that became infinite would make scores of 0 NaN."""

from __future__ import annotations

import ctypes

import pytest
import torch

import m5kernels_amd as m5
from m5kernels_amd import _lib

LEAST = 2.0 ** -126


def _call(**options):
    """paged_attention() has the same checks of them, behind that of its caches' device."""
    q, k = torch.zeros(4, 3, 64, dtype=torch.bfloat16), torch.zeros(2, 3, 64, dtype=torch.bfloat16)
    return m5.attention(q, k, k, **options)


@pytest.mark.parametrize("options,text", [
    (dict(softcap=1e-50), "softcap"), (dict(softcap=LEAST / 2), "softcap"), (dict(scale=1e-50), "scale"),
    (dict(scale=LEAST / 2), "scale"), (dict(scale=4.0, softcap=LEAST), "scale / softcap"),
    (dict(scale=1e29, softcap=1e-10), "scale / softcap"),
])
def test_refused(options, text):
    with pytest.raises(ValueError, match=text):
        _call(**options)


@pytest.mark.parametrize("options", [dict(softcap=LEAST, scale=LEAST), dict(softcap=1e-20), dict(scale=LEAST),
                                     dict(scale=1e29, softcap=1.0)])
def test_taken(options):
    with pytest.raises(ValueError, match="ROCm"):  # all that is left to refuse: the tensors are on the CPU
        _call(**options)


def test_the_c_entries_refuse_them():
    lib, p = _lib.load(), ctypes.c_void_p(64)
    for scale, cap in ((LEAST / 2, 0.0), (1.0, LEAST / 2), (4.0, LEAST), (1e29, 1e-10)):
        assert lib.m5k_attention(p, _lib.BF16, 4, 4, 64, 256, 64, p, 256, 64, p, 256, 64, 4, 2, scale, 0, 0, cap, None,
                                 None, 0, None, p, 1, None, 0, None) == 1
        assert b"scale" in lib.m5k_last_error()
