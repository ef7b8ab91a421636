"""Keys that paged_append turns in 64 bits on their way into a cache in 8 bits, where 32 bits would show: a magnitude
that FP32 does not have."""

from __future__ import annotations

import numpy as np
import pytest
import torch

import attention_reference as ref
import cache_codes_reference as codes
import m5kernels_amd as m5
from m5kernels_amd import _lib, hip

pytestmark = pytest.mark.gpu

U8, I8 = torch.uint8, torch.int8


def _between(magnitude, mode):
    """FP32 numbers that `magnitude` and its FP32 neighbour bring to different sides of a border between two codes of
    exponent 0, behind one that makes it the block's exponent."""
    b = codes.book(mode)
    found = [0.9 * float(b[-1]) / magnitude]
    for border in ((b[1:] + b[:-1]) / 2)[b[1:] < 0.85 * b[-1]].tolist():
        x = np.float32(border / magnitude)
        for y in (np.nextafter(x, np.float32(0)), x, np.nextafter(x, np.float32(999))):
            if (float(y) * magnitude < border) != (float(y) * float(np.float32(magnitude)) < border):
                found.append(float(y))
    return torch.tensor(found)


@pytest.mark.parametrize("native", [True, False])
@pytest.mark.parametrize("mode", [U8, I8])
def test_magnitude_in_64_bits(mode, native, device, monkeypatch):
    """A token at position 0, turned by nothing and scaled by yarn's magnitude."""
    if not native:
        monkeypatch.setattr(hip, "_fast", None)
    elif _lib.load_fast() is None:
        pytest.skip("the native front is not built")
    f, magnitude = m5.rope_frequencies(128, scaling="yarn", factor=40.0, original_length=4096, device="cpu")
    near = _between(magnitude, mode)
    assert near.numel() > 12 and magnitude != float(np.float32(magnitude))
    k = torch.zeros(2, 1, 128)
    k[0, 0, :min(near.numel(), 128)] = near[:128]
    k[1] = -k[0]
    table, starts, context = (torch.tensor(x, dtype=torch.int32) for x in ([[1]], [0, 1], [1]))
    want = torch.zeros(2, 2, 16, 128, dtype=mode), torch.zeros(2, 2, 1, dtype=U8)
    got = [t.to(device) for t in want]
    other = [t.clone() for t in want]
    v = [t.clone() for t in got]
    codes.append(ref.rotate(k, torch.tensor([0]), f, "half", magnitude), *want, table, starts, context)
    codes.append(ref.rotate(k, torch.tensor([0]), f, "half", float(np.float32(magnitude))), *other, table, starts,
                 context)
    assert (want[1][1] == 127).all() and int((want[0] != other[0]).sum()) > 20
    m5.paged_append(k.to(device), k.to(device), got[0], v[0], *(t.to(device) for t in (table, starts, context)),
                    frequencies=f.to(device), magnitude=magnitude, k_scales=got[1], v_scales=v[1])
    assert torch.equal(got[1].cpu(), want[1]) and torch.equal(got[0].cpu(), want[0])


def test_both_c_entries(device):
    """The entry with an FP32 magnitude and the one with 64 bits agree where FP32 has it."""
    k = torch.randn(2, 20, 64, generator=torch.Generator().manual_seed(1)).to(torch.bfloat16).to(device)
    f = m5.rope_frequencies(64, device=device)[0]
    table, starts, context = (torch.tensor(x, dtype=torch.int32, device=device) for x in ([[1, 0]], [0, 20], [25]))
    sides, p = [], _lib.ptr
    for name in ("m5k_paged_append_codes", "m5k_paged_append_codes64"):
        c = [torch.zeros(2, 2, 16, 64, dtype=U8, device=device) for _ in "kv"]
        e = [torch.zeros(2, 2, 1, dtype=U8, device=device) for _ in "kv"]
        rows, exps, q = (2048, 1024, 64), (2, 1), torch.empty_like(k)
        _lib.call(name, p(k), 1280, 64, p(k), 1280, 64, _lib.BF16, 20, 2, 64, _lib.QUANT_FP8, p(c[0]), *rows, p(e[0]),
                  *exps, p(c[1]), *rows, p(e[1]), *exps, 16, 2, 16, p(table), 2, 1, p(starts), p(context), p(k), 2, 1280,
                  64, p(q), p(f), 32, 0, 1.375, _lib.stream_of(k))
        sides.append([*c, *e, q])
    assert sides[0][0].any() and sides[0][4].any()
    assert all(torch.equal(a, b) for a, b in zip(*sides))
