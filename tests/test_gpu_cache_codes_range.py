"""Keys that paged_append turns beyond FP32's range on their way into a cache in 8 bits: infinities, so that their block is
NaN, and no other block is."""

from __future__ import annotations

import math

import pytest
import torch

import attention_reference as ref
import cache_codes_reference as codes
import m5kernels_amd as m5

pytestmark = pytest.mark.gpu

U8, I8, BF16, F32 = torch.uint8, torch.int8, torch.bfloat16, torch.float32
LARGEST = torch.finfo(F32).max


@pytest.mark.parametrize("mode", [U8, I8])
@pytest.mark.parametrize("dtype", [BF16, F32])
@pytest.mark.parametrize("sign", [1, -1])
def test_turned_beyond_the_range(sign, dtype, mode, device):
    """An eighth of a turn a position: 3e38 beside 3e38 becomes 4.2e38, 2e38 beside 2e38 2.8e38, in range."""
    f = torch.full((4,), math.pi / 4, dtype=torch.float64)
    k = torch.ones(2, 48, 64, dtype=F32)
    k[0, 17, 2], k[0, 17, 6] = sign * 3e38, -sign * 3e38
    k[1, 35, 1], k[1, 35, 5] = sign * 2e38, sign * 2e38
    k = k.to(dtype)
    table, starts, context = (torch.tensor(x, dtype=torch.int32) for x in ([[2, 0, 1]], [0, 48], [48]))
    turned = ref.rotate(k, torch.arange(48), f)
    assert (turned[0, 17].abs() > LARGEST).sum() == 1 and (turned.abs() > LARGEST).sum() == 1
    turned[turned.abs() > LARGEST] = float("inf")
    want = torch.zeros(3, 2, 16, 64, dtype=mode), torch.zeros(3, 2, 1, dtype=U8)
    got, v = ([t.to(device) for t in want] for _ in range(2))
    codes.append(turned, *want, table, starts, context)
    assert (want[1] == 255).sum() == 1 and want[1][0, 0, 0] == 255
    m5.paged_append(k.to(device), k.to(device), got[0], v[0], *(t.to(device) for t in (table, starts, context)),
                    frequencies=f.to(device), k_scales=got[1], v_scales=v[1])
    assert torch.equal(got[1].cpu(), want[1]) and torch.equal(got[0].cpu(), want[0])
    assert (v[1].cpu() < 255).all()
