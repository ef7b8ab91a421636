"""paged_attention() with query_starts in no order: what the rows hold then is nobody's promise, but the call ends, touches
nothing but its own output, and ordered calls before and after it agree."""

from __future__ import annotations

import pytest
import torch

import m5kernels_amd as m5
from m5kernels_amd import attention_ops, hip

pytestmark = pytest.mark.gpu

BF16 = torch.bfloat16


def _ints(device, *values):
    return torch.tensor(values, dtype=torch.int32, device=device)


@pytest.mark.parametrize("form,hq,hkv,tokens,width", [("few", 8, 1, 100, 4), ("tiles", 1024, 256, 100, 4),
                                                      ("few split", 8, 1, 40, 200)])
@pytest.mark.parametrize("starts", [(0, 70, 3, 100), (0, 1000, 2, 5), (90, 80, 40, 0), (0, -5, 2 ** 31 - 1, -(2 ** 31))])
def test_starts_in_no_order(starts, form, hq, hkv, tokens, width, device):
    g = torch.Generator().manual_seed(0)
    page, d = 16, 64
    kc, vc = (torch.randn(3 * width, hkv, page, d, generator=g).to(BF16).to(device) for _ in range(2))
    q = torch.randn(hq, tokens, d, generator=g).to(BF16).to(device)
    table = torch.arange(3 * width, dtype=torch.int32, device=device).view(3, width)
    context = _ints(device, 60, 50, 64)
    got = attention_ops._plan(1, tokens, hq, hkv, 3, width * page, hip._cu_count_of(0))
    assert got[1] == form.startswith("few") and (got[0] > 1) == form.endswith("split"), got
    ordered = _ints(device, 0, 12, 30, tokens)
    held = [t.clone() for t in (q, kc, vc, table)]
    want = m5.paged_attention(q, kc, vc, table, ordered, context)
    for _ in range(3):
        assert m5.paged_attention(q, kc, vc, table, _ints(device, *starts), context).shape == want.shape
        torch.cuda.synchronize()
        assert torch.equal(m5.paged_attention(q, kc, vc, table, ordered, context), want)
    assert all(torch.equal(a, b) for a, b in zip(held, (q, kc, vc, table)))
