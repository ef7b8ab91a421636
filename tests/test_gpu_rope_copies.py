"""Channels behind the rotated ones are copied: whatever their neighbours hold, they keep their values, infinities, NaN
and the sign of a zero included, in rope() and on the way into a cache; what two tokens for one place leave there."""

from __future__ import annotations

import math

import pytest
import torch

import m5kernels_amd as m5

pytestmark = pytest.mark.gpu

BF16, F16, F32 = torch.bfloat16, torch.float16, torch.float32


def _input(heads, tokens, d, rotary, dtype):
    x = torch.randn(heads, tokens, d, generator=torch.Generator().manual_seed(1)).to(dtype)
    special = torch.tensor([math.inf, -0.0, math.nan, 0.0, -math.inf, -0.0, 1.5], dtype=dtype)
    n = d - rotary
    for t in range(tokens):
        x[:, t, rotary:] = special.repeat(-(-n // 7) + 1)[t % 7:t % 7 + n]
    return x


def _same(got, want):
    nan = torch.isnan(want)
    assert torch.equal(torch.isnan(got), nan)
    got, want = got.masked_fill(nan, 0.0), want.masked_fill(nan, 0.0)
    assert torch.equal(got, want) and torch.equal(torch.signbit(got), torch.signbit(want))


@pytest.mark.parametrize("dtype", [BF16, F16, F32])
@pytest.mark.parametrize("layout", ["half", "interleaved"])
@pytest.mark.parametrize("d,rotary", [(64, 18), (64, 34), (64, 2), (128, 62), (40, 38), (64, 48)])
@pytest.mark.parametrize("aligned", [True, False])
def test_copied_channels(aligned, d, rotary, layout, dtype, device):
    x = _input(3, 29, d, rotary, dtype)
    f, p = m5.rope_frequencies(rotary, device=device)[0], torch.arange(29, dtype=torch.int32, device=device)
    on = x.to(device)
    if not aligned:  # rows one element further apart
        on = torch.cat([on, on[..., :1]], -1)[..., :d]
    got = m5.rope(on, p, f, layout=layout).cpu()
    assert torch.isfinite(got[..., :rotary]).all()
    _same(got[..., rotary:], x[..., rotary:])


@pytest.mark.parametrize("layout", ["half", "interleaved"])
def test_copied_channels_of_stored_keys(layout, device):
    d, rotary, page = 64, 18, 16
    k = _input(2, 29, d, rotary, BF16)
    kc, vc = (torch.zeros(2, 2, page, d, dtype=BF16, device=device) for _ in range(2))
    ints = lambda *x: torch.tensor(x, dtype=torch.int32, device=device)  # noqa: E731
    q = m5.paged_append(k.to(device), k.to(device), kc, vc, torch.tensor([[0, 1]], dtype=torch.int32, device=device),
                        ints(0, 29), ints(29), q=k.to(device), layout=layout,
                        frequencies=m5.rope_frequencies(rotary, device=device)[0])
    stored = torch.cat([kc[0], kc[1]], 1)[:, :29].cpu()
    _same(stored[..., rotary:], k[..., rotary:])
    _same(q.cpu()[..., rotary:], k[..., rotary:])
    _same(torch.cat([vc[0], vc[1]], 1)[:, :29].cpu(), k)


def test_tokens_for_one_place(device):
    """Two sequences whose tables name the same page: each element is one token's or the other's, the rest untouched."""
    k, v = (torch.randn(3, 40, 64, generator=torch.Generator().manual_seed(n)).to(BF16) for n in (1, 2))
    kc, vc = (torch.zeros(4, 3, 32, 64, dtype=BF16, device=device) for _ in range(2))
    ints = lambda *x: torch.tensor(x, dtype=torch.int32, device=device)  # noqa: E731
    table = torch.tensor([[2], [2]], dtype=torch.int32, device=device)
    m5.paged_append(k.to(device), v.to(device), kc, vc, table, ints(0, 20, 40), ints(20, 20))
    for cache, new in ((kc.cpu(), k), (vc.cpu(), v)):
        assert ((cache[2, :, :20] == new[:, :20]) | (cache[2, :, :20] == new[:, 20:])).all()
        assert (cache[2, :, 20:] == 0).all() and (cache[[0, 1, 3]] == 0).all()
