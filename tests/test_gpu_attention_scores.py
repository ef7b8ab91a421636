"""Scores of every size: huge ones, ones far below zero, infinite ones, in each form that a call can take."""

from __future__ import annotations

import math

import pytest
import torch

import m5kernels_amd as m5
from m5kernels_amd import attention_ops, hip

pytestmark = pytest.mark.gpu

BF16, F16 = torch.bfloat16, torch.float16
# name -> (query heads, key heads, tokens, keys, splits): waves that share 32 rows, tiles of 128 rows, each split or not.
FORMS = {"few": (4, 2, 40, 150, False), "few split": (4, 2, 3, 3000, True), "tiles": (256, 256, 130, 150, False),
         "tiles split": (3, 1, 47, 4500, True)}


def _shape(form):
    hq, hkv, tokens, keys, split = FORMS[form]
    got = attention_ops._plan(0, tokens, hq, hkv, 0, keys, hip._cu_count_of(0))
    assert got[1] == form.startswith("few") and (got[0] > 1) == split, got
    return hq, hkv, tokens, keys


def _whole(seed, lo, hi, *shape):
    """Whole numbers lo..hi as float64."""
    g = torch.Generator().manual_seed(seed)
    return torch.randint(lo, hi + 1, shape, generator=g).double()


def _softmax(score, visible):
    """Softmax over the visible keys in 64 bits: 0 where a row sees none, NaN where it sees infinities only."""
    p = torch.softmax(score.masked_fill(~visible, -math.inf), -1)
    return torch.where(visible.any(-1, keepdim=True), p, 0.0)


def _causal(tokens, keys):
    return torch.arange(keys)[None, :] <= torch.arange(tokens)[:, None] + keys - tokens


@pytest.mark.parametrize("form", FORMS)
@pytest.mark.parametrize("biased", [False, True])
@pytest.mark.parametrize("dtype,d,shift", [(F16, 64, 12), (F16, 128, 26), (BF16, 64, 21), (BF16, 64, 40),
                                           (BF16, 128, 110)])
@pytest.mark.parametrize("sign", [1, -1])
def test_huge_scores(sign, dtype, d, shift, biased, form, device):
    """Scores are multiples of 2^shift, all positive or all negative (down to below -10^35), and exact: q and k are
    whole numbers times a power of two.  Keys but a row's best weigh less than e^-4096, so that the output is the
    mean of the values of its best keys: n of them add up in FP32 to n 2^-24 of max |v|, n at most the keys, and
    each weight, a power of two that need not be whole, is rounded for the product by half a step."""
    hq, hkv, tokens, keys = _shape(form)
    up, down = shift // 2, shift - shift // 2
    q = (_whole(0, 1, 3, hq, tokens, d) * 2.0 ** up).to(dtype)
    k = (sign * _whole(1, 1, 3, hkv, keys, d) * 2.0 ** down).to(dtype)
    v = torch.randn(hkv, keys, d, generator=torch.Generator().manual_seed(2)).to(dtype)
    slopes = torch.zeros(hq) if biased else None
    got = m5.attention(q.to(device), k.to(device), v.to(device), causal=True, scale=1.0,
                       slopes=None if slopes is None else slopes.to(device)).cpu().double().view(tokens, hq, d)
    for h in range(0, hq, max(1, hq // 4)):
        score = q[h].double() @ k[h * hkv // hq].double().T
        vh = v[h * hkv // hq].double()
        p, half = _softmax(score, _causal(tokens, keys)), torch.finfo(dtype).eps / 2
        want = p @ vh
        bound = half * (want.abs() + p @ vh.abs()) + keys * 2.0 ** -24 * vh.abs().max()
        assert torch.isfinite(got[:, h]).all()
        assert ((got[:, h] - want).abs() <= bound * 1.01).all()


@pytest.mark.parametrize("form", FORMS)
@pytest.mark.parametrize("d,dtype", [(64, F16), (128, BF16)])
def test_scores_of_minus_infinity(d, dtype, form, device):
    """Keys of score -inf weigh nothing beside finite ones; a row that sees only such keys is NaN, as the quotient of
    two zeros is; a row that sees no key is 0."""
    hq, hkv, tokens, keys = _shape(form)
    g = torch.Generator().manual_seed(3)
    q, k, v = (torch.randn(h, n, d, generator=g).to(dtype) for h, n in ((hq, tokens), (hkv, keys), (hkv, keys)))
    q[:, :, 0] = q[:, :, 0].abs() + 0.5
    at = keys - tokens + tokens // 2  # what half of the rows see without them
    k[:, :at, 0] = -math.inf
    cut = torch.zeros_like(k)
    cut[:, at:] = k[:, at:]
    got = m5.attention(q.to(device), k.to(device), v.to(device), causal=True).cpu().view(tokens, hq, d)
    assert torch.isnan(got[:tokens // 2]).all()
    want = m5.attention(q[:, tokens // 2:].to(device), k[:, at:].to(device), v[:, at:].to(device),
                        causal=True).cpu().view(-1, hq, d)
    rest = got[tokens // 2:].double()
    # Two runs of the same softmax: each rounds its probabilities and its output by half a step, and its sums by less.
    assert (rest - want.double()).abs().max() <= 4 * torch.finfo(dtype).eps / 2 * v.double().abs().max()
    k[:] = -math.inf
    k[:, :, 1:] = 0.0
    lost = m5.attention(q.to(device), k[:, :1].to(device), v[:, :1].to(device), causal=True).cpu().view(tokens, hq, d)
    assert (lost[:-1] == 0).all() and torch.isnan(lost[-1]).all()


@pytest.mark.parametrize("page", [16, 24])
def test_scores_of_minus_infinity_on_pages(page, device):
    """The same over a cache: a sequence whose keys all score -inf, one whose visible keys lie on pages that the cache
    lacks (0), one that has a finite key behind them."""
    hkv, d, width = 2, 64, 6
    g = torch.Generator().manual_seed(4)
    kc, vc = (torch.randn(3 * width, hkv, page, d, generator=g).to(BF16) for _ in range(2))
    q = torch.randn(4, 3, d, generator=g).to(BF16)
    q[:, :, 0] = q[:, :, 0].abs() + 0.5
    table = torch.arange(3 * width, dtype=torch.int32).view(3, width).clone()
    kc[:2 * width, :, :, 0] = -math.inf
    table[1] = -1
    last = 5 * page + 3
    kc[2 * width:, :, :, 0] = -math.inf
    kc[2 * width + 5, :, 2, 0] = 0.0  # the last key of the third sequence
    ints = lambda *x: torch.tensor(x, dtype=torch.int32, device=device)  # noqa: E731
    got = m5.paged_attention(q.to(device), kc.to(device), vc.to(device), table.to(device), ints(0, 1, 2, 3),
                             ints(last, last, last)).cpu().view(3, 4, d)
    assert torch.isnan(got[0]).all() and (got[1] == 0).all()
    assert torch.equal(got[2], vc[2 * width + 5, :, 2].repeat_interleave(2, 0))


@pytest.mark.parametrize("form", FORMS)
@pytest.mark.parametrize("low", ["first", "last"])
@pytest.mark.parametrize("bad", [math.inf, -math.inf])
@pytest.mark.parametrize("d,dtype", [(64, F16), (128, BF16)])
def test_infinite_values_of_little_weight(d, dtype, bad, low, form, device):
    """An infinity that a row sees is its output, however small the weight (here e^-256, which FP32 has no number for),
    and whichever tile, wave or split meets it; the other channels stay what they are.  Half of the keys have that
    weight, so that whole tiles, waves and splits have no other."""
    hq, hkv, tokens, keys = _shape(form)
    q = torch.ones(hq, tokens, d, dtype=dtype)
    k = (_whole(5, 0, 3, hkv, keys, 1) / d).to(dtype).repeat(1, 1, d)
    v = torch.randn(hkv, keys, d, generator=torch.Generator().manual_seed(6)).to(dtype)
    half = keys // 2
    k[:, :half] = k[:, :half] if low == "last" else -256 / d
    k[:, half:] = k[:, half:] if low == "first" else -256 / d
    want = m5.attention(q.to(device), k.to(device), v.to(device), scale=1.0).cpu().view(tokens, hq, d)
    assert torch.isfinite(want).all()
    v[:, 40 if low == "first" else keys - 50, 5] = bad
    got = m5.attention(q.to(device), k.to(device), v.to(device), scale=1.0).cpu().view(tokens, hq, d)
    assert (got[:, :, 5] == bad).all()
    got[:, :, 5] = want[:, :, 5]
    assert torch.equal(got, want)


@pytest.mark.parametrize("scale,softcap", [(2.0 ** -126, 2.0 ** -126), (0.125, 1e-20), (1e29, 1.0)])
def test_smallest_and_largest_scales(scale, softcap, device):
    """A cap of next to nothing leaves the mean of the values; caps and scales without a normal FP32 number are refused
    by either front."""
    q, k, v = (torch.randn(2, n, 64, generator=torch.Generator().manual_seed(n)).to(BF16) for n in (5, 90, 90))
    q[0] = 0.0  # a score of 0 stays one
    got = m5.attention(q.to(device), k.to(device), v.to(device), scale=scale, softcap=softcap).cpu().double()
    score = q.double() @ k.double().transpose(1, 2) * scale
    want = torch.softmax(softcap * torch.tanh(score / softcap), -1) @ v.double()
    bound = 2.0 ** -8 * (want.abs() + v.double().abs().mean(1, keepdim=True)) + 2.0 ** -14
    if softcap == 1.0:  # weights of up to e^2 the mean's, off by the cap's 2^-22 and half a step
        bound = bound * 8
    assert ((got.view(5, 2, 64).transpose(0, 1) - want).abs() <= bound).all()
    for bad in (dict(softcap=1e-50), dict(scale=1e-50), dict(softcap=2.0 ** -127), dict(scale=4.0, softcap=2.0 ** -126)):
        with pytest.raises(ValueError, match="scale|softcap"):
            m5.attention(q.to(device), k.to(device), v.to(device), **bad)


@pytest.mark.parametrize("form", ["few", "few split", "tiles", "tiles split"])
@pytest.mark.parametrize("d,dtype", [(64, F16), (128, BF16)])
@pytest.mark.parametrize("softcap", [3.0, 127.0, 129.0, 200.0, 500.0])
def test_caps_that_bite(softcap, d, dtype, form, device):
    """Scores of both signs from far below the cap to five times it.  They are exact: q is one whole number a row, k
    whole numbers times a power of two, and q . k is below 2^24 steps.  So the capped score is off by what tanh and its
    product cost: the short form (caps to 128) by 2^-22 cap, the long one by its exponential, reciprocal, sum and
    result, four steps of at most 2^-23 cap, and either by the roundings of the argument (2^-23 of y sech^2 y, below
    half of that again), the scaling to base 2 and the difference from the maximum (2^-23 cap each): 2^-20 cap in
    all.  A weight is then off by that much twice (its own score and the sum's), its rounding adds half a step."""
    hq, hkv, tokens, keys = _shape(form)
    q, k = torch.zeros(hq, tokens, d), torch.zeros(hkv, keys, d)
    q[:, :, 0] = _whole(7, -4, 4, hq, tokens).float()
    k[:, :, 0] = _whole(8, -64, 64, hkv, keys).float() * 2.0 ** round(math.log2(5 * softcap / 256))
    q, k = q.to(dtype), k.to(dtype)
    v = torch.randn(hkv, keys, d, generator=torch.Generator().manual_seed(9)).to(dtype)
    got = m5.attention(q.to(device), k.to(device), v.to(device), scale=1.0, softcap=softcap).cpu().double()
    got, half, off = got.view(tokens, hq, d), torch.finfo(dtype).eps / 2, 2.0 ** -20 * softcap + keys * 2.0 ** -24
    bites = 0
    for h in range(0, hq, max(1, hq // 4)):
        score, vh = q[h].double() @ k[h * hkv // hq].double().T, v[h * hkv // hq].double()
        p = torch.softmax(softcap * torch.tanh(score / softcap), -1)
        tiny = keys * 2.0 ** -25 if dtype == F16 else 0.0  # probabilities below float16's normal range
        slack = (half + 2 * off) * (p @ vh.abs()) + tiny * vh.abs().max()
        want = p @ vh
        bound = slack + half * (want.abs() + slack)
        assert ((got[:, h] - want).abs() <= bound).all()
        bites += int(((torch.softmax(score, -1) @ vh - want).abs() > 4 * bound).sum())
    assert bites > 0  # without the cap the outputs are others


@pytest.mark.parametrize("form", FORMS)
@pytest.mark.parametrize("low", ["first", "last"])
@pytest.mark.parametrize("infinite", [False, True])
def test_huge_values_of_little_weight(infinite, low, form, device):
    """Finite values of weight e^-256 (2^-369) leave nothing in the output, also where infinities in another channel are
    kept.  They are as large as the sums hold: keys times 2^8, the largest weight against a running maximum, times 2^104
    is below 2^128 with 4500 keys."""
    hq, hkv, tokens, keys = _shape(form)
    q, half = torch.ones(hq, tokens, 64, dtype=BF16), keys // 2
    k = (_whole(5, 0, 3, hkv, keys, 1) / 64).to(BF16).repeat(1, 1, 64)
    v = torch.randn(hkv, keys, 64, generator=torch.Generator().manual_seed(6)).to(BF16)
    little = slice(0, half) if low == "first" else slice(half, keys)
    k[:, little] = -4.0
    v[:, 40 if low == "first" else keys - 50, 5] = math.inf if infinite else 0.0
    v[:, :, 6:8] = 0.0
    want = m5.attention(q.to(device), k.to(device), v.to(device), scale=1.0).view(tokens, hq, 64)
    v[:, little, 6], v[:, little, 7] = 2.0 ** 100, -2.0 ** 104
    got = m5.attention(q.to(device), k.to(device), v.to(device), scale=1.0).view(tokens, hq, 64)
    assert (got[..., 6:] == want[..., 6:]).all() and (got[..., 6:8] == 0).all()
    assert torch.equal(got[..., :6], want[..., :6])


@pytest.mark.parametrize("form", FORMS)
@pytest.mark.parametrize("low", ["first", "last"])
def test_nan_of_little_weight(low, form, device):
    hq, hkv, tokens, keys = _shape(form)
    q, half = torch.ones(hq, tokens, 64, dtype=F16), keys // 2
    k = (_whole(5, 0, 3, hkv, keys, 1) / 64).to(F16).repeat(1, 1, 64)
    v = torch.randn(hkv, keys, 64, generator=torch.Generator().manual_seed(6)).to(F16)
    k[:, :half] = k[:, :half] if low == "last" else -4.0
    k[:, half:] = k[:, half:] if low == "first" else -4.0
    v[:, 40 if low == "first" else keys - 50, 5] = math.nan
    got = m5.attention(q.to(device), k.to(device), v.to(device), scale=1.0).view(tokens, hq, 64)
    assert torch.isnan(got[..., 5]).all() and torch.isfinite(got[..., :5]).all() and torch.isfinite(got[..., 6:]).all()
