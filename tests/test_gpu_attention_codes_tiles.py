"""paged_attention over codes in the form whose waves share tiles of 128 rows: first keys, and the careful second run
that missing pages and numbers which are not finite bring about.  Every case asks the plan for its form."""

from __future__ import annotations

import pytest
import torch

import attention_reference as ref
import cache_codes_reference as codes
import m5kernels_amd as m5
from attention_sinks_reference import paged
from m5kernels_amd import _lib, hip
from m5kernels_amd import attention_ops as module

pytestmark = pytest.mark.gpu

BF16, F16, U8, I8 = torch.bfloat16, torch.float16, torch.uint8, torch.int8
NEW, CONTEXT, PAGE, BLOCK = [500, 300, 1], [700, 300, 40], 32, 16


def _case(mode, dtype, d, *, hq=40, hkv=40, seed=0):
    need = [-(-c // PAGE) for c in CONTEXT]
    pages = sum(need) + 2
    g = torch.Generator().manual_seed(seed)
    order = torch.randperm(pages, generator=g).to(torch.int32)
    table = torch.full((3, max(need) + 1), -1, dtype=torch.int32)
    at = 0
    for b, n in enumerate(need):
        table[b, :n] = order[at:at + n]
        at += n
    q = torch.randn(hq, sum(NEW), d, generator=g).to(dtype)
    kc, ks = codes.held(seed + 1, pages, hkv, PAGE, d, BLOCK, mode, 0.5)
    vc, vs = codes.held(seed + 2, pages, hkv, PAGE, d, BLOCK, mode, 0.5)
    return dict(q=q, k=kc, v=vc, ks=ks, vs=vs, table=table, starts=torch.tensor([0, *NEW]).cumsum(0).to(torch.int32),
                context=torch.tensor(CONTEXT, dtype=torch.int32))


def _got(c, device, **options):
    """The call, in tiles of 128 rows and one key split."""
    mode = _lib.QUANT_FP8 if c["k"].dtype == U8 else _lib.QUANT_INT8
    hq, tokens, d = c["q"].shape
    kind = module._coded_plan(mode, d, "softcap" in options)
    keys = module._reach(c["table"].shape[1] * PAGE, options.get("window", 0), options.get("sinks", 0), True)
    plan = module._plan(kind, tokens, hq, c["k"].shape[1], 3, keys, hip._cu_count_of(0))
    assert plan == (1, False), plan
    t = {n: x.to(device) for n, x in c.items()}
    return m5.paged_attention(t["q"], t["k"], t["v"], t["table"], t["starts"], t["context"], k_scales=t["ks"],
                              v_scales=t["vs"], **options)


def _want(c, **options):
    k, v = (codes.cache(c[n], c[n + "s"]).to(c["q"].dtype) for n in "kv")
    return paged(c["q"], k, v, c["table"], c["starts"], c["context"], **options)


def _sees(first, last, window=None, sinks=0):
    """Which rows see one of the first sequence's keys first .. last."""
    sees = torch.zeros(sum(NEW), dtype=torch.bool)
    p = torch.arange(CONTEXT[0] - NEW[0], CONTEXT[0])
    sees[:NEW[0]] = (p >= first) & ((p - last < (window or 1 << 30)) | (first < sinks))
    return sees


KINDS = [(U8, BF16, 64), (U8, BF16, 128), (I8, F16, 64), (I8, F16, 128), (U8, F16, 128)]


@pytest.mark.parametrize("mode,dtype,d", KINDS)
@pytest.mark.parametrize("options", [
    dict(window=40, sinks=5),  # apart from the windows of all rows but the first
    dict(window=100, sinks=300),  # inside some rows' windows, behind others'
    dict(window=1, sinks=130), dict(window=200, sinks=64), dict(window=65, sinks=1)])
def test_first_keys(options, mode, dtype, d, device):
    c = _case(mode, dtype, d)
    assert ref.close(_got(c, device, **options), *_want(c, **options)) <= 0


@pytest.mark.parametrize("options", [dict(window=40, sinks=5, softcap=20.0), dict(window=90, sinks=200, softcap=500.0)])
def test_first_keys_under_a_cap(options, device):
    c = _case(I8, F16, 64, hq=80)
    assert ref.close(_got(c, device, **options), *_want(c, **options)) <= 0


@pytest.mark.parametrize("mode,dtype,d", KINDS)
@pytest.mark.parametrize("options", [{}, dict(window=90, sinks=70)])
def test_lacking_pages(options, mode, dtype, d, device):
    """Keys on no page are left out, first ones among them."""
    c = _case(mode, dtype, d, seed=4)
    c["table"][0, 1], c["table"][0, 15], c["table"][1, 0] = -1, 5000, -7
    assert ref.close(_got(c, device, **options), *_want(c, **options)) <= 0


@pytest.mark.parametrize("mode,dtype,d", KINDS)
@pytest.mark.parametrize("options", [{}, dict(window=90, sinks=70)])
@pytest.mark.parametrize("which", ["ks", "vs"])
def test_lost_blocks(which, options, mode, dtype, d, device):
    """A block of NaN reaches the rows that see it in the heads that hold it, and no others: keys 400 .. 415, or the
    first keys 48 .. 63."""
    c = _case(mode, dtype, d, seed=8)
    want = [t.view(sum(NEW), 40, d) for t in _want(c, **options)]
    for page, block, first in ((12, 1, 400), (1, 1, 48)):
        at = int(c["table"][0, page])
        kept = int(c[which][at, 3, block])
        c[which][at, 3, block] = 255
        got = _got(c, device, **options).view(sum(NEW), 40, d).cpu()
        sees = _sees(first, first + 15, options.get("window"), options.get("sinks", 0))
        assert sees.any() and not sees.all()
        assert got[sees][:, 3].isnan().all()
        keep = torch.ones(sum(NEW), 40, dtype=torch.bool)
        keep[sees, 3] = False
        assert ref.close(got[keep], *(t[keep] for t in want)) <= 0
        c[which][at, 3, block] = kept


@pytest.mark.parametrize("d", [64, 128])
@pytest.mark.parametrize("which", ["k", "v"])
def test_hidden_codes_that_are_no_numbers(which, d, device):
    """E4M3's NaN in one key of a head that windows hide from some rows, in a page of all heads, and behind a context."""
    c = _case(U8, BF16, d, seed=12)
    options = dict(window=60, sinks=10)
    want = [t.view(sum(NEW), 40, d) for t in _want(c, **options)]
    c[which][int(c["table"][0, 13]), 5, 7, 3] = 0x7F  # key 423
    c[which][int(c["table"][2, 1]), :, 20] = 0xFF  # behind the third sequence's 40 keys
    assert int(c["table"][0, 14]) == c[which].shape[0] - 1
    c[which][-1] = 0x7F  # keys 448 .. 479
    got = _got(c, device, **options).view(sum(NEW), 40, d).cpu()
    one, page = _sees(423, 423, 60), _sees(448, 479, 60)
    assert int(one.sum()) == 60 and int(page.sum()) == 91
    lost = torch.zeros(sum(NEW), 40, d, dtype=torch.bool)
    lost[one, 5, 3 if which == "v" else slice(None)] = True
    lost[page] = True
    assert got[lost].isnan().all()
    assert ref.close(got[~lost], *(t[~lost] for t in want)) <= 0


@pytest.mark.parametrize("d", [64, 128])
@pytest.mark.parametrize("sign", [1, -1])
def test_infinities(sign, d, device):
    """Values beyond FP16's range are infinities in the rows that see them, and nothing elsewhere."""
    c = _case(I8, F16, d, seed=16)
    at = int(c["table"][0, 10])  # keys 320 .. 351; block of 320 .. 335
    c["v"][at, 2, :16] = 0
    c["v"][at, 2, 4, 9] = sign * 100  # key 324
    c["vs"][at, 2, 0] = 127 + 12
    options = dict(window=300)
    clean = {n: t.clone() for n, t in c.items()}
    clean["v"][at, 2, 4, 9] = 0
    without = [t.view(sum(NEW), 40, d) for t in _want(clean, **options)]
    got = _got(c, device, **options).view(sum(NEW), 40, d).cpu()
    sees = _sees(324, 324, 300)
    assert 0 < int(sees.sum()) < NEW[0]
    assert (got[sees][:, 2, 9] == sign * float("inf")).all()
    keep = torch.ones(sum(NEW), 40, d, dtype=torch.bool)
    keep[sees, 2, 9] = False
    assert ref.close(got[keep], *(t[keep] for t in without)) <= 0
