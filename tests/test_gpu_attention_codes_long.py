"""paged_attention over codes where one workgroup takes more keys than it looks pages and exponents up for at once: 32
tiles of 32 keys a wave (4096 keys among four waves), or 64 tiles of 64.  Blocks of 16 with exponents far apart, pages in
random order."""

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


def _case(new, context, mode, dtype, hq, hkv, d, page, seed=0):
    """Any finite codes, exponents of 16 keys 2^0 to 2^-7 of the largest."""
    need = [-(-c // page) for c in context]
    g = torch.Generator().manual_seed(seed)
    pages = sum(need)
    order = torch.randperm(pages, generator=g).to(torch.int32)
    table = torch.zeros(len(new), max(need), dtype=torch.int32)
    at = 0
    for b, n in enumerate(need):
        table[b, :n] = order[at:at + n]
        at += n
    c = dict(q=torch.randn(hq, sum(new), d, generator=g).to(dtype), table=table,
             starts=torch.tensor([0, *new]).cumsum(0).to(torch.int32),
             context=torch.tensor(context, dtype=torch.int32))
    for n, least in (("k", 127 - 15), ("v", 127 - 13)):
        x = torch.randint(0, 256, (pages, hkv, page, d), generator=g).to(U8)
        if mode == U8:
            x[(x & 127) == 127] = 0
        c[n] = x.view(mode)
        if mode == I8:
            c[n][c[n] == -128] = 0
        c[n + "s"] = torch.randint(least, least + 8, (pages, hkv, page // 16), generator=g).to(U8)
    return c


def _check(c, few, device, **options):
    mode = _lib.QUANT_FP8 if c["k"].dtype == U8 else _lib.QUANT_INT8
    hq, tokens, d = c["q"].shape
    keys = c["table"].shape[1] * c["k"].shape[2]
    reach = module._reach(keys, options.get("window", 0), options.get("sinks", 0), True)
    plan = module._plan(module._coded_plan(mode, d, False), tokens, hq, c["k"].shape[1], c["table"].shape[0], reach,
                        hip._cu_count_of(0))
    assert plan == (1, few), plan
    t = {n: x.to(device) for n, x in c.items()}
    got = m5.paged_attention(t["q"], t["k"], t["v"], t["table"], t["starts"], t["context"], k_scales=t["ks"],
                             v_scales=t["vs"], **options)
    k, v = (codes.cache(c[n], c[n + "s"]).to(c["q"].dtype) for n in "kv")
    assert ref.close(got, *paged(c["q"], k, v, c["table"], c["starts"], c["context"], **options)) <= 0


@pytest.mark.parametrize("page", [16, 64])
@pytest.mark.parametrize("mode,dtype", [(U8, BF16), (I8, BF16), (U8, F16), (I8, F16)])
@pytest.mark.parametrize("d", [64, 128])
def test_single_tokens(d, mode, dtype, page, device):
    """Two long sequences among 64: once and twice looked up again, ending inside a tile."""
    context = [1 + 3 * b for b in range(64)]
    context[5], context[40] = 9001, 4100
    c = _case([1] * 64, context, mode, dtype, 16, 8, d, page)
    _check(c, True, device)
    _check(c, True, device, window=8500, sinks=70)


@pytest.mark.parametrize("mode,dtype,d,page", [(U8, BF16, 128, 16), (I8, F16, 128, 64), (U8, F16, 64, 64),
                                               (I8, BF16, 64, 16)])
def test_tiles_of_128_rows(mode, dtype, d, page, device):
    c = _case([1100, 1], [5003, 4300], mode, dtype, 32, 32, d, page, seed=2)
    _check(c, False, device)
    _check(c, False, device, window=4400, sinks=70)
