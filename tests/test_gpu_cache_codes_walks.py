"""paged_append and paged_read in 8 bits where a workgroup walks over several heads (cache_walk_cases.py), against
cache_codes_reference.py bit for bit: the next head's values and exponents are on their way beside a head's."""

from __future__ import annotations

import pytest
import torch

import attention_reference as ref
import cache_codes_reference as codes
import m5kernels_amd as m5
from cache_walk_cases import CASES, HEADS
from test_gpu_cache_codes import Case, _randn, _same

pytestmark = pytest.mark.gpu

U8, I8 = torch.uint8, torch.int8


@pytest.mark.parametrize("mode,layout", [(U8, "half"), (I8, "interleaved")])
@pytest.mark.parametrize("name", CASES)
def test_walks(name, mode, layout, device):
    s = CASES[name]
    case = Case(s["new"], s["context"], hkv=HEADS, d=s["d"], page=s["page"], block=s["block"], mode=mode, seed=21)
    # Old blocks whose exponents differ from head to head, below and above those of the new tokens.
    for scales in (case.k_scales, case.v_scales):
        for h in range(HEADS):
            scales[:, h] = (scales[:, h].long() + (h % 5 - 2) * 2).to(U8)
    options, turned = {}, None
    if s["hq"]:
        f, _ = m5.rope_frequencies(s["d"], device="cpu")
        q = _randn(9, s["hq"], sum(s["new"]), s["d"])
        options = dict(q=q.to(device), frequencies=f.to(device), layout=layout)
        turned = ref.rotate(case.k, case.positions(), f, layout)
    out, got = case.append(device, **options)
    want = case.want(turned)
    _same(got, want)
    if s["hq"]:
        exact = ref.rotate(q, case.positions(), f, layout)
        # Two products and a sum in FP32, of a cosine and sine off by a unit, and the rounding to BF16.
        size = q.double().abs() + 3 * q.double().abs().amax(2, keepdim=True) * 2.0 ** -4
        assert ((out.cpu().double() - exact).abs() <= exact.abs() * 2.0 ** -8 + size * 2.0 ** -18).all()
    tokens = sum(s["new"])
    back = m5.paged_read(got["k_codes"], got["v_codes"], *case.tables(device), tokens, k_scales=got["k_scales"],
                         v_scales=got["v_scales"])
    for x, n in zip(back, "kv"):
        whole = codes.cache(want[n + "_codes"], want[n + "_scales"])
        rows = [ref.gather(whole, case.table[b], c, s["page"])[0][:, c - m:]
                for b, (c, m) in enumerate(zip(s["context"], s["new"]))]
        assert torch.equal(x.cpu(), torch.cat(rows, 1).to(x.dtype))
