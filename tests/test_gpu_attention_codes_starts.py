"""paged_attention over codes when the device holds starts and lengths of any value: rows of sequences whose own are in
order equal the reference, those of an empty context are 0, and nothing beside the output and the workspace is written."""

from __future__ import annotations

import ctypes

import pytest
import torch

import attention_reference as ref
import cache_codes_reference as codes
from attention_sinks_reference import paged
from m5kernels_amd import _lib, hip
from m5kernels_amd import attention_ops as module

pytestmark = pytest.mark.gpu

BF16, U8, I8 = torch.bfloat16, torch.uint8, torch.int8
PAGE, GUARD = 16, 4096
# query heads, key heads, width, table's pages a sequence, new tokens, (splits above 1, few)
FORMS = {"few": (8, 2, 64, 24, [4, 3, 5], False, True), "few split": (8, 1, 128, 300, [4, 3, 5], True, True),
         "tiles": (128, 128, 128, 24, [130, 4, 140], False, False)}


def _ints(device, values):
    return torch.tensor(values, dtype=torch.int32, device=device)


def _case(form, mode):
    hq, hkv, d, width, new, split, few = FORMS[form]
    g = torch.Generator().manual_seed(3)
    kc, ks = codes.held(1, 3 * 24, hkv, PAGE, d, PAGE, mode, 0.5)
    vc, vs = codes.held(2, 3 * 24, hkv, PAGE, d, PAGE, mode, 0.5)
    table = torch.full((3, width), -1, dtype=torch.int32)
    table[:, :24] = torch.randperm(3 * 24, generator=g).reshape(3, 24)
    return dict(q=torch.randn(hq, sum(new), d, generator=g).to(BF16), k=kc, v=vc, ks=ks, vs=vs, table=table)


def _guarded(n, dtype, device):
    whole = torch.full((n + 2 * GUARD,), 77, dtype=dtype, device=device)
    return whole, whole[GUARD:GUARD + n]


def _call(c, form, starts, context, window, sinks, device):
    """The C entry, its output and workspace inside larger buffers."""
    hq, hkv, d, width, new, split, few = FORMS[form]
    t = {n: x.to(device) for n, x in c.items()}
    held = {n: x.clone() for n, x in t.items()}
    tokens, mode = sum(new), _lib.QUANT_FP8 if c["k"].dtype == U8 else _lib.QUANT_INT8
    splits, is_few = module._plan(module._coded_plan(mode, d, False), tokens, hq, hkv, 3,
                                  module._reach(width * PAGE, window, sinks, True), hip._cu_count_of(0))
    assert (splits > 1, is_few) == (split and not window, few), (splits, is_few)
    whole, out = _guarded(tokens * hq * d, BF16, device)
    n = splits * tokens * hq * (d + 2) if splits > 1 else 0
    whole_ws, ws = _guarded(n, torch.float32, device)
    rows = [[*x.stride()[:3]] for x in (t["k"], t["v"])]
    exps = [[*x.stride()[:2]] for x in (t["ks"], t["vs"])]
    p, s, l = _lib.ptr, _ints(device, starts), _ints(device, context)
    _lib.call("m5k_paged_attention_codes", p(t["q"]), _lib.BF16, tokens, hq, d, *t["q"].stride()[:2], mode, p(t["k"]),
              *rows[0], p(t["ks"]), *exps[0], p(t["v"]), *rows[1], p(t["vs"]), *exps[1], PAGE, t["k"].shape[0], PAGE,
              hkv, p(t["table"]), width, 3, p(s), p(l), ctypes.c_float(d ** -0.5), window, sinks, ctypes.c_float(0.0),
              None, None, p(out), splits, p(ws) if n else None, n, _lib.stream_of(out))
    torch.cuda.synchronize()
    for w, k in ((whole, tokens * hq * d), (whole_ws, n)):
        assert (w[:GUARD] == 77).all() and (w[GUARD + k:] == 77).all()
    assert all(torch.equal(x, t[name]) for name, x in held.items())
    return out.view(tokens, hq * d).cpu()


@pytest.mark.parametrize("window,sinks", [(0, 0), (200, 3)])
@pytest.mark.parametrize("mode", [U8, I8])
@pytest.mark.parametrize("form", FORMS)
def test_lengths_of_any_value(form, mode, window, sinks, device):
    c, new = _case(form, mode), FORMS[form][4]
    starts = [0, new[0], new[0] + new[1], sum(new)]
    k, v = (codes.cache(c[n], c[n + "s"]).to(BF16) for n in "kv")
    own = [300, 40, 384]
    options = dict(window=window, sinks=sinks) if window else {}
    out, slack = paged(c["q"], k, v, c["table"], starts, own, **options)
    for bad in ((None, -2 ** 31, 2 ** 31 - 1), (2 ** 31 - 1, None, 0), (-7, 2 ** 30, None), (-1, None, None),
                (None, None, None)):
        context = [o if b is None else b for o, b in zip(own, bad)]
        got = _call(c, form, starts, context, window, sinks, device)
        for b, (s, e) in enumerate(zip(starts[:-1], starts[1:])):
            if bad[b] is None:
                assert ref.close(got[s:e], out[s:e], slack[s:e]) <= 0, (bad, b)
            elif bad[b] <= 0:
                assert not got[s:e].any(), (bad, b)


@pytest.mark.parametrize("starts", [(0, 70, 3, 12), (90, 80, 40, 0), (0, -5, 2 ** 31 - 1, -2 ** 31), (5, 5, 5, 2)])
@pytest.mark.parametrize("form", FORMS)
def test_starts_in_no_order(form, starts, device):
    """Rows may hold anything then: the call ends, and writes its own buffers alone."""
    c = _case(form, U8)
    _call(c, form, starts, [300, 40, 384], 0, 0, device)
    _call(c, form, starts, [2 ** 31 - 1, -5, 384], 200, 3, device)
