"""The masks, scores, pages and non-finite values of test_gpu_attention.py in each form that a call can take: waves that
share 32 rows ("few"), and tiles of 128 rows ("tiles"; many heads make the planner choose them), split and unsplit."""

from __future__ import annotations

import pytest
import torch

import attention_reference as ref
import m5kernels_amd as m5
from m5kernels_amd import attention_ops, hip

pytestmark = pytest.mark.gpu

BF16, F16 = torch.bfloat16, torch.float16
FORMS = {"few": (6, 3), "tiles": (256, 256)}


def _randn(seed, *shape, dtype=BF16):
    g = torch.Generator().manual_seed(seed)
    return torch.randn(*shape, generator=g).to(dtype)


def _ints(*values):
    return torch.tensor(values, dtype=torch.int32)


def _to(device, options):
    return {n: o.to(device) if isinstance(o, torch.Tensor) else o for n, o in options.items()}


def _slopes(hq):
    return torch.exp2(-4 * torch.arange(1, hq + 1).float() / hq)


def _check_form(form, paged, tokens, hq, hkv, sequences, keys, splits=None):
    got = attention_ops._plan(paged, tokens, hq, hkv, sequences, keys, hip._cu_count_of(0))
    assert got[1] == (form == "few") and (splits is None or (got[0] > 1) == splits), got


DENSE = [
    dict(), dict(causal=True), dict(window=40), dict(causal=True, window=70),
    dict(causal=True, document_starts=_ints(0, 1, 33, 33, 97, 150)), dict(document_starts=_ints(0, 64, 130)),
    dict(causal=True, prefix_lengths=_ints(45)), dict(causal=True, softcap=8.0), dict(softcap=500.0),
    dict(causal=True, slopes=True), dict(slopes=True, softcap=20.0, causal=True, document_starts=_ints(0, 100, 163)),
]


@pytest.mark.parametrize("form", FORMS)
@pytest.mark.parametrize("d,dtype", [(64, F16), (128, BF16)])
@pytest.mark.parametrize("options", DENSE)
def test_dense(options, d, dtype, form, device):
    hq, hkv = FORMS[form]
    options = dict(options)
    if options.get("slopes"):
        options["slopes"] = _slopes(hq)
    n = 163
    _check_form(form, 0, n, hq, hkv, len(options.get("document_starts", [0])) - 1, n, False)
    q, k, v = _randn(0, hq, n, d, dtype=dtype), _randn(1, hkv, n, d, dtype=dtype), _randn(2, hkv, n, d, dtype=dtype)
    got = m5.attention(q.to(device), k.to(device), v.to(device), **_to(device, options))
    assert ref.close(got, *ref.dense(q, k, v, **options)) <= 0


@pytest.mark.parametrize("hq,hkv,tokens", [(3, 1, 47), (1, 1, 129)])
def test_split_tiles(hq, hkv, tokens, device):
    """Tiles of 128 rows whose keys are split, some splits behind the causal mask of every row or before the window."""
    keys = 4500
    _check_form("tiles", 0, tokens, hq, hkv, 0, keys, True)
    q, k, v = _randn(0, hq, tokens, 64), _randn(1, hkv, keys, 64), _randn(2, hkv, keys, 64)
    for options in (dict(), dict(causal=True), dict(causal=True, window=700), dict(softcap=20.0, window=1500)):
        got = m5.attention(q.to(device), k.to(device), v.to(device), **options)
        assert ref.close(got, *ref.dense(q, k, v, **options)) <= 0


PAGED = [dict(), dict(window=50), dict(softcap=30.0), dict(slopes=True), dict(prefix_lengths=_ints(30, 0, 1000, 9))]


def _paged(form, page, d, dtype, seed=3):
    hq, hkv = FORMS[form]
    new, contexts = [90, 1, 0, 77], [150, 77, 20, 77]
    g = torch.Generator().manual_seed(seed)
    need = [-(-c // page) for c in contexts]
    pages, width = sum(need) + 2, max(need) + 1
    order = torch.randperm(pages, generator=g).to(torch.int32)
    table = torch.full((4, width), -1, dtype=torch.int32)
    kc, vc = (torch.full((pages, hkv, page, d), float("nan"), dtype=dtype) for _ in range(2))
    at = 0
    for b, (n, c) in enumerate(zip(need, contexts)):
        table[b, :n] = order[at:at + n]
        at += n
        j = torch.arange(c)
        kc[table[b].long()[j // page], :, j % page] = torch.randn(c, hkv, d, generator=g).to(dtype)
        vc[table[b].long()[j // page], :, j % page] = torch.randn(c, hkv, d, generator=g).to(dtype)
    starts = torch.tensor([0] + new).cumsum(0).to(torch.int32)
    q = torch.randn(hq, int(starts[-1]) + 5, d, generator=g).to(dtype)
    _check_form(form, 1, q.shape[1], hq, hkv, 4, width * page)
    return q, kc, vc, table, starts, _ints(*contexts)


@pytest.mark.parametrize("form", FORMS)
@pytest.mark.parametrize("page", [16, 24, 64, 5])
@pytest.mark.parametrize("d,dtype", [(64, F16), (128, BF16)])
@pytest.mark.parametrize("options", PAGED)
def test_paged(options, d, dtype, page, form, device):
    args, options = _paged(form, page, d, dtype), dict(options)
    if options.get("slopes"):
        options["slopes"] = _slopes(args[0].shape[0])
    got = m5.paged_attention(*(t.to(device) for t in args), **_to(device, options))
    assert ref.close(got, *ref.paged(*args, **options)) <= 0


@pytest.mark.parametrize("form", FORMS)
@pytest.mark.parametrize("page", [16, 24])
def test_pages_that_the_cache_lacks(page, form, device):
    q, kc, vc, table, starts, contexts = args = _paged(form, page, 64, BF16)
    table[0, 2], table[1, 0], table[3, 1] = kc.shape[0], -7, 2 ** 31 - 1
    got = m5.paged_attention(*(t.to(device) for t in args))
    assert ref.close(got, *ref.paged(*args)) <= 0


@pytest.mark.parametrize("form", FORMS)
@pytest.mark.parametrize("bad", [float("nan"), float("inf"), -float("inf")])
@pytest.mark.parametrize("d,dtype", [(64, F16), (128, BF16)])
def test_masked_places_hold_anything(bad, d, dtype, form, device):
    hq, hkv = FORMS[form]
    n, group = 200, hq // hkv
    _check_form(form, 0, n, hq, hkv, 2, n)
    q, k, v = _randn(0, hq, n, d, dtype=dtype), _randn(1, hkv, n, d, dtype=dtype), _randn(2, hkv, n, d, dtype=dtype)
    options = dict(causal=True, document_starts=_ints(0, 90, n).to(device))
    want = m5.attention(q.to(device), k.to(device), v.to(device), **options).cpu().view(n, hq, d)
    v[:, 150, 3], v[1, 40, 5], k[0, 180] = bad, bad, bad
    got = m5.attention(q.to(device), k.to(device), v.to(device), **options).cpu().view(n, hq, d)
    seen = torch.zeros(n, hq, d, dtype=torch.bool)
    seen[150:, :, 3] = True
    seen[40:90, group:2 * group, 5] = True
    seen[180:, :group] = True
    assert torch.equal(got[~seen], want[~seen])
    assert torch.isnan(got[150:180, :, 3]).all() if bad != bad else (got[150:180, :, 3] == bad).all()
    assert not torch.isfinite(got[40:90, group:2 * group, 5]).any()


def test_non_finite_values_in_key_splits(device):
    """One split of a single token's keys holds an infinity: the others' parts stay what they are."""
    q, k, v = _randn(0, 8, 1, 128), _randn(1, 2, 6000, 128), _randn(2, 2, 6000, 128)
    _check_form("few", 0, 1, 8, 2, 0, 6000, True)
    want = m5.attention(q.to(device), k.to(device), v.to(device)).cpu().view(8, 128)
    v[1, 5000, 7] = float("inf")
    got = m5.attention(q.to(device), k.to(device), v.to(device)).cpu().view(8, 128)
    assert (got[4:, 7] == float("inf")).all()
    got[4:, 7] = want[4:, 7]
    assert torch.equal(got, want)


def test_many_sequences_are_found(device):
    """More sequences than one round of 64 probes, empty ones among them, over a wide table."""
    b, page = 300, 16
    new = [(i * 7) % 4 for i in range(b)]
    contexts = [n + (i * 37) % 90 for i, n in enumerate(new)]
    hq, hkv, d = 4, 2, 64
    width = 8
    g = torch.Generator().manual_seed(0)
    kc, vc = (torch.randn(b * width, hkv, page, d, generator=g).to(BF16) for _ in range(2))
    table = torch.randperm(b * width, generator=g).view(b, width).to(torch.int32)
    starts = torch.tensor([0] + new).cumsum(0).to(torch.int32)
    q = torch.randn(hq, int(starts[-1]) + 3, d, generator=g).to(BF16)
    args = (q, kc, vc, table, starts, _ints(*contexts))
    got = m5.paged_attention(*(t.to(device) for t in args))
    assert ref.close(got, *ref.paged(*args)) <= 0


def test_two_streams_at_once(device):
    """Two split calls in flight on two streams have workspaces of their own."""
    sets = [(_randn(i, 8, 1, 128).to(device), _randn(i + 9, 2, 9000, 128).to(device)) for i in range(2)]
    want = [m5.attention(q, k, k) for q, k in sets]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream(device=device) for _ in sets]
    got = [[], []]
    for _ in range(8):
        for i, (s, (q, k)) in enumerate(zip(streams, sets)):
            with torch.cuda.stream(s):
                got[i].append(m5.attention(q, k, k))
    torch.cuda.synchronize()
    for w, outs in zip(want, got):
        assert all(torch.equal(o, w) for o in outs)
