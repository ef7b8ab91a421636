"""attention() and paged_attention() with a window and first keys that stay visible (`sinks`), against a plain form in
64 bits, at the sizes where the two stretches of keys meet, overlap or lie apart."""

from __future__ import annotations

import pytest
import torch

import attention_reference as ref
import attention_sinks_reference as sinks_ref
import m5kernels_amd as m5
from m5kernels_amd import _lib, hip
from m5kernels_amd import attention_ops as module

pytestmark = pytest.mark.gpu

BF16, F16 = torch.bfloat16, torch.float16


def _randn(seed, *shape, dtype=BF16):
    return torch.randn(*shape, generator=torch.Generator().manual_seed(seed)).to(dtype)


def _ints(*values):
    return torch.tensor(values, dtype=torch.int32)


def _dense(device, hq, hkv, tokens, keys, d, dtype, seed=0, **options):
    q, k, v = _randn(seed, hq, tokens, d, dtype=dtype), _randn(seed + 1, hkv, keys, d, dtype=dtype), _randn(
        seed + 2, hkv, keys, d, dtype=dtype)
    moved = {n: o.to(device) if isinstance(o, torch.Tensor) else o for n, o in options.items()}
    got = m5.attention(q.to(device), k.to(device), v.to(device), **moved)
    excess = ref.close(got, *sinks_ref.dense(q, k, v, **options))
    assert excess <= 0, excess


@pytest.mark.parametrize("causal", [False, True])
@pytest.mark.parametrize("window", [1, 2, 63, 64, 65, 1000])
@pytest.mark.parametrize("sinks", [1, 4, 32, 64, 65, 200, 5000])
def test_windows(sinks, window, causal, device):
    _dense(device, 2, 1, 300, 300, 64, F16, causal=causal, window=window, sinks=sinks)


@pytest.mark.parametrize("tokens,keys", [(1, 1), (1, 700), (3, 64), (129, 129), (200, 517), (200, 64), (5, 0),
                                         (1000, 1000)])
@pytest.mark.parametrize("d,dtype", [(64, F16), (128, BF16)])
def test_lengths(tokens, keys, d, dtype, device):
    """More tokens than keys, too: the first rows see nothing, or under no causal mask the first keys alone."""
    for causal in (True, False):
        _dense(device, 4, 2, tokens, keys, d, dtype, causal=causal, window=40, sinks=4)


@pytest.mark.parametrize("causal", [False, True])
@pytest.mark.parametrize("starts", [(0, 300), (0, 0, 300), (0, 1, 2, 64, 64, 128, 300), (0, 100, 250), (0, 0),
                                    (0, 65, 66, 299), (0, 200, 210, 300)])
@pytest.mark.parametrize("window,sinks", [(10, 3), (33, 70), (1, 1)])
def test_documents(window, sinks, starts, causal, device):
    _dense(device, 4, 2, 300, 300, 128, BF16, causal=causal, window=window, sinks=sinks, document_starts=_ints(*starts))


@pytest.mark.parametrize("d", [64, 128])
def test_tiles_of_128_rows(d, device):
    """Long documents whose rows share a workgroup with the beginnings of others, far from their own first keys."""
    starts = _ints(0, 700, 705, 1400, 1500)
    assert not module._plan(0, 1500, 64, 64, 4, module._reach(1500, 70, 5, True), 256)[1]
    _dense(device, 64, 64, 1500, 1500, d, BF16, causal=True, window=70, sinks=5, document_starts=starts)
    _dense(device, 64, 64, 1500, 1500, d, BF16, window=70, sinks=5, document_starts=starts)
    _dense(device, 64, 64, 1500, 1500, d, BF16, causal=True, window=200, sinks=130)


@pytest.mark.parametrize("d,dtype", [(64, F16), (128, BF16)])
@pytest.mark.parametrize("softcap,biased", [(20.0, False), (None, True), (5.0, True)])
def test_capped_and_biased_scores(softcap, biased, d, dtype, device):
    slopes = torch.exp2(-torch.arange(3, 7).float()) if biased else None
    _dense(device, 4, 2, 150, 390, d, dtype, causal=True, softcap=softcap, slopes=slopes, window=30, sinks=7)
    _dense(device, 4, 1, 500, 500, d, dtype, causal=True, softcap=softcap, slopes=slopes, window=30, sinks=7,
           document_starts=_ints(0, 130, 131, 480))


def _paged(device, new, context, *, hq=8, hkv=2, d=64, page=16, dtype=BF16, seed=0, spoil=False, **options):
    g = torch.Generator().manual_seed(seed)
    need = [-(-max(c, 0) // page) for c in context]
    pages = sum(need) + 2
    order = torch.randperm(pages, generator=g).to(torch.int32)
    table = torch.full((len(new), max(need) + 1), -1, dtype=torch.int32)
    at = 0
    for b, n in enumerate(need):
        table[b, :n] = order[at:at + n]
        at += n
    if spoil:
        table[0, 0] = -1
    q = torch.randn(hq, sum(new), d, generator=g).to(dtype)
    k, v = (torch.randn(pages, hkv, page, d, generator=g).to(dtype) for _ in range(2))
    args = (q, k, v, table, torch.tensor([0, *new]).cumsum(0).to(torch.int32), _ints(*context))
    moved = {n: o.to(device) if isinstance(o, torch.Tensor) else o for n, o in options.items()}
    got = m5.paged_attention(*(t.to(device) for t in args), **moved)
    excess = ref.close(got, *sinks_ref.paged(*args, **options))
    assert excess <= 0, excess


@pytest.mark.parametrize("page", [16, 24, 7, 64])
@pytest.mark.parametrize("window,sinks", [(1, 1), (40, 4), (64, 64), (100, 500), (17, 33)])
@pytest.mark.parametrize("d,dtype", [(64, F16), (128, BF16)])
def test_paged(d, dtype, window, sinks, page, device):
    _paged(device, [1, 1, 0, 1, 1], [1, 500, 9, 77, 0], d=d, dtype=dtype, page=page, window=window, sinks=sinks)
    _paged(device, [70, 1, 0, 129], [70, 300, 10, 660], d=d, dtype=dtype, page=page, window=window, sinks=sinks)


@pytest.mark.parametrize("page", [16, 24])
@pytest.mark.parametrize("d", [64, 128])
def test_far_behind_the_window(d, page, device):
    """Long contexts of which a few tiles at either end are read, in key splits where the window is long."""
    _paged(device, [1, 1], [20000, 9000], d=d, page=page, window=100, sinks=4)
    assert module._plan(1, 2, 8, 2, 2, module._reach(20064, 3000, 4, True), 256)[0] > 1
    _paged(device, [1, 1], [20000, 9000], d=d, page=page, window=3000, sinks=4)
    _paged(device, [40, 3], [5000, 9000], d=d, page=page, window=2000, sinks=300, softcap=20.0)


def test_lacking_first_page(device):
    _paged(device, [1, 30], [300, 200], d=128, window=50, sinks=20, spoil=True)


@pytest.mark.parametrize("d,dtype", [(64, F16), (128, BF16)])
def test_between_holds_anything(d, dtype, device):
    """Keys between the first ones and the window do not reach a row, NaN or not; the first ones do."""
    q, k, v = _randn(0, 4, 300, d, dtype=dtype), _randn(1, 2, 300, d, dtype=dtype), _randn(2, 2, 300, d, dtype=dtype)
    options = dict(causal=True, window=20, sinks=4)
    want = m5.attention(q.to(device), k.to(device), v.to(device), **options).cpu()
    v[:, 100, 3], k[:, 130], v[0, 120] = float("nan"), float("inf"), -float("inf")
    got = m5.attention(q.to(device), k.to(device), v.to(device), **options).cpu()
    untouched = torch.ones(300, dtype=torch.bool)
    untouched[100:150] = False
    assert torch.equal(got[untouched], want[untouched])
    v[:, 2, 5] = float("inf")
    got = m5.attention(q.to(device), k.to(device), v.to(device), **options).cpu().view(300, 4, d)
    assert (got[150:, :, 5] == float("inf")).all() and torch.isfinite(got[150:, :, 6:]).all()


def test_window_that_sees_all(device):
    """A window as long as the keys: the bits of the call without it do not have to match, the values do."""
    q, k = _randn(0, 4, 200, 128), _randn(1, 2, 200, 128)
    got = m5.attention(q.to(device), k.to(device), k.to(device), causal=True, window=200, sinks=3)
    assert ref.close(got, *ref.dense(q, k, k, causal=True)) <= 0


@pytest.mark.parametrize("documents", [False, True])
def test_both_fronts(documents, device, monkeypatch):
    front = _lib.load_fast()
    if front is None:
        pytest.skip("the native front is not built")
    q, k = _randn(0, 4, 200, 128).to(device), _randn(1, 2, 200, 128).to(device)
    starts = _ints(0, 70, 200).to(device) if documents else None
    got = front.attention(q, k, k, True, 16, starts, None, None, None, None, 4)
    assert got is not None
    assert front.attention(q, k, k, True, None, starts, None, None, None, None, 4) is None
    monkeypatch.setattr(hip, "_fast", None)
    want = m5.attention(q, k, k, causal=True, window=16, document_starts=starts, sinks=4)
    assert torch.equal(got, want)
