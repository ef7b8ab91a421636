"""attention() and paged_attention() against a plain form in 64 bits (attention_reference.py), at the sizes and masks
where tiles, pages, splits and intervals end.  The tolerance of each case is derived there, from roundings."""

from __future__ import annotations

import pytest
import torch

import attention_reference as ref
import m5kernels_amd as m5
from m5kernels_amd import attention_ops as attn_module

pytestmark = pytest.mark.gpu

BF16, F16 = torch.bfloat16, torch.float16


def _randn(seed, *shape, dtype=BF16):
    g = torch.Generator().manual_seed(seed)
    return torch.randn(*shape, generator=g).to(dtype)


def _ints(*values):
    return torch.tensor(values, dtype=torch.int32)


def _dense(device, hq, hkv, tokens, keys, d, dtype, seed=0, **options):
    q, k, v = _randn(seed, hq, tokens, d, dtype=dtype), _randn(seed + 1, hkv, keys, d, dtype=dtype), _randn(
        seed + 2, hkv, keys, d, dtype=dtype)
    moved = {n: o.to(device) if isinstance(o, torch.Tensor) else o for n, o in options.items()}
    got = m5.attention(q.to(device), k.to(device), v.to(device), **moved)
    assert got.shape == (tokens, hq * d) and got.dtype == dtype
    excess = ref.close(got, *ref.dense(q, k, v, **options))
    assert excess <= 0, excess


@pytest.mark.parametrize("dtype", [BF16, F16])
@pytest.mark.parametrize("d", [64, 128])
@pytest.mark.parametrize("tokens,keys", [(1, 1), (1, 63), (3, 64), (31, 65), (32, 1), (129, 129), (200, 517)])
def test_full(tokens, keys, d, dtype, device):
    _dense(device, 4, 2, tokens, keys, d, dtype)


@pytest.mark.parametrize("hq,hkv", [(1, 1), (3, 1), (7, 1), (14, 2), (5, 5), (64, 2)])
def test_shared_heads(hq, hkv, device):
    _dense(device, hq, hkv, 37, 91, 128, BF16, causal=True)


@pytest.mark.parametrize("tokens,keys", [(1, 70), (70, 70), (200, 64), (64, 200), (130, 131), (5, 0)])
def test_causal_aligned_at_the_end(tokens, keys, device):
    """More tokens than keys: the first of them see nothing and are 0."""
    _dense(device, 4, 4, tokens, keys, 64, BF16, causal=True)


@pytest.mark.parametrize("causal", [False, True])
@pytest.mark.parametrize("window", [1, 2, 63, 64, 65, 1000])
def test_window(window, causal, device):
    _dense(device, 2, 1, 300, 300, 64, F16, causal=causal, window=window)


@pytest.mark.parametrize("causal", [False, True])
@pytest.mark.parametrize("starts", [(0, 300), (0, 0, 300), (0, 1, 2, 64, 64, 128, 300), (0, 100, 250), (0, 0),
                                    (0, 65, 66, 299)])
def test_documents(starts, causal, device):
    """Empty documents, single tokens, and rows behind the last document (0)."""
    _dense(device, 4, 2, 300, 300, 128, BF16, causal=causal, document_starts=_ints(*starts))


@pytest.mark.parametrize("prefix", [0, 1, 40, 64, 299, 5000, -3])
def test_prefix(prefix, device):
    _dense(device, 3, 3, 300, 300, 64, BF16, causal=True, prefix_lengths=_ints(prefix))


def test_prefix_of_each_document(device):
    _dense(device, 3, 3, 300, 300, 64, BF16, causal=True, document_starts=_ints(0, 100, 100, 299),
           prefix_lengths=_ints(30, 7, 500))


@pytest.mark.parametrize("d,dtype", [(64, F16), (128, BF16)])
@pytest.mark.parametrize("softcap,biased", [(20.0, False), (0.5, False), (1e4, False), (None, True), (5.0, True)])
def test_capped_and_biased_scores(softcap, biased, d, dtype, device):
    slopes = torch.exp2(-torch.arange(1, 5).float()) if biased else None
    _dense(device, 4, 2, 150, 190, d, dtype, causal=True, softcap=softcap, slopes=slopes)
    _dense(device, 4, 2, 90, 190, d, dtype, softcap=softcap, slopes=slopes, scale=0.3)


def test_documents_with_bias_and_window(device):
    _dense(device, 4, 1, 400, 400, 128, BF16, causal=True, window=50, slopes=torch.tensor([0.5, 0.25, 0.0, -0.01]),
           document_starts=_ints(0, 130, 131, 400))


@pytest.mark.parametrize("tokens,keys", [(1, 5000), (2, 4097), (33, 3000)])
@pytest.mark.parametrize("d", [64, 128])
def test_key_splits(tokens, keys, d, device):
    """Few rows over many keys: the keys are split and the parts joined."""
    assert attn_module._plan(0, tokens, 8, 2, 0, keys, 256)[0] > 1
    _dense(device, 8, 2, tokens, keys, d, BF16, causal=True)
    _dense(device, 8, 2, tokens, keys, d, BF16, causal=True, window=300)


def test_large_scores(device):
    """Scores of several hundred, rising along the keys, so that the running maximum moves in every tile."""
    q, k, v = _randn(0, 1, 40, 64), _randn(1, 1, 700, 64), _randn(2, 1, 700, 64)
    k = (k.float() * torch.linspace(0.1, 40, 700)[None, :, None]).to(BF16)
    got = m5.attention(q.to(device), k.to(device), v.to(device))
    assert ref.close(got, *ref.dense(q, k, v)) <= 0


@pytest.mark.parametrize("bad", [float("nan"), float("inf"), -float("inf")])
@pytest.mark.parametrize("d,dtype", [(64, F16), (128, BF16)])
def test_masked_places_hold_anything(bad, d, dtype, device):
    """Non-finite keys and values reach the rows that see them and no others."""
    q, k, v = _randn(0, 4, 200, d, dtype=dtype), _randn(1, 2, 200, d, dtype=dtype), _randn(2, 2, 200, d, dtype=dtype)
    options = dict(causal=True, document_starts=_ints(0, 90, 200))
    want = m5.attention(q.to(device), k.to(device), v.to(device), causal=True,
                        document_starts=options["document_starts"].to(device))
    v[:, 150, 3], v[1, 40, 5], k[0, 180] = bad, bad, bad
    got = m5.attention(q.to(device), k.to(device), v.to(device), causal=True,
                       document_starts=options["document_starts"].to(device)).cpu().view(200, 4, d)
    want = want.cpu().view(200, 4, d)
    seen = torch.zeros(200, 4, d, dtype=torch.bool)
    seen[150:, :, 3] = True
    seen[40:90, 2:, 5] = True
    seen[180:, :2] = True
    assert torch.equal(got[~seen], want[~seen])
    value = got[150:180, :, 3]
    assert torch.isnan(value).all() if bad != bad else (value == bad).all()
    assert not torch.isfinite(got[40:90, 2:, 5]).any()


def test_opposite_infinities_make_nan(device):
    q, k, v = _randn(0, 1, 8, 64), _randn(1, 1, 8, 64), _randn(2, 1, 8, 64)
    v[0, 2, 0], v[0, 5, 0] = float("inf"), -float("inf")
    got = m5.attention(q.to(device), k.to(device), v.to(device), causal=True).cpu()
    assert torch.isfinite(got[:2]).all() and (got[2:5, 0] == float("inf")).all() and torch.isnan(got[5:, 0]).all()
    assert torch.isfinite(got[:, 1:]).all()


def test_views_of_a_projection(device):
    """Heads as strided views of one [tokens, all heads * D] tensor, rows of it not at multiples of 16 bytes, and
    an expanded key head."""
    for width in (8 * 64, 8 * 64 + 4):
        y = _randn(3, 50, width)
        heads = y[:, :512].view(50, 8, 64) if width == 512 else y[:, :512].unflatten(1, (8, 64))
        q, k, v = heads[:, :4].transpose(0, 1), heads[:, 4:6].transpose(0, 1), heads[:, 6:].transpose(0, 1)
        yd = y.to(device)
        hd = yd[:, :512].unflatten(1, (8, 64))
        got = m5.attention(hd[:, :4].transpose(0, 1), hd[:, 4:6].transpose(0, 1), hd[:, 6:].transpose(0, 1),
                           causal=True)
        assert ref.close(got, *ref.dense(q, k, v, causal=True)) <= 0
    k1 = _randn(4, 1, 50, 64).expand(2, 50, 64)
    got = m5.attention(hd[:, :4].transpose(0, 1), k1.to(device).expand(2, 50, 64), k1.to(device).expand(2, 50, 64))
    assert ref.close(got, *ref.dense(q, k1, k1)) <= 0


def test_no_tokens(device):
    e = torch.empty(2, 0, 64, dtype=BF16, device=device)
    assert m5.attention(e, e, e).shape == (0, 128)


# ---- over a paged cache -----------------------------------------------------------------------------


def _cache(hkv, d, dtype, page, table_width, contexts, seed, spare=2, fill=float("nan")):
    """Caches whose unowned slots hold `fill`, and a table of pages in random order (unused entries -1)."""
    g = torch.Generator().manual_seed(seed)
    need = [-(-max(c, 0) // page) for c in contexts]
    order = torch.randperm(sum(need) + spare, generator=g).to(torch.int32)
    table = torch.full((len(contexts), table_width), -1, dtype=torch.int32)
    kc = torch.full((sum(need) + spare, hkv, page, d), fill, dtype=dtype)
    vc = kc.clone()
    at = 0
    for b, (n, c) in enumerate(zip(need, contexts)):
        table[b, :n] = order[at:at + n]
        at += n
        j = torch.arange(max(c, 0))
        kc[table[b].long()[j // page], :, j % page] = torch.randn(len(j), hkv, d, generator=g).to(dtype)
        vc[table[b].long()[j // page], :, j % page] = torch.randn(len(j), hkv, d, generator=g).to(dtype)
    return kc, vc, table


def _paged(device, hq, hkv, d, dtype, page, new, contexts, behind=0, extra_width=1, **options):
    width = max(1, max(-(-max(c, 0) // page) for c in contexts) + extra_width)
    kc, vc, table = _cache(hkv, d, dtype, page, width, contexts, 5)
    starts = torch.tensor([0] + new).cumsum(0).to(torch.int32)
    context = _ints(*contexts)
    q = _randn(6, hq, int(starts[-1]) + behind, d, dtype=dtype)
    moved = {n: o.to(device) if isinstance(o, torch.Tensor) else o for n, o in options.items()}
    got = m5.paged_attention(q.to(device), kc.to(device), vc.to(device), table.to(device), starts.to(device),
                             context.to(device), **moved)
    excess = ref.close(got, *ref.paged(q, kc, vc, table, starts, context, **options))
    assert excess <= 0, excess
    return got


@pytest.mark.parametrize("page", [1, 7, 16, 24, 64, 100, 512])
@pytest.mark.parametrize("d,dtype", [(64, F16), (128, BF16)])
def test_pages(page, d, dtype, device):
    """Pages that end inside a tile, single-key pages, pages longer than a tile; what lies behind the context is NaN."""
    _paged(device, 4, 2, d, dtype, page, [1, 70, 3, 130], [200, 70, 65, 333])


@pytest.mark.parametrize("group", [1, 3, 7, 8, 16])
def test_single_tokens(group, device):
    _paged(device, 2 * group, 2, 128, BF16, 16, [1] * 9, [1, 2, 15, 16, 17, 64, 65, 700, 1500])


def test_idle_slots_and_rows_behind(device):
    """Contexts of 0, sequences without new tokens, a context shorter than its tokens, rows behind the last sequence."""
    got = _paged(device, 4, 2, 64, BF16, 16, [1, 0, 1, 5, 0], [0, 40, 33, 3, 0], behind=150)
    assert (got[-150:] == 0).all() and (got[0] == 0).all()


def test_long_context_is_split(device):
    assert attn_module._plan(1, 1, 8, 1, 1, 9000, 256)[0] > 1
    _paged(device, 8, 1, 128, BF16, 64, [1], [8765])
    _paged(device, 8, 1, 64, BF16, 16, [2, 1], [3000, 40], behind=3)


@pytest.mark.parametrize("options", [dict(window=100), dict(window=1), dict(softcap=10.0), dict(scale=0.2),
                                     dict(slopes=torch.tensor([0.5, 0.1, 0.01, 0.0])),
                                     dict(prefix_lengths=_ints(50, 0, 1000, 100), softcap=30.0)])
def test_masks_and_scores(options, device):
    _paged(device, 4, 2, 128, BF16, 16, [100, 1, 40, 64], [400, 300, 40, 64], **options)


def test_pages_that_the_cache_lacks(device):
    """Entries outside the cache inside a context: their keys are left out, other sequences are untouched."""
    kc, vc, table = _cache(2, 64, BF16, 16, 20, [200, 100], 7)
    table[0, 3], table[0, 7], table[1, 0] = -1, kc.shape[0], 2 ** 30
    starts, context, q = _ints(0, 3, 40), _ints(200, 100), _randn(8, 4, 40, 64)
    got = m5.paged_attention(q.to(device), kc.to(device), vc.to(device), table.to(device), starts.to(device),
                             context.to(device))
    assert ref.close(got, *ref.paged(q, kc, vc, table, starts, context)) <= 0


def test_strided_caches(device):
    """K and V interleaved in one allocation, slots before heads."""
    kc, vc, table = _cache(2, 64, BF16, 16, 9, [130], 9)
    both = torch.stack([kc, vc], 1).transpose(2, 3).contiguous().to(device)  # [pages, 2, slots, heads, D]
    starts, context, q = _ints(0, 130), _ints(130), _randn(8, 4, 130, 64)
    got = m5.paged_attention(q.to(device), both[:, 0].transpose(1, 2), both[:, 1].transpose(1, 2), table.to(device),
                             starts.to(device), context.to(device))
    assert ref.close(got, *ref.paged(q, kc, vc, table, starts, context)) <= 0


def test_offsets_past_32_bits(device):
    """A cache of over 2^31 elements: the last pages lie behind what 32-bit offsets reach."""
    page, hkv, d = 64, 8, 128
    pages = (1 << 31) // (hkv * page * d) + 40
    kc = torch.zeros(pages, hkv, page, d, dtype=BF16, device=device)
    vc = torch.zeros_like(kc)
    small_k, small_v, _ = _cache(hkv, d, BF16, page, 4, [256], 11, spare=0)
    table = torch.arange(pages - 4, pages, dtype=torch.int32)[None]
    kc[pages - 4:], vc[pages - 4:] = small_k.to(device), small_v.to(device)
    starts, context, q = _ints(0, 2), _ints(250), _randn(12, 8, 2, d)
    got = m5.paged_attention(q.to(device), kc, vc, table.to(device), starts.to(device), context.to(device))
    near = torch.arange(4, dtype=torch.int32)[None]
    assert ref.close(got, *ref.paged(q, small_k, small_v, near, starts, context)) <= 0


def test_other_streams_and_replays(device):
    """Two captured calls with their own workspaces and lengths that change between replays, on a side stream."""
    kc, vc, table = _cache(2, 128, BF16, 16, 128, [2000, 2000], 13)
    q = _randn(14, 8, 2, 128)
    starts, context = _ints(0, 1, 2), _ints(2000, 1500)
    dev = [t.to(device) for t in (q, kc, vc, table, starts, context)]
    m5.paged_attention(*dev)
    torch.cuda.synchronize()
    side = torch.cuda.Stream(device=device)
    graphs, outs = [], []
    for _ in range(2):
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=side):
            outs.append(m5.paged_attention(*dev))
        graphs.append(graph)
    for lengths in ((2000, 1500), (1, 700), (64, 0), (1999, 3)):
        dev[5].copy_(_ints(*lengths))
        eager = m5.paged_attention(*dev)
        for graph in graphs:
            graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(outs[0], eager) and torch.equal(outs[1], eager)
        assert ref.close(eager, *ref.paged(q, kc, vc, table, starts, _ints(*lengths))) <= 0


def test_same_bits_every_time(device):
    q, k = _randn(0, 8, 2, 128).to(device), _randn(1, 2, 6000, 128).to(device)
    first = m5.attention(q, k, k, causal=True)
    for _ in range(5):
        assert torch.equal(m5.attention(q, k, k, causal=True), first)
