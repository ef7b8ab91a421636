"""paged_attention over a cache in 8 bits against a plain form in 64 bits: the same reference and slack as for 16-bit
caches, on the values that the codes stand for (exact in the inputs' type)."""

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


def _ints(*values):
    return torch.tensor(values, dtype=torch.int32)


def _case(new, context, *, hq=8, hkv=2, d=64, page=32, block=16, mode=U8, dtype=BF16, seed=0):
    need = [-(-max(c, 0) // page) for c in context]
    pages = sum(need) + 2
    g = torch.Generator().manual_seed(seed)
    order = torch.randperm(pages, generator=g).to(torch.int32)
    table = torch.full((len(new), max(need) + 1), -1, dtype=torch.int32)
    at = 0
    for b, n in enumerate(need):
        table[b, :n] = order[at:at + n]
        at += n
    q = torch.randn(hq, sum(new), d, generator=g).to(dtype)
    kc, ks = codes.held(seed + 1, pages, hkv, page, d, block, mode, 0.5)
    vc, vs = codes.held(seed + 2, pages, hkv, page, d, block, mode, 0.5)
    return dict(q=q, k=kc, v=vc, ks=ks, vs=vs, table=table, starts=torch.tensor([0, *new]).cumsum(0).to(torch.int32),
                context=_ints(*context))


def _got(c, device, **options):
    moved = {n: o.to(device) if isinstance(o, torch.Tensor) else o for n, o in options.items()}
    t = {n: x.to(device) for n, x in c.items()}
    return m5.paged_attention(t["q"], t["k"], t["v"], t["table"], t["starts"], t["context"], k_scales=t["ks"],
                              v_scales=t["vs"], **moved)


def _want(c, **options):
    k, v = (codes.cache(c[n], c[n + "s"]).to(c["q"].dtype) for n in "kv")
    return paged(c["q"], k, v, c["table"], c["starts"], c["context"], **options)


def _check(c, device, **options):
    got = _got(c, device, **options)
    assert got.dtype == c["q"].dtype
    excess = ref.close(got, *_want(c, **options))
    assert excess <= 0, excess


@pytest.mark.parametrize("mode", [U8, I8])
@pytest.mark.parametrize("dtype", [BF16, F16])
@pytest.mark.parametrize("d,page,block", [(64, 16, 16), (64, 48, 48), (128, 64, 64), (128, 96, 32), (128, 256, 128)])
def test_single_tokens(d, page, block, dtype, mode, device):
    _check(_case([1] * 9, [1, 0, 15, 16, 17, 64, 65, 200, 333], d=d, page=page, block=block, mode=mode, dtype=dtype),
           device)


@pytest.mark.parametrize("mode", [U8, I8])
@pytest.mark.parametrize("dtype", [BF16, F16])
@pytest.mark.parametrize("d,page,block", [(64, 16, 16), (64, 48, 48), (128, 64, 64), (128, 96, 32), (128, 256, 128)])
def test_chunks(d, page, block, dtype, mode, device):
    _check(_case([70, 1, 0, 129, 33], [70, 300, 10, 260, 1000], d=d, page=page, block=block, mode=mode, dtype=dtype),
           device)


def _forms(tokens, heads, kv_heads, sequences, keys, mode=U8, d=128, modified=False):
    kind = module._coded_plan(_lib.QUANT_FP8 if mode == U8 else _lib.QUANT_INT8, d, modified)
    return module._plan(kind, tokens, heads, kv_heads, sequences, keys, 256)


@pytest.mark.parametrize("mode,dtype", [(U8, BF16), (I8, F16), (I8, BF16)])
@pytest.mark.parametrize("d", [64, 128])
def test_tiles_of_128_rows(d, dtype, mode, device):
    """Rows enough for the form whose waves share key tiles, unsplit, with and without the rest of the options."""
    c = _case([700, 350, 1], [900, 350, 40], hq=128, hkv=64, d=d, mode=mode, dtype=dtype, page=32, block=32)
    splits, few = _forms(1051, 128, 64, 3, c["table"].shape[1] * 32, mode, d)
    assert not few and splits == 1
    _check(c, device)
    _check(c, device, softcap=20.0, slopes=torch.exp2(-8 * torch.arange(1, 129).float() / 128))


@pytest.mark.parametrize("mode", [U8, I8])
@pytest.mark.parametrize("new,context", [([1], [5000]), ([2], [4097]), ([33, 1], [3000, 700]), ([300], [9000])])
@pytest.mark.parametrize("d", [64, 128])
def test_key_splits(new, context, d, mode, device):
    c = _case(new, context, d=d, mode=mode, page=64, block=64)
    assert _forms(sum(new), 8, 2, len(new), c["table"].shape[1] * 64, mode, d)[0] > 1
    _check(c, device)
    _check(c, device, window=300)


@pytest.mark.parametrize("options", [
    dict(window=1), dict(window=65), dict(softcap=5.0), dict(softcap=1000.0), dict(scale=0.3),
    dict(slopes=torch.exp2(-torch.arange(1, 9).float())), dict(prefix_lengths=_ints(0, 250, 3, 64)),
    dict(window=40, sinks=5), dict(window=40, sinks=5, softcap=30.0), dict(window=100, sinks=300)])
@pytest.mark.parametrize("new", [[1, 1, 1, 1], [90, 1, 37, 150]])
def test_options(new, options, device):
    _check(_case(new, [300, 310, 37, 400], d=128), device, **options)
    _check(_case(new, [300, 310, 37, 400], d=64, mode=I8, dtype=F16), device, **options)


@pytest.mark.parametrize("hq,hkv", [(1, 1), (7, 1), (14, 2), (5, 5), (64, 2)])
def test_shared_heads(hq, hkv, device):
    _check(_case([1, 20], [200, 100], hq=hq, hkv=hkv, d=128), device)


def test_padded_batch(device):
    """Idle slots, rows behind the last sequence, a context shorter than its tokens."""
    c = _case([1, 0, 5, 1], [40, 0, 3, 0], d=64)
    c["q"] = torch.cat([c["q"], torch.ones(8, 6, 64, dtype=BF16)], 1)
    got = _got(c, device).cpu().view(13, 8, 64)
    assert not got[7:].any() and not got[6].any() and not got[1:3].any() and got[:1].any() and got[3:6].any()
    _check(c, device)


@pytest.mark.parametrize("d", [64, 128])
@pytest.mark.parametrize("new", [[1, 1], [130, 60]])
def test_lacking_pages_and_lost_blocks(new, d, device):
    """Keys on no page are left out; a block of NaN reaches the rows that see it, and no others."""
    c = _case(new, [300, 200], d=d, page=32, block=16)
    c["table"][0, 3], c["table"][1, 0] = -1, 5000
    _check(c, device)
    lost = int(c["table"][0, 5])  # positions 160 .. 175 of the first sequence
    c["vs"][lost, 1, 0] = 255
    got, want = _got(c, device).cpu(), _want(c)[0]
    position = torch.arange(300 - new[0], 300)
    sees = torch.zeros(sum(new), dtype=torch.bool)
    sees[:new[0]] = position >= 160
    heads = got.view(sum(new), 8, d)
    assert heads[sees][:, 4:].isnan().all()
    assert torch.isfinite(heads[:, :4]).all() and torch.isfinite(heads[~sees]).all()
    c["vs"][lost, 1, 0] = c["vs"][lost, 1, 1]
    c["ks"][lost, 1, 0] = 255
    heads = _got(c, device).cpu().view(sum(new), 8, d)
    assert heads[sees][:, 4:].isnan().all()
    assert torch.isfinite(heads[:, :4]).all() and torch.isfinite(heads[~sees]).all()
    del want


@pytest.mark.parametrize("new", [[1], [200], [250]])
def test_codes_that_are_not_numbers(new, device):
    """E4M3's NaN in a key that the window hides, and behind the context; then where a row sees it."""
    c = _case(new, [400], d=64, page=16, block=16)
    want = _got(c, device, window=20)
    first = int(c["table"][0, 10])  # positions 160 .. 175: seen by the first rows of the longest chunk alone
    c["k"][first, :, 3], c["v"][first, :, 7, 5] = 0x7F, 0xFF
    c["v"][int(c["table"][0, 25 - 1]), :, 15] = 0x7F  # position 399, seen by the last
    c["v"][-1], c["k"][-1] = 0x7F, 0x7F
    got = _got(c, device, window=20)
    position = torch.arange(400 - new[0], 400)
    hit = (position == 399) | ((position >= 163) & (position < 163 + 24))
    assert torch.equal(got[~hit.to(device)], want[~hit.to(device)])
    assert got[position == 399].isnan().all()
    sees = (position >= 167) & (position < 183)
    assert int(sees.sum()) == (16 if new[0] == 250 else 0)
    assert got[sees].reshape(-1, 8, 64)[..., 5].isnan().all()


def test_pages_behind_32_bits(device):
    """Codes more than 2^32 bytes into the cache, pages in descending order."""
    pages, hkv, page, d = 33000, 16, 64, 128
    small = _case([40, 1], [300, 200], hq=16, hkv=hkv, d=d, page=page, block=64)
    k = torch.zeros(pages, hkv, page, d, dtype=U8, device=device)
    scales = torch.zeros(pages, hkv, 1, dtype=U8, device=device)
    n = small["k"].shape[0]
    at = torch.arange(pages - 1, pages - 1 - n, -1)
    table = torch.where(small["table"] < 0, -1, pages - 1 - small["table"]).to(torch.int32).to(device)
    k[at.to(device)], scales[at.to(device)] = small["k"].to(device), small["ks"].to(device)
    got = m5.paged_attention(small["q"].to(device), k, k, table, small["starts"].to(device),
                             small["context"].to(device), k_scales=scales, v_scales=scales)
    assert ref.close(got, *_want({**small, "v": small["k"], "vs": small["ks"]})) <= 0


@pytest.mark.parametrize("starts,context", [((0, 9, 4, 12), (20, 20, 20)), ((3, 3, 12, 12), (30, 2 ** 31 - 1, 5)),
                                            ((0, -5, 2 ** 31 - 1, 6), (10, -7, 2 ** 31 - 1)),
                                            ((0, 4, 8, 12), (-2 ** 31, 2 ** 30, 4))])
@pytest.mark.parametrize("options", [{}, dict(window=7, sinks=3)])
def test_any_starts_and_lengths(options, starts, context, device):
    """What the device holds is not checked: the call stays inside its buffers, and its rows are finite."""
    for kw in (dict(d=64), dict(d=128, mode=I8), dict(d=128, hq=256, hkv=128)):
        c = _case([4, 4, 4], [20, 20, 20], page=16, block=16, **kw)
        c["starts"], c["context"] = _ints(*starts), _ints(*context)
        got = _got(c, device, **options)
        assert got.shape == (12, c["q"].shape[0] * kw["d"])


def test_a_serving_step_in_a_graph(device):
    """Append and attention captured together and replayed for step after step, with the lengths on the device."""
    c = _case([1, 1], [33, 90], d=128, page=32, block=32)
    t = {n: x.to(device) for n, x in c.items()}
    f, _ = m5.rope_frequencies(128, device=device)
    k, v = (torch.zeros(2, 2, 128, dtype=BF16, device=device) for _ in range(2))

    def step(s):
        q = m5.paged_append(k, v, s["k"], s["v"], s["table"], s["starts"], s["context"], q=s["q"], frequencies=f,
                            k_scales=s["ks"], v_scales=s["vs"])
        return m5.paged_attention(q, s["k"], s["v"], s["table"], s["starts"], s["context"], k_scales=s["ks"],
                                  v_scales=s["vs"], window=40, sinks=4)

    eager = {n: x.clone() if n in ("k", "v", "ks", "vs") else x for n, x in t.items()}
    step(t)
    for n in ("k", "v", "ks", "vs"):
        t[n].copy_(eager[n])
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = step(t)
    for n in ("k", "v", "ks", "vs"):
        t[n].copy_(eager[n])
    g = torch.Generator().manual_seed(1)
    for i in range(5):
        k.copy_(torch.randn(2, 2, 128, generator=g).mul(2.0 ** i))
        v.copy_(torch.randn(2, 2, 128, generator=g))
        t["q"].copy_(torch.randn(8, 2, 128, generator=g))
        graph.replay()
        torch.cuda.synchronize()
        want = step(eager)
        assert torch.equal(out, want)
        assert all(torch.equal(t[n], eager[n]) for n in ("k", "v", "ks", "vs"))
        t["context"] += 1


def test_two_streams_at_once(device):
    """Two calls in key splits under way together: each has a workspace of its own."""
    sides = [{n: x.to(device) for n, x in _case([1], [9000], d=128, page=64, block=64, seed=s).items()} for s in (0, 5)]

    def call(c):
        return m5.paged_attention(c["q"], c["k"], c["v"], c["table"], c["starts"], c["context"], k_scales=c["ks"],
                                  v_scales=c["vs"])

    want = [call(c) for c in sides]
    streams = [torch.cuda.Stream() for _ in sides]
    torch.cuda.synchronize()
    for _ in range(5):
        got = []
        for c, stream in zip(sides, streams):
            with torch.cuda.stream(stream):
                got.append(call(c))
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(got, want))


def test_window_behind_a_lost_block(device):
    """A NaN block that the window has left behind is not seen."""
    c = _case([1], [400], d=128, page=16, block=16)
    want = _got(c, device, window=100)
    c["vs"][int(c["table"][0, 2])] = 255
    c["ks"][int(c["table"][0, 3])] = 255
    assert torch.equal(_got(c, device, window=100), want)
    assert _got(c, device, window=100, sinks=40).isnan().all()


@pytest.mark.parametrize("mode", [U8, I8])
@pytest.mark.parametrize("dtype", [BF16, F16])
def test_small_and_large_values(dtype, mode, device):
    """Blocks whose values are far apart: values of 2^-20 (FP16 rounds them) beside others of 2^10."""
    c = _case([1, 40], [100, 90], d=64, mode=mode, dtype=dtype)
    c["vs"][:, :, 0] = 127 - 26
    c["vs"][:, :, 1] = 127 + 3
    c["ks"][:, :, 0] = 127 - 10
    _check(c, device)


def test_appended(device):
    """The operators together: chunks, then single tokens, written into 8 bits and attended over, against 64 bits on the
    values that the reference cache holds."""
    g = torch.Generator().manual_seed(0)
    hq, hkv, d, page, block = 14, 2, 128, 32, 16
    pages = 40
    table = torch.randperm(pages, generator=g)[:36].reshape(3, 12).to(torch.int32)
    cpu = {n: torch.zeros(pages, hkv, page, d, dtype=U8) for n in ("k", "v")}
    exps = {n: torch.zeros(pages, hkv, page // block, dtype=U8) for n in ("k", "v")}
    c, e = ({n: t.to(device) for n, t in x.items()} for x in (cpu, exps))
    f, _ = m5.rope_frequencies(96, device="cpu")
    context = torch.zeros(3, dtype=torch.int32)
    for step in range(7):
        new = [[200, 3, 64], [100, 1, 1]][step] if step < 2 else [1, 1, step % 2]
        starts = torch.tensor([0, *new]).cumsum(0).to(torch.int32)
        context = context + torch.tensor(new, dtype=torch.int32)
        t = sum(new)
        q, k, v = (torch.randn(h, t, d, generator=g).to(BF16) for h in (hq, hkv, hkv))
        tables = [x.to(device) for x in (table, starts, context)]
        turned = m5.paged_append(k.to(device), v.to(device), c["k"], c["v"], *tables, q=q.to(device),
                                 frequencies=f.to(device), k_scales=e["k"], v_scales=e["v"])
        positions = torch.cat([torch.arange(int(n) - m, int(n)) for n, m in zip(context, new)])
        codes.append(ref.rotate(k, positions, f), cpu["k"], exps["k"], table, starts, context)
        codes.append(v.double(), cpu["v"], exps["v"], table, starts, context)
        values = [codes.cache(cpu[n], exps[n]).to(BF16) for n in "kv"]
        for options in ({}, dict(window=50, sinks=4)):
            got = m5.paged_attention(turned, c["k"], c["v"], *tables, k_scales=e["k"], v_scales=e["v"], **options)
            assert ref.close(got, *paged(turned.cpu(), *values, table, starts, context, **options)) <= 0


@pytest.mark.parametrize("sinks", [None, 4])
def test_both_fronts(sinks, device, monkeypatch):
    front = _lib.load_fast()
    if front is None:
        pytest.skip("the native front is not built")
    c = {n: t.to(device) for n, t in _case([1, 30], [900, 41], d=128).items()}
    got = front.paged_attention(c["q"], c["k"], c["v"], c["table"], c["starts"], c["context"], None,
                                16 if sinks else None, None, None, None, sinks, c["ks"], c["vs"])
    monkeypatch.setattr(hip, "_fast", None)
    want = m5.paged_attention(c["q"], c["k"], c["v"], c["table"], c["starts"], c["context"], k_scales=c["ks"],
                              v_scales=c["vs"], window=16 if sinks else None, sinks=sinks)
    assert got is not None and torch.equal(got, want)


def test_views_and_refusals_on_the_device(device):
    c = {n: t.to(device) for n, t in _case([1, 30], [100, 41], d=64, hkv=2).items()}
    want = m5.paged_attention(c["q"], c["k"], c["v"], c["table"], c["starts"], c["context"], k_scales=c["ks"],
                              v_scales=c["vs"])
    slot = torch.zeros(c["k"].shape[0], 32, 6, 64, dtype=U8, device=device)  # slots before heads, K and V side by side
    slot[:, :, 1:3], slot[:, :, 3:5] = c["k"].transpose(1, 2), c["v"].transpose(1, 2)
    exps = torch.zeros(c["k"].shape[0], 4, 2, dtype=U8, device=device)
    exps[:, :2], exps[:, 2:] = c["ks"], c["vs"]
    got = m5.paged_attention(c["q"], slot[:, :, 1:3].transpose(1, 2), slot[:, :, 3:5].transpose(1, 2), c["table"],
                             c["starts"], c["context"], k_scales=exps[:, :2], v_scales=exps[:, 2:])
    assert torch.equal(got, want)
    with pytest.raises(ValueError, match="contiguous"):
        bad = torch.zeros(c["k"].shape[0], 2, 4, dtype=U8, device=device)[:, :, ::2]
        m5.paged_attention(c["q"], c["k"], c["v"], c["table"], c["starts"], c["context"], k_scales=bad, v_scales=bad)
    with pytest.raises(ValueError, match="dtype"):
        m5.paged_attention(c["q"].float(), c["k"], c["v"], c["table"], c["starts"], c["context"], k_scales=c["ks"],
                           v_scales=c["vs"])


def test_graphs_and_streams(device):
    """Two captured calls that run in turn, replayed with other lengths: each as the eager call."""
    one, two = _case([1, 1], [2000, 700], d=128), _case([40, 1], [300, 2100], d=128, seed=9)
    sides = [{n: t.to(device) for n, t in c.items()} for c in (one, two)]

    def call(c):
        return m5.paged_attention(c["q"], c["k"], c["v"], c["table"], c["starts"], c["context"], k_scales=c["ks"],
                                  v_scales=c["vs"], window=500, sinks=4)

    graphs, outs = [], []
    for c in sides:
        call(c)
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            outs.append(call(c))
        graphs.append(graph)
    for step in range(3):
        for c in sides:
            c["context"] -= 7
        for graph in graphs:
            graph.replay()
        for c, out in zip(sides, outs):
            assert torch.equal(out, call(c))
    stream = torch.cuda.Stream()
    stream.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(stream):
        got = call(sides[0])
    torch.cuda.current_stream().wait_stream(stream)
    assert torch.equal(got, call(sides[0]))
