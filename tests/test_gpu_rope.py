"""rope() and paged_append() against 64-bit forms (attention_reference.py), and the serving step as a whole."""

from __future__ import annotations

import math

import pytest
import torch

import attention_reference as ref
import m5kernels_amd as m5

pytestmark = pytest.mark.gpu

BF16, F16, F32 = torch.bfloat16, torch.float16, torch.float32


def _randn(seed, *shape, dtype=BF16):
    g = torch.Generator().manual_seed(seed)
    return torch.randn(*shape, generator=g).to(dtype)


def _excess(got, want, x, magnitude=1.0):
    """|got - want| past its bound: half a step of the output, and for the FP32 steps (sine and cosine to 2^-22, two
    products and a sum of half a step each) 2^-21 of the pair's size, which is below sqrt(2) max|x|."""
    eps = torch.finfo(got.dtype).eps / 2
    work = 2.0 ** -21 * 1.5 * magnitude * x.double().abs().amax()
    tiny = torch.finfo(got.dtype).smallest_normal * torch.finfo(got.dtype).eps
    return float((got.cpu().double() - want).abs().sub(eps * (want.abs() + work) + work + tiny).max())


@pytest.mark.parametrize("dtype", [BF16, F16, F32])
@pytest.mark.parametrize("layout", ["half", "interleaved"])
@pytest.mark.parametrize("d,rotary", [(128, 128), (128, 96), (64, 18), (64, 2), (40, 40), (7, 6), (256, 34),
                                      (2048, 512)])
@pytest.mark.parametrize("heads,tokens", [(1, 1), (3, 77)])
def test_rope(heads, tokens, d, rotary, layout, dtype, device):
    f, _ = m5.rope_frequencies(rotary, device="cpu")
    x, p = _randn(1, heads, tokens, d, dtype=dtype), torch.arange(tokens, dtype=torch.int32) * 37 - 5
    got = m5.rope(x.to(device), p.to(device), f.to(device), layout=layout)
    assert got.is_contiguous() and got.shape == x.shape
    assert _excess(got, ref.rotate(x, p, f, layout), x) <= 0
    assert torch.equal(got.cpu()[..., rotary:], x[..., rotary:])


def test_far_positions_keep_their_angles(device):
    """Positions up to 2^31 - 1: the 64-bit angle itself is good to 2^-53 of its size there, 2.4e-7 rad."""
    f, magnitude = m5.rope_frequencies(64, scaling="yarn", factor=16.0, original_length=4096, device="cpu")
    x = _randn(2, 2, 5, 64, dtype=F32)
    p = torch.tensor([0, 999_999, 16_777_217, 2 ** 31 - 1, -(2 ** 31)], dtype=torch.int32)
    got = m5.rope(x.to(device), p.to(device), f.to(device), magnitude=magnitude).cpu().double()
    want = ref.rotate(x, p, f, "half", magnitude)
    near = 2.0 ** -21 * 1.5 * magnitude * float(x.abs().max())
    assert (got - want)[:, :3].abs().max() <= near + 2.0 ** -24 * 6
    assert (got - want)[:, 3:].abs().max() <= near + 2.0 ** -24 * 6 + 8 * 2.0 ** 31 * 2.0 ** -53


def test_many_heads_and_long_prompts(device):
    """Several heads a thread, the last group of them partial."""
    f, _ = m5.rope_frequencies(96, device="cpu")
    x, p = _randn(3, 11, 5000, 128), torch.arange(5000, dtype=torch.int32)
    for layout in ("half", "interleaved"):
        got = m5.rope(x.to(device), p.to(device), f.to(device), layout=layout)
        assert _excess(got, ref.rotate(x, p, f, layout), x) <= 0


def test_views_are_read_in_place(device):
    f, _ = m5.rope_frequencies(64, device="cpu")
    y, p = _randn(4, 30, 6 * 64 + 3), torch.arange(30, dtype=torch.int32)
    for ofs in (0, 3):
        heads = y[:, ofs:ofs + 384].unflatten(1, (6, 64)).transpose(0, 1)
        on = y.to(device)[:, ofs:ofs + 384].unflatten(1, (6, 64)).transpose(0, 1)
        assert _excess(m5.rope(on, p.to(device), f.to(device)), ref.rotate(heads, p, f), heads) <= 0
    wide = y[:, ::2][:, :64].unsqueeze(0)
    assert _excess(m5.rope(wide.to(device), p.to(device), f.to(device)), ref.rotate(wide, p, f), wide) <= 0


def test_agrees_with_the_projection_postprocess(device):
    """The tables of qk_norm_rope are these angles in BF16: with a norm of 1 both rotate alike, to the tables'
    rounding (half a step of the two products, 2^-9 * sqrt(2) each way) and each output's own."""
    f, _ = m5.rope_frequencies(96, device=device)
    x = _randn(5, 20, 4 * 128).to(device)
    p = torch.arange(20, dtype=torch.int32, device=device)
    angle = torch.outer(p.double(), f)
    gamma = torch.ones(128, dtype=BF16, device=device)
    got = m5.qk_norm_rope(x, gamma, angle.cos().to(BF16), angle.sin().to(BF16), epsilon=1e-6)
    z = x.double().view(20, 4, 128).transpose(0, 1)
    z = (z / torch.sqrt((z * z).mean(-1, keepdim=True) + 1e-6)).to(F32)
    want = m5.rope(z, p, f)
    assert (got.double() - want.double()).abs().max() <= 4 * 2.0 ** -8 * float(z.abs().max())


# ---- the paged cache ------------------------------------------------------------------------------


def _append_case(device, hkv, d, dtype, page, new, contexts, behind, rotary, layout, hq=0, table=None):
    starts = torch.tensor([0] + new).cumsum(0).to(torch.int32)
    context = torch.tensor(contexts, dtype=torch.int32)
    tokens = int(starts[-1]) + behind
    width = max(1, -(-max(contexts) // page))
    g = torch.Generator().manual_seed(1)
    pages = width * len(new) + 2
    if table is None:
        table = torch.randperm(pages, generator=g)[:width * len(new)].view(len(new), width).to(torch.int32)
    k, v = _randn(2, hkv, tokens, d, dtype=dtype), _randn(3, hkv, tokens, d, dtype=dtype)
    q = _randn(4, hq, tokens, d, dtype=dtype) if hq else None
    kc, vc = _randn(5, pages, hkv, page, d, dtype=dtype), _randn(6, pages, hkv, page, d, dtype=dtype)
    f = m5.rope_frequencies(rotary, device="cpu")[0] if rotary else None
    kd, vd = kc.to(device), vc.to(device)
    got = m5.paged_append(k.to(device), v.to(device), kd, vd, table.to(device), starts.to(device), context.to(device),
                          q=None if q is None else q.to(device), frequencies=None if f is None else f.to(device),
                          layout=layout)
    position = torch.zeros(tokens, dtype=torch.int64)
    kw, vw, written = kc.double(), vc.double(), torch.zeros(pages, page, dtype=torch.bool)
    for b, n in enumerate(new):
        s = int(starts[b])
        position[s:s + n] = torch.arange(n) + contexts[b] - n
    turned = k.double() if f is None else ref.rotate(k, position, f, layout)
    for b, n in enumerate(new):
        for i in range(n):
            t, p = int(starts[b]) + i, contexts[b] - n + i
            if p < 0 or p >= width * page or not 0 <= int(table[b, p // page]) < pages:
                continue
            at = int(table[b, p // page])
            kw[at, :, p % page], vw[at, :, p % page], written[at, p % page] = turned[:, t], v[:, t].double(), True
    assert torch.equal(vd.cpu().double(), vw)
    kg = kd.cpu().transpose(1, 2)
    kw = kw.transpose(1, 2)
    assert torch.equal(kg[~written].double(), kw[~written])
    assert _excess(kg[written], kw[written], k) <= 0 if written.any() else True
    if q is None:
        assert got is None
    else:
        end = int(starts[-1])
        assert _excess(got[:, :end], ref.rotate(q, position, f, layout)[:, :end], q) <= 0
        assert (got[:, end:] == 0).all()


@pytest.mark.parametrize("page", [1, 16, 24])
@pytest.mark.parametrize("layout", ["half", "interleaved"])
@pytest.mark.parametrize("dtype,d,rotary,hq", [(BF16, 128, 128, 14), (F16, 64, 18, 4), (F32, 64, 64, 2),
                                               (BF16, 64, 0, 0), (BF16, 30, 30, 2), (F16, 128, 96, 0)])
def test_append(dtype, d, rotary, hq, layout, page, device):
    """Chunks and single tokens, an empty sequence, an idle slot, a context shorter than its tokens, rows behind."""
    _append_case(device, 2, d, dtype, page, [1, 0, 50, 1, 4], [33, 40, 50, 0, 2], 7, rotary, layout, hq)


def test_append_skips_what_the_cache_lacks(device):
    table = torch.tensor([[0, -1, 2], [9999, 4, 5]], dtype=torch.int32)
    _append_case(device, 2, 64, BF16, 16, [40, 45], [40, 48], 0, 64, "half", 2, table)
    _append_case(device, 2, 64, BF16, 16, [3, 3], [30, 48], 0, 64, "half", 2, table)


def test_append_into_strided_caches(device):
    both = torch.zeros(6, 16, 2, 2, 64, dtype=BF16, device=device)  # [pages, slots, K and V, heads, D]
    kc, vc = both[:, :, 0].transpose(1, 2), both[:, :, 1].transpose(1, 2)
    k, v = _randn(1, 2, 20, 64).to(device), _randn(2, 2, 20, 64).to(device)
    table = torch.tensor([[3, 1]], dtype=torch.int32, device=device)
    one = lambda *x: torch.tensor(x, dtype=torch.int32, device=device)  # noqa: E731
    assert m5.paged_append(k, v, kc, vc, table, one(0, 20), one(30)) is None
    flat_k = torch.cat([kc[3], kc[1]], 1)
    assert torch.equal(flat_k[:, 10:30], k) and (flat_k[:, :10] == 0).all() and (flat_k[:, 30:] == 0).all()
    assert torch.equal(torch.cat([vc[3], vc[1]], 1)[:, 10:30], v) and (both[[0, 2, 4, 5]] == 0).all()


def test_prompt_and_tokens_through_the_whole_step(device):
    """Projection, append with rotation, attention, quantized output projection: a prompt in chunks and then token by
    token gives the rows that causal attention over the whole sequence gives, within both roundings; the step of
    single tokens is captured once and replayed, the lengths moving on the device."""
    hq, hkv, d, hidden, page, n = 8, 2, 128, 512, 16, 75
    g = torch.Generator().manual_seed(0)
    x = torch.randn(2, n, hidden, generator=g).to(BF16).to(device)
    w = (torch.randn((hq + 2 * hkv) * d, hidden, generator=g) / math.sqrt(hidden)).to(BF16).to(device)
    wo = (torch.randn(hidden, hq * d, generator=g) / math.sqrt(hq * d)).to(BF16).to(device)
    wq, ws = m5.quantize(wo, "int8")
    f, _ = m5.rope_frequencies(d, device=device)
    kc, vc = (torch.full((12, hkv, page, d), float("nan"), dtype=BF16, device=device) for _ in range(2))
    table = torch.randperm(12, generator=g)[:10].view(2, 5).to(torch.int32).to(device)

    def step(rows, starts, context):
        y = m5.gemm(rows, w, "bf16", output_dtype=BF16)
        heads = y.view(-1, hq + 2 * hkv, d).transpose(0, 1)
        q = m5.paged_append(heads[hq:hq + hkv], heads[hq + hkv:], kc, vc, table, starts, context, q=heads[:hq],
                            frequencies=f)
        o = m5.paged_attention(q, kc, vc, table, starts, context)
        codes, scales = m5.quantize(o, "int8")
        return o, m5.gemm(codes, wq, "int8", a_scales=scales, b_scales=ws, output_dtype=BF16)

    ints = lambda *v: torch.tensor(v, dtype=torch.int32, device=device)  # noqa: E731
    got = torch.zeros(2, n, hq * d, dtype=BF16, device=device)
    for begin, end in ((0, 33), (33, 64)):
        rows = torch.cat([x[0, begin:end], x[1, begin:end]])
        o, _ = step(rows, ints(0, end - begin, 2 * (end - begin)), ints(end, end))
        got[0, begin:end], got[1, begin:end] = o[:end - begin], o[end - begin:]
    row, starts, context = x[:, 64].clone(), ints(0, 1, 2), ints(65, 65)
    step(row, starts, context)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=torch.cuda.Stream(device=device)):
        o, projected = step(row, starts, context)
    for i in range(64, n):
        row.copy_(x[:, i])
        context.fill_(i + 1)
        graph.replay()
        eager, eager_projected = step(row, starts, context)
        torch.cuda.synchronize()
        assert torch.equal(o, eager) and torch.equal(projected, eager_projected)
        got[:, i] = o
    for b in range(2):
        y = m5.gemm(x[b], w, "bf16", output_dtype=BF16).view(n, -1, d).transpose(0, 1)
        p = torch.arange(n, dtype=torch.int32, device=device)
        want = m5.attention(m5.rope(y[:hq], p, f), m5.rope(y[hq:hq + hkv], p, f), y[hq + hkv:], causal=True)
        # The projection's sums have another order with other row counts: its BF16 outputs differ by a step now and
        # then (2^-7 relative), in q, k and v.  Scores of size |q||k|/sqrt(D) move by 2 * 2^-7 of that at most.
        assert (got[b].double() - want.double()).norm() <= 2.0 ** -6 * want.double().norm()
