"""paged_append into a cache in 8 bits and paged_read, against cache_codes_reference.py: codes and scales are equal, bit
for bit, since a scale is a power of two and keys are turned in 64 bits."""

from __future__ import annotations

import pytest
import torch

import attention_reference as ref
import cache_codes_reference as codes
import m5kernels_amd as m5
from m5kernels_amd import _lib, hip

pytestmark = pytest.mark.gpu

BF16, F16, F32, U8, I8 = torch.bfloat16, torch.float16, torch.float32, torch.uint8, torch.int8


def _randn(seed, *shape, dtype=BF16, spread=0.7):
    g = torch.Generator().manual_seed(seed)
    x = torch.randn(*shape, generator=g)
    return (x * torch.exp2(spread * torch.randn(shape[0], shape[1], 1, generator=g))).to(dtype)


def _ints(*values):
    return torch.tensor(values, dtype=torch.int32)


class Case:
    """A cache, tables and new tokens on the CPU; `new` and `context` a sequence."""

    def __init__(self, new, context, *, hkv=3, d=64, page=32, block=16, mode=U8, dtype=BF16, seed=0):
        self.need = [-(-max(c, 1) // page) for c in context]
        pages = sum(self.need) + 2
        g = torch.Generator().manual_seed(seed)
        order = torch.randperm(pages, generator=g).to(torch.int32)
        self.table = torch.full((len(new), max(self.need) + 1), -1, dtype=torch.int32)
        at = 0
        for b, n in enumerate(self.need):
            self.table[b, :n] = order[at:at + n]
            at += n
        self.starts = torch.tensor([0, *new]).cumsum(0).to(torch.int32)
        self.context = _ints(*context)
        self.k_codes, self.k_scales = codes.held(seed + 1, pages, hkv, page, d, block, mode)
        self.v_codes, self.v_scales = codes.held(seed + 2, pages, hkv, page, d, block, mode)
        t = sum(new)
        self.k, self.v = _randn(seed + 3, hkv, t, d, dtype=dtype), _randn(seed + 4, hkv, t, d, dtype=dtype)

    def cache(self):
        return {n: getattr(self, n) for n in ("k_codes", "v_codes", "k_scales", "v_scales")}

    def tables(self, device):
        return [t.to(device) for t in (self.table, self.starts, self.context)]

    def append(self, device, **options):
        """The call on the device: its result, and the cache behind it."""
        c = {n: t.to(device) for n, t in self.cache().items()}
        out = m5.paged_append(self.k.to(device), self.v.to(device), c["k_codes"], c["v_codes"], *self.tables(device),
                              k_scales=c["k_scales"], v_scales=c["v_scales"], **options)
        return out, c

    def want(self, k=None):
        c = {n: t.clone() for n, t in self.cache().items()}
        codes.append(self.k.double() if k is None else k, c["k_codes"], c["k_scales"], self.table, self.starts,
                     self.context)
        codes.append(self.v.double(), c["v_codes"], c["v_scales"], self.table, self.starts, self.context)
        return c

    def positions(self):
        return torch.cat([torch.arange(int(c) - int(e - s), int(c)) for s, e, c in
                          zip(self.starts[:-1], self.starts[1:], self.context)])


def _same(got, want):
    for name, t in want.items():
        assert torch.equal(got[name].cpu(), t), name


@pytest.mark.parametrize("mode", [U8, I8])
@pytest.mark.parametrize("dtype", [BF16, F16, F32])
@pytest.mark.parametrize("d,page,block", [(64, 16, 16), (64, 48, 48), (64, 64, 64), (64, 128, 128), (128, 16, 16),
                                          (128, 64, 16), (128, 96, 32), (128, 48, 48), (128, 64, 64), (128, 256, 128)])
def test_append(d, page, block, dtype, mode, device):
    """One token, none, chunks that begin and end inside blocks and on their borders, fresh sequences."""
    case = Case([1, 0, 70, 33, 1, 16, 150, 1], [1, 40, 70, 100, 17, 48, 151, 16], d=d, page=page, block=block,
                mode=mode, dtype=dtype)
    out, got = case.append(device)
    assert out is None
    _same(got, case.want())


@pytest.mark.parametrize("mode", [U8, I8])
@pytest.mark.parametrize("layout", ["half", "interleaved"])
@pytest.mark.parametrize("d,pairs,block", [(64, 32, 16), (64, 5, 64), (128, 64, 16), (128, 48, 64), (128, 17, 32),
                                           (128, 64, 128)])
def test_turned_keys(d, pairs, block, layout, mode, device):
    case = Case([1, 37, 0, 160], [300, 37, 5, 1000], d=d, page=128, block=block, mode=mode, seed=3)
    f, _ = m5.rope_frequencies(2 * pairs, device="cpu")
    q = _randn(9, 5, 198, d)
    out, got = case.append(device, q=q.to(device), frequencies=f.to(device), layout=layout, magnitude=1.25)
    positions = case.positions()
    _same(got, case.want(ref.rotate(case.k, positions, f, layout, 1.25)))
    exact = ref.rotate(q, positions, f, layout, 1.25)
    # Two products and a sum in FP32, of a cosine and sine off by a unit, and the rounding to BF16.
    size = 1.25 * (q.double().abs() + 3 * q.double().abs().amax(2, keepdim=True) * 2.0 ** -4)
    assert ((out.cpu().double() - exact).abs() <= exact.abs() * 2.0 ** -8 + size * 2.0 ** -18).all()


def test_far_positions(device):
    """The angle of a position of ten thousand radians and more keeps the keys' codes."""
    case = Case([3, 1], [200003, 77], d=64, page=16, block=16, seed=5)
    f, _ = m5.rope_frequencies(64, device="cpu")
    _, got = case.append(device, frequencies=f.to(device))
    _same(got, case.want(ref.rotate(case.k, case.positions(), f)))


@pytest.mark.parametrize("mode", [U8, I8])
def test_token_by_token(mode, device):
    """A sequence that grows by single tokens of rising size: each raises its block's scale, and the older codes are
    rounded again; what lies behind the context stays."""
    case = Case([1], [40], hkv=2, d=128, page=32, block=32, mode=mode)
    want = {n: t.clone() for n, t in case.cache().items()}
    got = {n: t.to(device) for n, t in case.cache().items()}
    table = case.table.to(device)
    for step in range(40):
        k, v = (_randn(100 * s + step, 2, 1, 128) * 2.0 ** (step // 4 - 3) for s in (1, 2))
        starts, context = _ints(0, 1), _ints(step + 1)
        m5.paged_append(k.to(device), v.to(device), got["k_codes"], got["v_codes"], table, starts.to(device),
                        context.to(device), k_scales=got["k_scales"], v_scales=got["v_scales"])
        codes.append(k.double(), want["k_codes"], want["k_scales"], case.table, starts, context)
        codes.append(v.double(), want["v_codes"], want["v_scales"], case.table, starts, context)
        if step % 7 == 6:
            _same(got, want)
    _same(got, want)


@pytest.mark.parametrize("mode", [U8, I8])
@pytest.mark.parametrize("size", [0.0, 2.0 ** -126, 2.0 ** -140, 2.0 ** 100, 3e38 / 4])
def test_sizes(size, mode, device):
    """All zeros, numbers at both ends of FP32's range, one of them alone in its block."""
    case = Case([30], [41], hkv=2, d=64, page=16, block=16, mode=mode, dtype=F32)
    for x in (case.k, case.v):
        x.clamp_(-4, 4).mul_(size)
    case.k_scales.zero_()
    case.k_codes.zero_()
    _, got = case.append(device)
    _same(got, case.want())


@pytest.mark.parametrize("mode", [U8, I8])
@pytest.mark.parametrize("bad", [float("nan"), float("inf"), -float("inf")])
def test_nonfinite(bad, mode, device):
    """A block that gets a value that is not finite is NaN, and no other; its next tokens do not change that."""
    case = Case([20, 5], [41, 9], hkv=2, d=64, page=16, block=16, mode=mode)
    case.k[1, 4, 7] = bad  # position 25
    case.v[0, 22, 0] = bad
    _, got = case.append(device)
    _same(got, case.want())
    assert (got["k_scales"].cpu() == 255).sum() == 1
    k, v = m5.paged_read(got["k_codes"], got["v_codes"], *case.tables(device), 25, k_scales=got["k_scales"],
                         v_scales=got["v_scales"])
    lost = torch.zeros(2, 25, dtype=torch.bool)
    lost[1, :11] = True  # positions 21 .. 31 of the block 16 .. 31
    assert torch.equal(torch.isnan(k).all(2).cpu(), lost) and torch.equal(torch.isnan(k).any(2).cpu(), lost)
    assert torch.isnan(v[0, 20:]).all() and torch.isfinite(v[1]).all()


def test_what_is_not_stored(device):
    """Negative positions, pages that the cache lacks and tokens behind the table; rows behind the last sequence."""
    case = Case([6, 40, 4, 3], [4, 60, 64, 2], hkv=2, d=64, page=16, block=16)
    case.table[1, 2], case.table[1, 3] = -1, 1000
    case.table = case.table[:, :3].contiguous()  # the third sequence's positions 60 .. 63 lie behind it
    case.k, case.v = (_randn(s, 2, 60, 64) for s in (3, 4))
    q = _randn(8, 2, 60, 64)
    f, _ = m5.rope_frequencies(64, device="cpu")
    out, got = case.append(device, q=q.to(device), frequencies=f.to(device))
    positions = torch.cat([case.positions(), torch.zeros(7, dtype=torch.int64)])
    _same(got, case.want(ref.rotate(case.k, positions, f)))
    assert not out[:, 53:].any() and out[:, :53].abs().sum(2).all()
    k, v = m5.paged_read(got["k_codes"], got["v_codes"], *case.tables(device), 60, k_scales=got["k_scales"],
                         v_scales=got["v_scales"], dtype=F32)
    absent = ((positions < 0) | (positions >= 48)).clone()
    absent[6:46] |= (positions[6:46] >= 32)
    absent[53:] = True
    assert torch.equal((k == 0).all(2).all(0).cpu(), absent) and torch.equal((v == 0).all(2).all(0).cpu(), absent)


@pytest.mark.parametrize("starts,context", [((0, 9, 4, 12), (20, 20, 20)), ((3, 3, 12, 12), (30, 2 ** 31 - 1, 5)),
                                            ((0, -5, 2 ** 31 - 1, 6), (10, -7, 2 ** 31 - 1)),
                                            ((0, 4, 8, 12), (-2 ** 31, 2 ** 30, 4))])
def test_any_starts_and_lengths(starts, context, device):
    """What the device holds is not checked: whatever it is, only pages that the table names are written."""
    case = Case([4, 4, 4], [20, 20, 20], hkv=2, d=64, page=16, block=16)
    case.starts, case.context = _ints(*starts), _ints(*context)
    _, got = case.append(device)
    named = torch.zeros(case.k_codes.shape[0], dtype=torch.bool)
    named[case.table[case.table >= 0].long()] = True
    for name, t in case.cache().items():
        assert torch.equal(got[name].cpu()[~named], t[~named]), name
    k, _ = m5.paged_read(got["k_codes"], got["v_codes"], *case.tables(device), 12, k_scales=got["k_scales"],
                         v_scales=got["v_scales"])
    assert k.shape == (2, 12, 64)


@pytest.mark.parametrize("mode", [U8, I8])
@pytest.mark.parametrize("dtype", [BF16, F16, F32])
@pytest.mark.parametrize("d,page,block", [(64, 16, 16), (64, 96, 48), (128, 64, 64), (128, 256, 128)])
def test_read(d, page, block, dtype, mode, device):
    case = Case([1, 0, 70, 33, 300], [1, 40, 70, 100, 311], d=d, page=page, block=block, mode=mode)
    c = {n: t.to(device) for n, t in case.cache().items()}
    got = m5.paged_read(c["k_codes"], c["v_codes"], *case.tables(device), 410, k_scales=c["k_scales"],
                        v_scales=c["v_scales"], dtype=dtype)
    for x, name in zip(got, "kv"):
        whole = codes.cache(getattr(case, name + "_codes"), getattr(case, name + "_scales"))
        rows = []
        for b, c_b in enumerate(case.context.tolist()):
            every, _ = ref.gather(whole, case.table[b], c_b, page)
            rows.append(every[:, c_b - int(case.starts[b + 1] - case.starts[b]):])
        want = torch.cat([*rows, torch.zeros(3, 6, d)], 1).to(dtype)
        assert x.dtype == dtype and torch.equal(x.cpu(), want)


@pytest.mark.parametrize("mode", [U8, I8])
def test_every_code_and_scale(mode, device):
    """All codes under all exponents, rounded once to each type."""
    every = torch.arange(256).to(U8).view(mode)
    if mode == I8:
        every[every == -128] = 0
    page = every.repeat(16).reshape(1, 1, 64, 64).expand(64, 1, 64, 64).contiguous()
    scales = torch.arange(256).reshape(64, 1, 4).to(U8)
    table = torch.arange(64, dtype=torch.int32).reshape(1, 64)
    want = codes.cache(page, scales).reshape(1, 4096, 64)
    args = [t.to(device) for t in (page, page, table, _ints(0, 4096), _ints(4096))]
    for dtype in (F32, BF16, F16):
        k, v = m5.paged_read(*args, 4096, k_scales=scales.to(device), v_scales=scales.to(device), dtype=dtype)
        assert torch.equal(k.isnan(), v.isnan())
        assert torch.equal(k.cpu().nan_to_num(nan=7.0, posinf=None), want.to(dtype).nan_to_num(nan=7.0, posinf=None))


def test_strided(device):
    """Channels of a wider product, heads and tokens in either order, caches that are views of larger ones."""
    case = Case([1, 37], [19, 50], hkv=4, d=64, page=32, block=16)
    wide = torch.zeros(38, 3, 4, 64, dtype=BF16)
    wide[:, 1], wide[:, 2] = case.k.transpose(0, 1), case.v.transpose(0, 1)
    wide = wide.to(device)
    big = {}
    for n, t in case.cache().items():
        big[n] = torch.full((t.shape[0], 9, *t.shape[2:]), 77, dtype=t.dtype, device=device)
        big[n][:, 2:6] = t.to(device)
    view = {n: t[:, 2:6] for n, t in big.items()}
    m5.paged_append(wide[:, 1].transpose(0, 1), wide[:, 2].transpose(0, 1), view["k_codes"], view["v_codes"],
                    *case.tables(device), k_scales=view["k_scales"], v_scales=view["v_scales"])
    _same(view, case.want())
    assert all((t[:, 6:] == 77).all() and (t[:, :2] == 77).all() for t in big.values())
    odd = torch.zeros(4, 38, 65, dtype=BF16, device=device)[..., 1:]  # rows at no multiple of 16 bytes: copied
    odd.copy_(case.k.to(device))
    fresh = {n: t.to(device) for n, t in case.cache().items()}
    m5.paged_append(odd, case.v.to(device), fresh["k_codes"], fresh["v_codes"], *case.tables(device),
                    k_scales=fresh["k_scales"], v_scales=fresh["v_scales"])
    _same(fresh, case.want())
    with pytest.raises(ValueError, match="multiples of 16"):
        shifted = torch.zeros(case.k_codes.numel() + 8, dtype=U8, device=device)[8:].view(case.k_codes.shape)
        m5.paged_append(case.k.to(device), case.v.to(device), shifted, fresh["v_codes"], *case.tables(device),
                        k_scales=fresh["k_scales"], v_scales=fresh["v_scales"])
    with pytest.raises(ValueError, match="expanded"):
        m5.paged_append(case.k.to(device), case.v.to(device), fresh["k_codes"], fresh["v_codes"], *case.tables(device),
                        k_scales=fresh["k_scales"], v_scales=fresh["v_scales"][:1].expand_as(fresh["v_scales"]))


def test_codes_behind_32_bits(device):
    """A cache of more than 2^32 bytes: its last page is written and read."""
    pages, hkv, page, d = 33000, 16, 64, 128
    c = torch.zeros(pages, hkv, page, d, dtype=U8, device=device)
    scales = torch.zeros(pages, hkv, 1, dtype=U8, device=device)
    k = _randn(0, hkv, 70, d).to(device)
    table = torch.tensor([[pages - 1, 0]], dtype=torch.int32, device=device)
    args = (table, _ints(0, 70).to(device), _ints(70).to(device))
    v_scales = scales.clone()
    m5.paged_append(k, k, c, c.clone(), *args, k_scales=scales, v_scales=v_scales)
    want = torch.zeros(2, hkv, page, d, dtype=U8), torch.zeros(2, hkv, 1, dtype=U8)
    codes.append(k.cpu().double(), *want, torch.tensor([[1, 0]]), [0, 70], [70])
    assert torch.equal(c[[0, -1]].cpu(), want[0]) and torch.equal(scales[[0, -1]].cpu(), want[1])
    got, _ = m5.paged_read(c, c, *args, 70, k_scales=scales, v_scales=scales, dtype=F32)
    assert torch.equal(got.cpu().double()[:, :64], codes.cache(*want)[1])


@pytest.mark.parametrize("rotated", [False, True])
def test_both_fronts(rotated, device, monkeypatch):
    """The native front takes plain calls and gives the Python front's bits."""
    front = _lib.load_fast()
    if front is None:
        pytest.skip("the native front is not built")
    case = Case([1, 30], [20, 41], d=128, page=32, block=16)
    f = m5.rope_frequencies(128, device=device)[0] if rotated else None
    q = _randn(8, 6, 31, 128).to(device) if rotated else None
    sides = []
    for native in (True, False):
        c = {n: t.to(device) for n, t in case.cache().items()}
        call = (case.k.to(device), case.v.to(device), c["k_codes"], c["v_codes"], *case.tables(device))
        read = (c["k_codes"], c["v_codes"], *case.tables(device), 31)
        if native:
            out = front.paged_append(*call, q, f, "half", 1.0, c["k_scales"], c["v_scales"])
            assert out is not None and (out is True) != rotated
            back = front.paged_read(*read, c["k_scales"], c["v_scales"], F16)
        else:
            monkeypatch.setattr(hip, "_fast", None)
            out = m5.paged_append(*call, q=q, frequencies=f, k_scales=c["k_scales"], v_scales=c["v_scales"])
            back = m5.paged_read(*read, k_scales=c["k_scales"], v_scales=c["v_scales"], dtype=F16)
        sides.append([*c.values(), *back, *([out] if rotated else [])])
    for a, b in zip(*sides):
        assert a.dtype == b.dtype and torch.equal(a, b)


def test_no_tokens(device):
    case = Case([0], [5], d=64, page=16, block=16)
    out, got = case.append(device)
    assert out is None
    _same(got, case.cache())
    k, v = m5.paged_read(got["k_codes"], got["v_codes"], *case.tables(device), 0, k_scales=got["k_scales"],
                         v_scales=got["v_scales"])
    assert k.shape == v.shape == (3, 0, 64)


def test_streams_and_graphs(device):
    """On a stream of its own, and captured: each replay takes what the buffers hold then."""
    case = Case([1, 1], [20, 33], hkv=2, d=128, page=32, block=32)
    c = {n: t.to(device) for n, t in case.cache().items()}
    k, v = case.k.to(device), case.v.to(device)
    table, starts, context = case.tables(device)

    def call():
        m5.paged_append(k, v, c["k_codes"], c["v_codes"], table, starts, context, k_scales=c["k_scales"],
                        v_scales=c["v_scales"])
        return m5.paged_read(c["k_codes"], c["v_codes"], table, starts, context, 2, k_scales=c["k_scales"],
                             v_scales=c["v_scales"])

    stream = torch.cuda.Stream()
    stream.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(stream):
        call()
    torch.cuda.current_stream().wait_stream(stream)
    _same(c, case.want())
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = call()
    want = case.want()
    for step in range(4):
        new_k, new_v = (_randn(50 + 2 * step + s, 2, 2, 128) for s in (0, 1))
        k.copy_(new_k)
        v.copy_(new_v)
        context += 1
        case.context += 1
        graph.replay()
        torch.cuda.synchronize()
        codes.append(new_k.double(), want["k_codes"], want["k_scales"], case.table, case.starts, case.context)
        codes.append(new_v.double(), want["v_codes"], want["v_scales"], case.table, case.starts, case.context)
        _same(c, want)
        again = m5.paged_read(c["k_codes"], c["v_codes"], table, starts, context, 2, k_scales=c["k_scales"],
                              v_scales=c["v_scales"])
        assert torch.equal(again[0], out[0]) and torch.equal(again[1], out[1])
