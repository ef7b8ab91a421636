"""Cases of the attention step behind the Q/K/V projection: rotary positions, the paged cache that keys
and values are appended to, attention of new tokens over that cache, and attention without one.

Heads are 128 or 64 wide and come head-major, [heads, tokens, width], as the projections give them;
attention returns [tokens, heads * width], which the output projection takes.  The transformer is the
harness's (56 heads of 128, 96 rotated channels, 128 to 9914 tokens); shared heads, cache lengths and
pages are those that a server meets.

``own`` chooses between the package's operators and their plain form; ``listed`` names the cases, ``draw``
gives others of the same ranges, ``prepare`` makes what a program holds before the call, ``run`` is one
pass, ``work`` the bytes and operations that a pass cannot do without, ``exact`` the same in 64 bits.
"""

from __future__ import annotations

import math
import sys
from pathlib import Path

import torch

own = False

_DTYPES = {"bf16": torch.bfloat16, "fp16": torch.float16, "fp32": torch.float32}
_MAX_BYTES = 2.5e9  # a cache's keys and values that one pass reads
_MAX_SCORES = 56 * 9914 * 9914  # (head, row, key) triples, as in the largest listed case


def listed():
    return [
        # One decoded token at a far position of a context stretched 16 times: a launch and its host work.
        dict(name="rope_m1_far", kind="rope", m=1, heads=56, d=128, rotary=96, layout="half", scaling="yarn",
             factor=16.0, first=400000, dtype="bf16"),
        # Every head of a long video prompt, pairs of neighbouring channels.
        dict(name="rope_m9914_interleaved", kind="rope", m=9914, heads=56, d=128, rotary=128, layout="interleaved",
             scaling="none", factor=1.0, first=0, dtype="bf16"),
        # One token of each of 64 running sequences, its query rotated in the same call; short pages.
        dict(name="append_decode_b64", kind="append", hq=56, hkv=8, d=128, rotary=128, layout="half", dtype="bf16",
             page=16, new=_text([1] * 64), context=_text(65 + 61 * b for b in range(64))),
        # Chunks of four prompts, one of them a single odd token, of a model with half-width heads.
        dict(name="append_chunks_b4", kind="append", hq=32, hkv=32, d=64, rotary=32, layout="interleaved",
             dtype="fp16", page=64, new="2048 1 511 1536", context="2048 777 4607 1536"),
        # One token of one sequence whose cache is long: the only parallelism is along the keys.
        dict(name="paged_decode_long", kind="paged", hq=64, hkv=8, d=128, dtype="bf16", page=64, new="1",
             context="131073", window=0, softcap=0.0, slopes=False, prefix=False),
        # A serving step of 64 sequences of all lengths, seven query heads to a key head, one slot idle.
        dict(name="paged_decode_b64", kind="paged", hq=56, hkv=8, d=128, dtype="bf16", page=16, new=_text([1] * 64),
             context=_text((b * 2741) % 8191 for b in range(64)), window=0, softcap=0.0, slopes=False, prefix=False),
        # Chunked prefill beside running sequences.
        dict(name="paged_chunk_mixed", kind="paged", hq=32, hkv=8, d=128, dtype="bf16", page=64,
             new="1024 1 1 512 1 333 1 1", context="8192 4097 517 512 2050 3333 6001 63", window=0,
             softcap=0.0, slopes=False, prefix=False),
        # Capped scores over a sliding window, half-width heads, pages of no power of two.
        dict(name="paged_window_softcap", kind="paged", hq=16, hkv=16, d=64, dtype="fp16", page=24,
             new="700 129 1", context="2500 129 4000", window=1024, softcap=50.0, slopes=False, prefix=False),
        # The harness's shortest attention.
        dict(name="attention_m128_h56", kind="attention", hq=56, hkv=56, d=128, dtype="bf16", lengths="128",
             causal=False, window=0, softcap=0.0, slopes=False, prefix=False),
        # Its longest, a long video prompt that sees all of itself: the largest case.
        dict(name="attention_m9914_h56", kind="attention", hq=56, hkv=56, d=128, dtype="bf16", lengths="9914",
             causal=False, window=0, softcap=0.0, slopes=False, prefix=False),
        # Documents of all lengths packed in one row, causal, with a bias that grows with the distance.
        dict(name="attention_documents_bias", kind="attention", hq=32, hkv=8, d=128, dtype="bf16",
             lengths="4096 17 1500 1 2048 0 530", causal=True, window=0, softcap=0.0, slopes=True,
             prefix=False),
        # A prefix that every token sees, capped scores, half-width heads, an odd length.
        dict(name="attention_prefix_softcap", kind="attention", hq=16, hkv=4, d=64, dtype="fp16", lengths="1999",
             causal=True, window=0, softcap=30.0, slopes=False, prefix=True),
    ]


def _text(numbers):
    return " ".join(str(n) for n in numbers)


def _numbers(case, field):
    return [int(n) for n in case[field].split()]


def _log_int(rng, lo, hi):
    return max(lo, min(hi, round(math.exp(rng.uniform(math.log(lo), math.log(hi))))))


def draw(rng):
    kind = rng.choice(["rope", "append", "paged", "paged", "paged", "attention", "attention", "attention"])
    d = rng.choice([64, 128, 128])
    dtype = rng.choice(["bf16", "bf16", "fp16"])
    hkv = _log_int(rng, 1, 56)
    hq = hkv * rng.choice([g for g in (1, 1, 2, 3, 4, 7, 8, 16) if g * hkv <= 64])
    layout = rng.choice(["half", "interleaved"])
    rotary = rng.choice([d, d, d // 2, 3 * d // 4, d // 4 + 2])
    if kind == "rope":
        scaling = rng.choice(["none", "linear", "ntk", "yarn"])
        return dict(kind=kind, m=_log_int(rng, 1, 9914), heads=rng.randint(1, 56), d=d, rotary=rotary, layout=layout,
                    scaling=scaling, factor=1.0 if scaling == "none" else rng.choice([2.0, 8.0, 32.0]),
                    first=rng.choice([0, 0, _log_int(rng, 1, 1000000)]), dtype=rng.choice([dtype, dtype, "fp32"]))
    if kind == "attention":
        lengths = [_log_int(rng, 1, 9914)]
        if rng.random() < 0.5:
            lengths = [rng.choice([0, 1, _log_int(rng, 2, 4096)]) for _ in range(rng.randint(2, 9))]
            lengths.append(rng.randint(1, 99))
        causal = rng.random() < 0.6
        prefix = causal and rng.random() < 0.25
        m = sum(lengths)
        while hq * m * m > _MAX_SCORES:
            lengths = [n // 2 for n in lengths[:-1]] + [lengths[-1] // 2 + 1]
            m = sum(lengths)
        return dict(kind=kind, hq=hq, hkv=hkv, d=d, dtype=dtype, lengths=_text(lengths), causal=causal,
                    window=_log_int(rng, 1, 2048) if not prefix and rng.random() < 0.25 else 0,
                    softcap=rng.choice([0.0, 0.0, 0.0, 20.0, 50.0]), slopes=rng.random() < 0.25, prefix=prefix)
    page = rng.choice([16, 16, 32, 64, 128, 24, 7])
    b = _log_int(rng, 1, 64)
    decode = rng.random() < 0.5
    new = [1 if decode or rng.random() < 0.4 else _log_int(rng, 1, 1500) for _ in range(b)]
    if kind == "append":
        return dict(kind=kind, hq=hq, hkv=hkv, d=d, rotary=rotary, layout=layout, dtype=dtype, page=page,
                    new=_text(new), context=_text(n + rng.choice([0, _log_int(rng, 1, 1000)]) for n in new))
    longest = _log_int(rng, 64, 131072)
    context = [n + _log_int(rng, 1, longest) for n in new]
    while (sum(context) * hkv * d * 4 > _MAX_BYTES or b * max(context) * hkv * d * 4 > 4 * _MAX_BYTES
           or b * max(new) * max(context) * hq > _MAX_SCORES):
        new = [(n + 1) // 2 for n in new]
        context = [max(n, c // 2) for n, c in zip(new, context)]
    prefix = rng.random() < 0.15
    return dict(kind=kind, hq=hq, hkv=hkv, d=d, dtype=dtype, page=page, new=_text(new), context=_text(context),
                window=_log_int(rng, 1, 4096) if not prefix and rng.random() < 0.25 else 0,
                softcap=rng.choice([0.0, 0.0, 0.0, 20.0, 50.0]), slopes=rng.random() < 0.25, prefix=prefix)


# ---- inputs ---------------------------------------------------------------------------------


def _frequencies(case):
    """Radians a position of each rotated pair, in 64 bits, and the factor on cosine and sine."""
    r = case["rotary"]
    pairs = torch.arange(0, r, 2, dtype=torch.float64)
    scaling, factor = case.get("scaling", "none"), case.get("factor", 1.0)
    base = 10000.0
    if scaling == "ntk" and r > 2:
        base *= factor ** (r / (r - 2))
    f = base ** (-pairs / r)
    if scaling == "linear":
        return f / factor, 1.0
    if scaling == "yarn":
        keep = ((4096 * f / (2 * math.pi) - 1.0) / (32.0 - 1.0)).clamp(0.0, 1.0)
        return (1.0 - keep) * f / factor + keep * f, 0.1 * math.log(factor) + 1.0
    return f, 1.0


def _starts(lengths):
    return torch.tensor([0] + lengths, dtype=torch.int64).cumsum(0).to(torch.int32).cuda()


def _pages(g, case):
    """A page table over pages in random order, and how many there are (some that no sequence owns)."""
    width = max(1, -(-max(_numbers(case, "context")) // case["page"]))
    need = [-(-c // case["page"]) for c in _numbers(case, "context")]
    count = sum(need) + 3
    order = torch.randperm(count, generator=g, device="cuda").to(torch.int32)
    table = torch.zeros(len(need), width, dtype=torch.int32, device="cuda")
    at = 0
    for b, n in enumerate(need):
        table[b, :n] = order[at:at + n]
        at += n
    return table, count


def prepare(case, seed):
    """Inputs on the GPU from the seed alone: normalized queries and keys, a cache that is full up to
    the context (behind it, what a page held before)."""
    g = torch.Generator(device="cuda").manual_seed(int(seed))
    dtype, d, kind = _DTYPES[case["dtype"]], case["d"], case["kind"]

    def randn(*shape):
        return torch.randn(*shape, generator=g, device="cuda", dtype=torch.float32).to(dtype)

    s = {"case": dict(case)}
    if kind in ("rope", "append"):
        f, s["magnitude"] = _frequencies(case)
        s["frequencies"] = f.cuda()
    if kind == "rope":
        s["x"] = randn(case["heads"], case["m"], d)
        s["positions"] = torch.arange(case["first"], case["first"] + case["m"], dtype=torch.int32, device="cuda")
        return s
    hq, hkv = case["hq"], case["hkv"]
    if case.get("slopes"):
        s["slopes"] = torch.exp2(-8.0 * torch.arange(1, hq + 1, device="cuda", dtype=torch.float32) / hq)
    if kind == "attention":
        m = sum(_numbers(case, "lengths"))
        s["q"], s["k"], s["v"] = randn(hq, m, d), randn(hkv, m, d), randn(hkv, m, d)
        if len(_numbers(case, "lengths")) > 1:
            s["starts"] = _starts(_numbers(case, "lengths"))
        if case["prefix"]:
            s["prefix"] = torch.tensor(_prefixes(_numbers(case, "lengths")), dtype=torch.int32, device="cuda")
        return s
    t = sum(_numbers(case, "new"))
    s["table"], count = _pages(g, case)
    s["starts"] = _starts(_numbers(case, "new"))
    s["context"] = torch.tensor(_numbers(case, "context"), dtype=torch.int32, device="cuda")
    s["q"] = randn(hq, t, d)
    s["k_cache"], s["v_cache"] = randn(count, hkv, case["page"], d), randn(count, hkv, case["page"], d)
    if kind == "append":
        s["k"], s["v"] = randn(hkv, t, d), randn(hkv, t, d)
    elif case["prefix"]:
        s["prefix"] = torch.tensor(_prefixes(_numbers(case, "context")), dtype=torch.int32, device="cuda")
    return s


def _prefixes(lengths):
    """A prompt of about a third of each sequence that all of its tokens see."""
    return [n // 3 + n % 5 for n in lengths]


# ---- one pass --------------------------------------------------------------------------------


def run(s):
    return _OWN[s["case"]["kind"]](s, s["case"]) if own else _PLAIN[s["case"]["kind"]](s, s["case"])


def _package():
    path = str(Path(__file__).resolve().parent.parent / "m5-max-kernels_amd")
    if path not in sys.path:
        sys.path.insert(0, path)
    import m5kernels_amd

    return m5kernels_amd


def _own_rope(s, c):
    return _package().rope(s["x"], s["positions"], s["frequencies"], layout=c["layout"], magnitude=s["magnitude"])


def _own_append(s, c):
    q = _package().paged_append(
        s["k"], s["v"], s["k_cache"], s["v_cache"], s["table"], s["starts"], s["context"], q=s["q"],
        frequencies=s["frequencies"], layout=c["layout"], magnitude=s["magnitude"])
    return {"q": q, "k_cache": s["k_cache"], "v_cache": s["v_cache"]}


def _own_paged(s, c):
    return _package().paged_attention(
        s["q"], s["k_cache"], s["v_cache"], s["table"], s["starts"], s["context"], window=c["window"] or None,
        softcap=c["softcap"] or None, slopes=s.get("slopes"), prefix_lengths=s.get("prefix"))


def _own_attention(s, c):
    return _package().attention(
        s["q"], s["k"], s["v"], causal=c["causal"], window=c["window"] or None, document_starts=s.get("starts"),
        prefix_lengths=s.get("prefix"), softcap=c["softcap"] or None, slopes=s.get("slopes"))


_OWN = {"rope": _own_rope, "append": _own_append, "paged": _own_paged, "attention": _own_attention}


# ---- the plain form ---------------------------------------------------------------------------


def _rotated(x, positions, s, layout):
    """x [heads, M, D] in 32 bits; the angles of far positions need 64."""
    angle = positions.double()[:, None] * s["frequencies"][None, :]
    c, n = (angle.cos() * s["magnitude"]).float(), (angle.sin() * s["magnitude"]).float()
    x = x.float()
    r = c.shape[1]
    if layout == "half":
        a, b = x[..., :r], x[..., r:2 * r]
        y = torch.cat([a * c - b * n, b * c + a * n], -1)
    else:
        a, b = x[..., 0:2 * r:2], x[..., 1:2 * r:2]
        y = torch.stack([a * c - b * n, b * c + a * n], -1).flatten(-2)
    return torch.cat([y, x[..., 2 * r:]], -1)


def _plain_rope(s, c):
    return _rotated(s["x"], s["positions"], s, c["layout"]).to(s["x"].dtype)


def _places(s, tokens):
    """Of every token: its sequence, its index among that sequence's new tokens, its position."""
    starts = s["starts"].long()
    token = torch.arange(tokens, device="cuda")
    seq = torch.searchsorted(starts[1:], token, right=True)
    index = token - starts[seq]
    new = starts[seq + 1] - starts[seq]
    return seq, index, s["context"].long()[seq] - new + index


def _plain_append(s, c):
    seq, _, position = _places(s, s["k"].shape[1])
    page, slot = s["table"].long()[seq, position // c["page"]], position % c["page"]
    dtype = s["k"].dtype
    s["k_cache"][page, :, slot] = _rotated(s["k"], position, s, c["layout"]).to(dtype).transpose(0, 1)
    s["v_cache"][page, :, slot] = s["v"].transpose(0, 1)
    q = _rotated(s["q"], position, s, c["layout"]).to(dtype)
    return {"q": q, "k_cache": s["k_cache"], "v_cache": s["v_cache"]}


def _softmax_product(score, visible, v):
    """softmax over the visible keys times v, and 0 where none is visible."""
    score.masked_fill_(~visible, -math.inf)
    top = score.amax(-1, keepdim=True)
    p = score.sub_(top.masked_fill(top == -math.inf, 0.0)).exp_()
    total = p.sum(-1, keepdim=True)
    return torch.matmul(p, v) / total.masked_fill(total == 0, 1.0)


def _plain_paged(s, c):
    hq, hkv, d = c["hq"], c["hkv"], c["d"]
    b, most, scale = len(_numbers(c, "new")), max(_numbers(c, "new")), 1.0 / math.sqrt(d)
    seq, index, _ = _places(s, s["q"].shape[1])
    q = torch.zeros(b, hq, most, d, device="cuda")
    q[seq, :, index] = s["q"].float().transpose(0, 1)

    def gathered(cache):
        return cache[s["table"].long()].permute(0, 2, 1, 3, 4).reshape(b, hkv, -1, d).float()

    k = gathered(s["k_cache"]).transpose(2, 3).contiguous()
    keys = k.shape[3]
    score = torch.matmul(q.reshape(b, hkv, -1, d), k).mul_(scale).reshape(b, hq, most, keys)
    del k
    context, new = s["context"].long()[:, None, None], (s["starts"][1:] - s["starts"][:-1]).long()[:, None, None]
    position = context - new + torch.arange(most, device="cuda")[None, :, None]
    key = torch.arange(keys, device="cuda")[None, None, :]
    reach = position + 1
    if "prefix" in s:
        reach = torch.maximum(reach, s["prefix"].long()[:, None, None])
    visible = (key < reach) & (key < context)
    if c["window"]:
        visible &= position - key < c["window"]
    if c["softcap"]:
        score.div_(c["softcap"]).tanh_().mul_(c["softcap"])
    if "slopes" in s:
        score -= s["slopes"][None, :, None, None] * (position - key).abs().float()[:, None]
    visible = visible[:, None].expand(b, hq, most, keys).reshape(b, hkv, -1, keys)
    o = _softmax_product(score.reshape(b, hkv, -1, keys), visible, gathered(s["v_cache"])).reshape(b, hq, most, d)
    return o[seq, :, index].reshape(-1, hq * d).to(s["q"].dtype)


def _plain_attention(s, c):
    hq, hkv, d = c["hq"], c["hkv"], c["d"]
    m, group, scale = s["q"].shape[1], hq // hkv, 1.0 / math.sqrt(d)
    token = torch.arange(m, device="cuda")
    score = torch.matmul(s["q"].float().reshape(hkv, group * m, d), s["k"].float().transpose(1, 2).contiguous())
    score = score.mul_(scale).reshape(hkv, group, m, m)
    row, key = token[:, None], token[None, :]
    if "starts" in s:
        starts = s["starts"].long()
        document = torch.searchsorted(starts[1:], token, right=True)
        visible, first = document[:, None] == document[None, :], starts[document][:, None]
    else:
        document, first = torch.zeros_like(token), torch.zeros_like(row)
        visible = torch.ones(m, m, dtype=torch.bool, device="cuda")
    if c["causal"]:
        before = key <= row
        if "prefix" in s:
            before |= key - first < s["prefix"].long()[document][:, None]
        visible &= before
    if c["window"]:
        visible &= (row - key).abs() < c["window"]
    if c["softcap"]:
        score.div_(c["softcap"]).tanh_().mul_(c["softcap"])
    if "slopes" in s:
        score -= s["slopes"].reshape(hkv, group, 1, 1) * (row - key).abs().float()
    o = _softmax_product(score, visible, s["v"].float()[:, None].expand(hkv, group, m, d))
    return o.reshape(hq, m, d).transpose(0, 1).reshape(m, hq * d).to(s["q"].dtype)


_PLAIN = {"rope": _plain_rope, "append": _plain_append, "paged": _plain_paged, "attention": _plain_attention}


# ---- what a pass cannot do without --------------------------------------------------------------


def _pairs(first, count, keys, causal, window, prefix):
    """Visible (row, key) pairs of `count` rows at positions first.. over `keys` keys."""
    p = torch.arange(first, first + count, dtype=torch.int64)
    hi = torch.clamp(torch.maximum(p + 1, torch.tensor(prefix)), max=keys) if causal else torch.full_like(p, keys)
    lo = torch.zeros_like(p)
    if window:
        lo = torch.clamp(p - window + 1, min=0)
        hi = torch.minimum(hi, p + window)
    return int((hi - lo).clamp(min=0).sum())


def work(case):
    kind, d, size = case["kind"], case["d"], 4 if case["dtype"] == "fp32" else 2
    if kind == "rope":
        values = case["heads"] * case["m"]
        return {"bytes": 2.0 * values * d * size + 4 * case["m"] + 4 * case["rotary"],
                "flops": 3.0 * values * case["rotary"]}
    hq, hkv = case["hq"], case["hkv"]
    if kind == "append":
        t = sum(_numbers(case, "new"))
        return {"bytes": 2.0 * t * (hq + 2 * hkv) * d * size + 8 * len(_numbers(case, "new")) + 4 * t,
                "flops": 3.0 * t * (hq + hkv) * case["rotary"]}
    if kind == "paged":
        prefixes = _prefixes(_numbers(case, "context")) if case["prefix"] else [0] * len(_numbers(case, "new"))
        pairs = keys = 0
        for n, c, f in zip(_numbers(case, "new"), _numbers(case, "context"), prefixes):
            if c >= n:
                pairs += _pairs(c - n, n, c, True, case["window"], f)
                keys += min(c, n + case["window"] - 1) if case["window"] else c
        rows = sum(_numbers(case, "new"))
    else:
        prefixes = _prefixes(_numbers(case, "lengths")) if case["prefix"] else [0] * len(_numbers(case, "lengths"))
        lengths = _numbers(case, "lengths")
        pairs = sum(_pairs(0, n, n, case["causal"], case["window"], f) for n, f in zip(lengths, prefixes))
        rows = keys = sum(lengths)
    return {"bytes": 2.0 * (keys * hkv + rows * hq) * d * size, "flops": 4.0 * d * hq * pairs}


# ---- the same in 64 bits --------------------------------------------------------------------------


def _rotated64(x, positions, case):
    f, magnitude = _frequencies(case)
    angle = torch.outer(positions.double(), f.cuda())
    turn = torch.polar(torch.full_like(angle, magnitude), angle)
    r, x = case["rotary"], x.double()
    head = x[..., :r]
    z = torch.complex(*head.chunk(2, -1)) if case["layout"] == "half" else torch.view_as_complex(
        head.reshape(*head.shape[:-1], r // 2, 2).contiguous())
    z = z * turn
    y = torch.cat([z.real, z.imag], -1) if case["layout"] == "half" else torch.view_as_real(z).flatten(-2)
    return torch.cat([y, x[..., r:]], -1)


def _attend64(q, k, v, first, case, prefix, slopes):
    """q [rows, D] of one head at positions first.., k and v [keys, D]."""
    rows, keys = q.shape[0], k.shape[0]
    if rows == 0 or keys == 0:
        return torch.zeros_like(q)
    score = (q @ k.T) / math.sqrt(q.shape[1])
    if case["softcap"]:
        score = case["softcap"] * torch.tanh(score / case["softcap"])
    apart = (first + torch.arange(rows, device="cuda"))[:, None] - torch.arange(keys, device="cuda")[None, :]
    if slopes is not None:
        score = score - slopes * apart.abs()
    hidden = torch.zeros(rows, keys, dtype=torch.bool, device="cuda")
    if case.get("causal", True):
        hidden |= (apart < 0) & (torch.arange(keys, device="cuda")[None, :] >= prefix)
    if case["window"]:
        hidden |= apart.abs() >= case["window"]
    score = score.masked_fill(hidden, -math.inf)
    return torch.nan_to_num(torch.softmax(score, -1), nan=0.0) @ v


def exact(case, seed):
    s = prepare(case, seed)
    kind = case["kind"]
    if kind == "rope":
        return _rotated64(s["x"], s["positions"], case)
    hq, hkv = case["hq"], case["hkv"]
    group = hq // hkv
    slopes = [float(x) for x in s["slopes"].cpu().double()] if "slopes" in s else [None] * hq
    if kind == "attention":
        q, k, v = s["q"].double(), s["k"].double(), s["v"].double()
        out = torch.zeros(q.shape[1], hq, case["d"], dtype=torch.float64, device="cuda")
        prefixes = _prefixes(_numbers(case, "lengths")) if case["prefix"] else [0] * len(_numbers(case, "lengths"))
        at = 0
        for n, prefix in zip(_numbers(case, "lengths"), prefixes):
            for h in range(hq):
                out[at:at + n, h] = _attend64(q[h, at:at + n], k[h // group, at:at + n], v[h // group, at:at + n], 0,
                                              case, prefix, slopes[h])
            at += n
        return out.reshape(q.shape[1], -1)
    page, at = case["page"], 0
    if kind == "append":
        spans = zip(_numbers(case, "new"), _numbers(case, "context"))
        position = torch.cat([torch.arange(c - n, c) for n, c in spans]).cuda()
        k, k_cache, v_cache = _rotated64(s["k"], position, case), s["k_cache"].double(), s["v_cache"].double()
        for b, n in enumerate(_numbers(case, "new")):
            p = position[at:at + n]
            where = s["table"][b].long()[p // page]
            for h in range(hkv):
                k_cache[where, h, p % page] = k[h, at:at + n]
                v_cache[where, h, p % page] = s["v"][h, at:at + n].double()
            at += n
        return {"q": _rotated64(s["q"], position, case), "k_cache": k_cache, "v_cache": v_cache}
    out = torch.zeros(s["q"].shape[1], hq, case["d"], dtype=torch.float64, device="cuda")
    prefixes = _prefixes(_numbers(case, "context")) if case["prefix"] else [0] * len(_numbers(case, "new"))
    for b, (n, c) in enumerate(zip(_numbers(case, "new"), _numbers(case, "context"))):
        where = s["table"][b, :-(-c // page)].long()
        for h in range(hkv if c >= n else 0):
            k, v = (t[where, h].reshape(-1, case["d"])[:c].double() for t in (s["k_cache"], s["v_cache"]))
            for j in range(h * group, (h + 1) * group):
                out[at:at + n, j] = _attend64(s["q"][j, at:at + n].double(), k, v, c - n, case, prefixes[b], slopes[j])
        at += n
    return out.reshape(s["q"].shape[1], -1)
