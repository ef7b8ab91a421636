"""Cases of the attention step over a cache held in 8 bits, and of attention with a sliding window and a few
first tokens that stay visible.

The cache holds E4M3 or INT8 codes and, for each block of tokens and key head, the exponent of a power-of-two scale.
``append`` writes new keys and values into it (turned to their positions where the case says so) and reads
the blocks that it touched back; ``read`` reads long stretches back; ``paged`` is attention of new tokens over a cache,
in 8 or 16 bits; ``attention`` is attention without one.  The transformer is the harness's (56 heads of 128, 128 to 9914
tokens) and that of the cases beside this file; cache lengths, pages and windows are those that a server meets.

``own`` chooses between the package's operators and their plain form; ``listed`` names the cases, ``draw``
gives others of the same ranges, ``prepare`` makes what a program holds before the call, ``run`` is one
pass, ``work`` the bytes and operations that a pass cannot do without, ``exact`` the same in 64 bits.
"""

from __future__ import annotations

import functools
import math
import sys
from pathlib import Path

import torch

own = False

_DTYPES = {"bf16": torch.bfloat16, "fp16": torch.float16, "fp32": torch.float32}
_LARGEST = {"fp8": 448.0, "int8": 127.0}  # of a code's magnitude
# What a drawn case may take, so that it costs no more than the largest listed one.
_MAX_BYTES = 1.2e9  # a cache's keys and values that one pass reads, in 16 bits
_MAX_VALUES = 1.2e8  # keys and values that one pass appends, or reads back
_MAX_FLOPS = 2.7e11
_MAX_SCORES = 56 * 9914 * 9914  # (head, row, key) triples that the plain form holds


def listed():
    return [
        # One token of each of 64 running sequences goes into blocks that are partly full; its query is turned in
        # the same call.
        dict(name="append8_decode_b64", kind="append", hq=56, hkv=8, d=128, rotary=128, layout="half", dtype="bf16",
             codes="fp8", page=16, block=16, new=_text([1] * 64), context=_text(65 + 61 * b for b in range(64))),
        # Chunks of four prompts, one of them a single odd token, keys turned already (by the projection).
        dict(name="append8_chunks_b4", kind="append", hq=0, hkv=32, d=64, rotary=0, layout="half", dtype="fp16",
             codes="int8", page=64, block=64, new="2048 1 511 1536", context="2048 777 4607 1536"),
        # A long prompt's cache handed on to a machine that keeps 16 bits.
        dict(name="read8_long", kind="read", hkv=8, d=128, dtype="bf16", codes="fp8", page=64, block=64,
             new="32769", context="32769"),
        # Parts of running sequences, half-width heads, several blocks to a page.
        dict(name="read8_ragged_b33", kind="read", hkv=16, d=64, dtype="fp16", codes="int8", page=48, block=16,
             new=_text(1 + 37 * b for b in range(33)), context=_text(1 + 37 * b + 11 * (b % 3) for b in range(33))),
        # One decoded token of a short conversation: a launch and its host work.
        dict(name="paged8_decode_single", kind="paged", hq=56, hkv=8, d=128, dtype="bf16", codes="fp8", page=64,
             block=64, new="1", context="301", window=0, sinks=0, softcap=0.0, slopes=False, prefix=False),
        # One token of one sequence whose cache is long: the only parallelism is along the keys.
        dict(name="paged8_decode_long", kind="paged", hq=64, hkv=8, d=128, dtype="bf16", codes="fp8", page=64,
             block=64, new="1", context="131073", window=0, sinks=0, softcap=0.0, slopes=False, prefix=False),
        # A serving step of 64 sequences of all lengths, seven query heads to a key head, one slot idle.
        dict(name="paged8_decode_b64", kind="paged", hq=56, hkv=8, d=128, dtype="bf16", codes="int8", page=16,
             block=16, new=_text([1] * 64), context=_text((b * 2741) % 8191 for b in range(64)), window=0, sinks=0,
             softcap=0.0, slopes=False, prefix=False),
        # Chunked prefill beside running sequences.
        dict(name="paged8_chunk_mixed", kind="paged", hq=32, hkv=8, d=128, dtype="bf16", codes="fp8", page=64,
             block=64, new="1024 1 1 512 1 333 1 1", context="8192 4097 517 512 2050 3333 6001 63", window=0, sinks=0,
             softcap=0.0, slopes=False, prefix=False),
        # Sequences that have outgrown their window, in 8 bits, half-width heads, capped scores.
        dict(name="paged8_sinks_softcap", kind="paged", hq=16, hkv=16, d=64, dtype="fp16", codes="int8", page=48,
             block=16, new="700 129 1 33", context="2500 129 4000 20011", window=1024, sinks=4, softcap=50.0,
             slopes=False, prefix=False),
        # Running sequences far behind their window, each with the first tokens it keeps, in 16 bits.
        dict(name="paged_sinks_decode_b32", kind="paged", hq=56, hkv=8, d=128, dtype="bf16", codes="none", page=16,
             block=0, new=_text([1] * 32), context=_text(100 + 997 * b for b in range(32)), window=4096, sinks=4,
             softcap=0.0, slopes=False, prefix=False),
        # A long prompt over a window and its first tokens: the largest case.
        dict(name="attention_sinks_m9914_h56", kind="attention", hq=56, hkv=56, d=128, dtype="bf16", lengths="9914",
             causal=True, window=1024, sinks=4, softcap=0.0, slopes=False, prefix=False),
        # Documents of all lengths packed in one row, each with its own first tokens, half-width heads.
        dict(name="attention_sinks_documents", kind="attention", hq=32, hkv=8, d=64, dtype="fp16",
             lengths="4096 17 1500 1 2048 0 530", causal=True, window=256, sinks=64, softcap=0.0, slopes=False,
             prefix=False),
    ]


def _text(numbers):
    return " ".join(str(n) for n in numbers)


def _numbers(case, field):
    return [int(n) for n in case[field].split()]


def _log_int(rng, lo, hi):
    return max(lo, min(hi, round(math.exp(rng.uniform(math.log(lo), math.log(hi))))))


def draw(rng):
    kind = rng.choice(["append", "append", "read", "paged", "paged", "paged", "paged", "attention", "attention"])
    d = rng.choice([64, 128, 128])
    dtype = rng.choice(["bf16", "bf16", "fp16"])
    codes = rng.choice(["fp8", "fp8", "int8"])
    hkv = _log_int(rng, 1, 56)
    hq = hkv * rng.choice([g for g in (1, 1, 2, 3, 4, 7, 8, 16) if g * hkv <= 64])
    page = rng.choice([16, 16, 32, 48, 64, 128])
    block = rng.choice([16, page] + [32] * (page % 32 == 0))
    b = _log_int(rng, 1, 64)
    decode = rng.random() < 0.5
    new = [1 if decode or rng.random() < 0.4 else _log_int(rng, 1, 1500) for _ in range(b)]
    window, sinks = _log_int(rng, 1, 4096), _log_int(rng, 1, 256)
    softcap, slopes = rng.choice([0.0, 0.0, 0.0, 20.0, 50.0]), rng.random() < 0.25
    if kind == "append":
        rotary = rng.choice([0, 0, d, d // 2, d // 4 + 2])
        while 2 * sum(new) * hkv * d > _MAX_VALUES:
            new = [(n + 1) // 2 for n in new]
        return dict(kind=kind, hq=hq if rotary else 0, hkv=hkv, d=d, rotary=rotary,
                    layout=rng.choice(["half", "interleaved"]), dtype=dtype, codes=codes, page=page, block=block,
                    new=_text(new), context=_text(n + rng.choice([0, _log_int(rng, 1, 1000)]) for n in new))
    if kind == "read":
        context = [_log_int(rng, 1, 32768) for _ in range(b)]
        while 2 * sum(context) * hkv * d > 2 * _MAX_VALUES:
            context = [(c + 1) // 2 for c in context]
        return dict(kind=kind, hkv=hkv, d=d, dtype=rng.choice([dtype, dtype, "fp32"]), codes=codes, page=page,
                    block=block, new=_text(rng.randint(1, c) for c in context), context=_text(context))
    if kind == "attention":
        lengths = [_log_int(rng, 1, 9914)]
        if rng.random() < 0.5:
            lengths = [rng.choice([0, 1, _log_int(rng, 2, 4096)]) for _ in range(rng.randint(2, 9))]
            lengths.append(rng.randint(1, 99))
        m = sum(lengths)
        while hq * m * m > _MAX_SCORES:
            lengths = [n // 2 for n in lengths[:-1]] + [lengths[-1] // 2 + 1]
            m = sum(lengths)
        case = dict(kind=kind, hq=hq, hkv=hkv, d=d, dtype=dtype, lengths=_text(lengths), causal=rng.random() < 0.75,
                    window=window, sinks=sinks, softcap=softcap, slopes=slopes, prefix=False)
        while work(case)["flops"] > _MAX_FLOPS:
            case["window"] = case["window"] * 3 // 4
        return case
    longest = _log_int(rng, 64, 131072)
    context = [n + _log_int(rng, 1, longest) for n in new]
    while (sum(context) * hkv * d * 4 > _MAX_BYTES or b * max(context) * hkv * d * 4 > 4 * _MAX_BYTES
           or 4 * d * b * max(new) * max(context) * hq > _MAX_FLOPS):
        new = [(n + 1) // 2 for n in new]
        context = [max(n, c // 2) for n, c in zip(new, context)]
    if rng.random() < 0.35:
        codes, block, page = "none", 0, rng.choice([16, 16, 32, 64, 128, 24, 7])
    sliding = codes == "none" or rng.random() < 0.35
    return dict(kind=kind, hq=hq, hkv=hkv, d=d, dtype=dtype, codes=codes, page=page, block=block, new=_text(new),
                context=_text(context), window=window if sliding else 0, sinks=sinks if sliding else 0, softcap=softcap,
                slopes=slopes, prefix=not sliding and rng.random() < 0.15)


# ---- inputs ---------------------------------------------------------------------------------


def _frequencies(case):
    """Radians a position of each rotated pair, in 64 bits."""
    return 10000.0 ** (-torch.arange(0, case["rotary"], 2, dtype=torch.float64) / case["rotary"])


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


def _scaled(x, e):
    """x times 2 to the whole numbers e, exact while neither leaves the range (torch.ldexp goes by a rounded power)."""
    power = ((e.long() + 1023) << 52).view(torch.float64)
    return x * (power if x.dtype == torch.float64 else power.float())


def _held(x, case):
    """A cache [pages, heads, page, d] as its codes and exponent bytes."""
    p, h, n, d = x.shape
    x = x.reshape(p, h, n // case["block"], case["block"], d)
    fraction, e = torch.frexp(x.abs().amax((3, 4)) / _LARGEST[case["codes"]])
    e = e - (fraction == 0.5).int()
    x = _scaled(x, -e[..., None, None])
    codes = x.to(torch.float8_e4m3fn).view(torch.uint8) if case["codes"] == "fp8" else x.round().to(torch.int8)
    return codes.reshape(p, h, n, d), (e + 127).to(torch.uint8)


def prepare(case, seed):
    """Inputs on the GPU from the seed alone: normal queries and values, keys whose channels differ in size, new tokens
    of which some are larger than those in the cache; the cache is full up to the context (behind it, what a page held
    before)."""
    g = torch.Generator(device="cuda").manual_seed(int(seed))
    dtype, d, kind, hkv = _DTYPES[case["dtype"]], case["d"], case["kind"], case["hkv"]

    def randn(*shape):
        return torch.randn(*shape, generator=g, device="cuda", dtype=torch.float32)

    s = {"case": dict(case)}
    if case.get("slopes"):
        s["slopes"] = torch.exp2(-8.0 * torch.arange(1, case["hq"] + 1, device="cuda", dtype=torch.float32) / case["hq"])
    if kind == "attention":
        m = sum(_numbers(case, "lengths"))
        s["q"], s["k"], s["v"] = (randn(h, m, d).to(dtype) for h in (case["hq"], hkv, hkv))
        if len(_numbers(case, "lengths")) > 1:
            s["starts"] = _starts(_numbers(case, "lengths"))
        return s
    new, context = _numbers(case, "new"), _numbers(case, "context")
    s["table"], count = _pages(g, case)
    s["starts"] = _starts(new)
    s["context"] = torch.tensor(context, dtype=torch.int32, device="cuda")
    uneven = torch.exp2(0.5 * randn(hkv, 1, d))
    k_cache, v_cache = randn(count, hkv, case["page"], d).mul_(uneven), randn(count, hkv, case["page"], d)
    if case["codes"] == "none":
        s["k_cache"], s["v_cache"] = k_cache.to(dtype), v_cache.to(dtype)
    else:
        s["k_cache"], s["k_scales"] = _held(k_cache, case)
        s["v_cache"], s["v_scales"] = _held(v_cache, case)
    del k_cache, v_cache
    if kind == "read":
        s["tokens"] = sum(new)
    elif kind == "paged":
        s["q"] = randn(case["hq"], sum(new), d).to(dtype)
        if case["prefix"]:
            s["prefix"] = torch.tensor(_prefixes(context), dtype=torch.int32, device="cuda")
    else:
        t = sum(new)
        size = torch.exp2(0.5 * randn(1, t, 1))
        s["k"], s["v"] = (randn(hkv, t, d) * uneven * size).to(dtype), (randn(hkv, t, d) * size).to(dtype)
        if case["rotary"]:
            s["frequencies"] = _frequencies(case).cuda()
            s["q"] = randn(case["hq"], t, d).to(dtype)
        # What is read back behind the append: every block that it touched, from its first token on.
        touched = [c - (c - n) // case["block"] * case["block"] for n, c in zip(new, context)]
        s["read_starts"], s["tokens"] = _starts(touched), sum(touched)
    return s


def _prefixes(lengths):
    """A prompt of about a third of each sequence that all of its tokens see."""
    return [n // 3 + n % 5 for n in lengths]


# ---- one pass --------------------------------------------------------------------------------


def run(s):
    return _OWN[s["case"]["kind"]](s, s["case"]) if own else _PLAIN[s["case"]["kind"]](s, s["case"])


@functools.lru_cache(maxsize=None)
def _package():
    path = str(Path(__file__).resolve().parent.parent / "m5-max-kernels_amd")
    if path not in sys.path:
        sys.path.insert(0, path)
    import m5kernels_amd

    return m5kernels_amd


def _own_append(s, c):
    q = _package().paged_append(
        s["k"], s["v"], s["k_cache"], s["v_cache"], s["table"], s["starts"], s["context"], q=s.get("q"),
        frequencies=s.get("frequencies"), layout=c["layout"], k_scales=s["k_scales"], v_scales=s["v_scales"])
    k, v = _package().paged_read(
        s["k_cache"], s["v_cache"], s["table"], s["read_starts"], s["context"], s["tokens"], k_scales=s["k_scales"],
        v_scales=s["v_scales"], dtype=s["k"].dtype)
    return {"k": k, "v": v} if q is None else {"q": q, "k": k, "v": v}


def _own_read(s, c):
    return _package().paged_read(
        s["k_cache"], s["v_cache"], s["table"], s["starts"], s["context"], s["tokens"], k_scales=s["k_scales"],
        v_scales=s["v_scales"], dtype=_DTYPES[c["dtype"]])


def _own_paged(s, c):
    return _package().paged_attention(
        s["q"], s["k_cache"], s["v_cache"], s["table"], s["starts"], s["context"], window=c["window"] or None,
        softcap=c["softcap"] or None, slopes=s.get("slopes"), prefix_lengths=s.get("prefix"), sinks=c["sinks"] or None,
        k_scales=s.get("k_scales"), v_scales=s.get("v_scales"))


def _own_attention(s, c):
    return _package().attention(
        s["q"], s["k"], s["v"], causal=c["causal"], window=c["window"], document_starts=s.get("starts"),
        softcap=c["softcap"] or None, slopes=s.get("slopes"), sinks=c["sinks"])


_OWN = {"append": _own_append, "read": _own_read, "paged": _own_paged, "attention": _own_attention}


# ---- the plain form ---------------------------------------------------------------------------


def _rotated(x, positions, s, layout):
    """x [heads, M, D] in 64 bits, which the angles of far positions and values next to a code's border need."""
    angle = positions.double()[:, None] * s["frequencies"][None, :]
    c, n = angle.cos(), angle.sin()
    x = x.double()
    r = c.shape[1]
    if layout == "half":
        a, b = x[..., :r], x[..., r:2 * r]
        y = torch.cat([a * c - b * n, b * c + a * n], -1)
    else:
        a, b = x[..., 0:2 * r:2], x[..., 1:2 * r:2]
        y = torch.stack([a * c - b * n, b * c + a * n], -1).flatten(-2)
    return torch.cat([y, x[..., 2 * r:]], -1)


def _places(starts, context, tokens):
    """Of every token: its sequence, and its position."""
    starts = starts.long()
    token = torch.arange(tokens, device="cuda")
    seq = torch.searchsorted(starts[1:], token, right=True)
    return seq, context.long()[seq] - starts[seq + 1] + token


def _values(codes):
    """What codes stand for, before their scale."""
    return codes.view(torch.float8_e4m3fn).float() if codes.dtype == torch.uint8 else codes.float()


def _codes(x, e, like):
    """Codes of x [..., D] under exponents e [...], ties to the even code."""
    x = _scaled(x, -e[..., None])
    if like.dtype == torch.int8:
        return x.round().to(torch.int8)
    step = _scaled(torch.ones_like(x), torch.frexp(x)[1].clamp(min=-5) - 4)  # 3 bits behind the first, 2^-9 at least
    return ((x / step).round() * step).float().to(torch.float8_e4m3fn).view(torch.uint8)


def _exponents(top, like):
    """The least e with top <= largest code * 2^e, as far as a byte goes."""
    fraction, e = torch.frexp(top / (448.0 if like.dtype == torch.uint8 else 127.0))
    return (e - (fraction == 0.5).int()).clamp(-127, 127).masked_fill(top == 0, -127)


def _read_back(codes, scales, s, starts, tokens, dtype):
    seq, position = _places(starts, s["context"], tokens)
    page, block = s["case"]["page"], s["case"]["block"]
    at, slot = s["table"].long()[seq, position // page], position % page
    e = scales[at, :, slot // block].int() - 127
    return _scaled(_values(codes[at, :, slot]), e[..., None]).transpose(0, 1).to(dtype).contiguous()


def _written(x, cache, scales, s, seq, position):
    """Writes x [tokens, heads, D], in 64 bits, into the cache."""
    page, block = s["case"]["page"], s["case"]["block"]
    at, slot = s["table"].long()[seq, position // page], position % page
    part = slot // block
    tops = torch.zeros(scales.shape, dtype=torch.float64, device="cuda").transpose(1, 2)  # pages, blocks, heads
    flat = tops.reshape(-1, tops.shape[2])
    where = (at * tops.shape[1] + part)[:, None].expand(-1, flat.shape[1])
    flat = flat.scatter_reduce(0, where, x.abs().amax(-1), "amax")
    e_new = _exponents(flat.gather(0, where), cache)
    # The block of a sequence's first new token may hold older ones: it keeps its exponent if that is the larger.
    first = s["starts"][:-1].long()
    p0, at0, part0 = position[first], at[first], part[first]
    rows = part0[:, None] * block + torch.arange(block, device="cuda")
    old = (rows < slot[first][:, None])[..., None]  # sequences, block, 1
    before = scales[at0, :, part0].int() - 127
    after = torch.where(old[:, :1, 0], torch.maximum(before, e_new[first]), e_new[first])
    held = cache[at0[:, None], :, rows]  # sequences, block, heads, D
    moved = _codes(_values(held).double(), (after - before)[:, None], cache)
    cache[at0[:, None], :, rows] = torch.where(old[..., None], moved, held)
    in_first = (position // block) == (p0 // block)[seq]
    e = torch.where(in_first[:, None], after[seq], e_new)
    scales[at, :, part] = (e + 127).to(torch.uint8)
    cache[at, :, slot] = _codes(x, e, cache)


def _plain_append(s, c):
    seq, position = _places(s["starts"], s["context"], s["k"].shape[1])
    k = _rotated(s["k"], position, s, c["layout"]) if c["rotary"] else s["k"].double()
    _written(k.transpose(0, 1), s["k_cache"], s["k_scales"], s, seq, position)
    _written(s["v"].double().transpose(0, 1), s["v_cache"], s["v_scales"], s, seq, position)
    dtype = s["k"].dtype
    out = {} if "q" not in s else {"q": _rotated(s["q"], position, s, c["layout"]).to(dtype)}
    out["k"] = _read_back(s["k_cache"], s["k_scales"], s, s["read_starts"], s["tokens"], dtype)
    out["v"] = _read_back(s["v_cache"], s["v_scales"], s, s["read_starts"], s["tokens"], dtype)
    return out


def _plain_read(s, c):
    return (_read_back(s["k_cache"], s["k_scales"], s, s["starts"], s["tokens"], _DTYPES[c["dtype"]]),
            _read_back(s["v_cache"], s["v_scales"], s, s["starts"], s["tokens"], _DTYPES[c["dtype"]]))


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
    tokens = s["q"].shape[1]
    seq, _ = _places(s["starts"], s["context"], tokens)
    index = torch.arange(tokens, device="cuda") - s["starts"].long()[seq]
    q = torch.zeros(b, hq, most, d, device="cuda")
    q[seq, :, index] = s["q"].float().transpose(0, 1)

    def gathered(name):
        x = s[name + "_cache"][s["table"].long()]
        if c["codes"] == "none":
            x = x.float()
        else:
            e = s[name + "_scales"][s["table"].long()].int() - 127
            x = _scaled(_values(x).unflatten(3, (-1, c["block"])), e[..., None, None]).flatten(3, 4)
        return x.permute(0, 2, 1, 3, 4).reshape(b, hkv, -1, d)

    k = gathered("k").transpose(2, 3).contiguous()
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
        visible &= (position - key < c["window"]) | (key < c["sinks"])
    if c["softcap"]:
        score.div_(c["softcap"]).tanh_().mul_(c["softcap"])
    if "slopes" in s:
        score -= s["slopes"][None, :, None, None] * (position - key).abs().float()[:, None]
    visible = visible[:, None].expand(b, hq, most, keys).reshape(b, hkv, -1, keys)
    o = _softmax_product(score.reshape(b, hkv, -1, keys), visible, gathered("v")).reshape(b, hq, most, d)
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
        visible, first = torch.ones(m, m, dtype=torch.bool, device="cuda"), torch.zeros_like(row)
    if c["causal"]:
        visible &= key <= row
    visible &= ((row - key).abs() < c["window"]) | (key - first < c["sinks"])
    if c["softcap"]:
        score.div_(c["softcap"]).tanh_().mul_(c["softcap"])
    if "slopes" in s:
        score -= s["slopes"].reshape(hkv, group, 1, 1) * (row - key).abs().float()
    o = _softmax_product(score, visible, s["v"].float()[:, None].expand(hkv, group, m, d))
    return o.reshape(hq, m, d).transpose(0, 1).reshape(m, hq * d).to(s["q"].dtype)


_PLAIN = {"append": _plain_append, "read": _plain_read, "paged": _plain_paged, "attention": _plain_attention}


# ---- what a pass cannot do without --------------------------------------------------------------


def _pairs(first, count, keys, causal, window, sinks, prefix):
    """Visible (row, key) pairs of `count` rows at positions first.. over `keys` keys."""
    p = torch.arange(first, first + count, dtype=torch.int64)
    hi = torch.clamp(torch.maximum(p + 1, torch.tensor(prefix)), max=keys) if causal else torch.full_like(p, keys)
    lo, kept = torch.zeros_like(p), torch.zeros_like(p)
    if window:
        lo = torch.clamp(p - window + 1, min=0)
        kept = torch.minimum(lo, torch.tensor(sinks))
        hi = torch.minimum(hi, p + window)
        if not causal:
            kept = kept + (torch.clamp(torch.tensor(sinks), max=keys) - hi).clamp(min=0)
    return int((hi - lo).clamp(min=0).sum() + kept.sum())


def work(case):
    kind, d, size = case["kind"], case["d"], 4 if case["dtype"] == "fp32" else 2
    hkv = case["hkv"]
    if kind == "read":
        t = sum(_numbers(case, "new"))
        return {"bytes": 2.0 * t * hkv * d * (1 + size) + 2.0 * t * hkv / case["block"], "flops": 2.0 * t * hkv * d}
    hq = case["hq"]
    if kind == "append":
        new, block = _numbers(case, "new"), case["block"]
        t = sum(new)
        touched = sum(c - (c - n) // block * block for n, c in zip(new, _numbers(case, "context")))
        return {"bytes": 2.0 * t * (hkv + hq) * d * size + 2.0 * hkv * d * (t + touched * size)
                + 4.0 * hkv * touched / block,
                "flops": 3.0 * t * (hq + hkv) * case["rotary"] + 2.0 * hkv * d * (2 * t + touched)}
    window, sinks, held = case["window"], case["sinks"], size
    if kind == "paged":
        prefixes = _prefixes(_numbers(case, "context")) if case["prefix"] else [0] * len(_numbers(case, "new"))
        pairs = keys = 0
        for n, c, f in zip(_numbers(case, "new"), _numbers(case, "context"), prefixes):
            if c >= n:
                pairs += _pairs(c - n, n, c, True, window, sinks, f)
                keys += min(c, n + window - 1 + sinks) if window else c
        rows = sum(_numbers(case, "new"))
        held = size if case["codes"] == "none" else 1.0 + 1.0 / (case["block"] * d)
    else:
        lengths = _numbers(case, "lengths")
        pairs = sum(_pairs(0, n, n, case["causal"], window, sinks, 0) for n in lengths)
        rows = keys = sum(lengths)
    return {"bytes": 2.0 * (keys * hkv * held + rows * hq * size) * d, "flops": 4.0 * d * hq * pairs}


# ---- the same in 64 bits --------------------------------------------------------------------------


def _turned64(x, positions, case):
    angle = torch.outer(positions.double(), _frequencies(case).cuda())
    turn = torch.polar(torch.ones_like(angle), angle)
    r, x = case["rotary"], x.double()
    head = x[..., :r]
    z = torch.complex(*head.chunk(2, -1)) if case["layout"] == "half" else torch.view_as_complex(
        head.reshape(*head.shape[:-1], r // 2, 2).contiguous())
    z = z * turn
    y = torch.cat([z.real, z.imag], -1) if case["layout"] == "half" else torch.view_as_real(z).flatten(-2)
    return torch.cat([y, x[..., r:]], -1)


def _codebook(kind):
    """The magnitudes that codes have, ascending: neighbours differ in the last bit of their code."""
    if kind == "int8":
        return torch.arange(128, dtype=torch.float64, device="cuda")
    return torch.tensor([m / 512 if e == 0 else (8 + m) * 2.0 ** (e - 10) for e in range(16) for m in range(8)][:127],
                        dtype=torch.float64, device="cuda")


def _nearest64(x, kind):
    """x to the nearest of the codebook, of two as near the even one."""
    book = _codebook(kind)
    y = x.abs()
    hi = torch.searchsorted(book, y).clamp(max=book.numel() - 1)
    lo = (hi - 1).clamp(min=0)
    below, above = y - book[lo], book[hi] - y
    pick = torch.where((below < above) | ((below == above) & (lo % 2 == 0)), lo, hi)
    return torch.copysign(book[pick], x)


def _power64(e):
    """2 to the whole numbers e of -127 .. 128, each as Python has it."""
    return torch.tensor([2.0 ** k for k in range(-127, 129)], dtype=torch.float64, device="cuda")[e.long() + 127]


def _least64(top, kind):
    """The least e with top <= largest * 2^e for each value of a vector."""
    found = []
    for t in top.tolist():
        e = -127 if t == 0 else math.ceil(math.log2(t / _LARGEST[kind]))
        while t and t <= math.ldexp(_LARGEST[kind], e - 1):
            e -= 1
        while t > math.ldexp(_LARGEST[kind], e):
            e += 1
        found.append(min(127, max(-127, e)))
    return torch.tensor(found, dtype=torch.float64, device="cuda")


def _decoded64(codes, scales, where, block, kind):
    """Keys of the pages `where` [n]: [heads, n * page, D]."""
    book = _codebook(kind)
    c = codes[where].long()
    magnitude, negative = (c & 127, c > 127) if kind == "fp8" else (c.abs(), c < 0)
    x = torch.where(negative, -book[magnitude.clamp(max=book.numel() - 1)], book[magnitude.clamp(max=book.numel() - 1)])
    x = x * _power64(scales[where].int() - 127).repeat_interleave(block, 2)[..., None]
    return x.transpose(0, 1).flatten(1, 2)


def _appended64(x, cache, scales, s, case):
    """Values of the touched blocks behind the append of x [heads, tokens, D], as they are read back."""
    block, page, kind, at, out = case["block"], case["page"], case["codes"], 0, []
    for b, (n, c) in enumerate(zip(_numbers(case, "new"), _numbers(case, "context"))):
        first = (c - n) // block * block
        where = s["table"][b, first // page:-(-c // page)].long()
        skip = first - first // page * page
        held = _decoded64(cache, scales, where, block, kind)[:, skip:skip + c - n - first]
        e_held = scales[where[0], :, skip // block].double() - 127
        for lo in range(first, c, block):
            hi = min(lo + block, c)
            new = x[:, at + max(lo, c - n) - (c - n):at + hi - (c - n)]
            e = _least64(new.abs().amax((1, 2)), kind)
            if lo < c - n:
                e = torch.maximum(e, e_held)
                new = torch.cat([held, new], 1)
            unit = _power64(e)[:, None, None]
            out.append(_nearest64(new / unit, kind) * unit)
        at += n
    return torch.cat(out, 1)


def _attend64(q, k, v, first, case, prefix, slopes):
    """q [rows, D] of one head at positions first.., k and v [keys, D]."""
    rows, keys = q.shape[0], k.shape[0]
    if rows == 0 or keys == 0:
        return torch.zeros_like(q)
    score = (q @ k.T) / math.sqrt(q.shape[1])
    if case["softcap"]:
        score = case["softcap"] * torch.tanh(score / case["softcap"])
    key = torch.arange(keys, device="cuda")[None, :]
    apart = (first + torch.arange(rows, device="cuda"))[:, None] - key
    if slopes is not None:
        score = score - slopes * apart.abs()
    hidden = torch.zeros(rows, keys, dtype=torch.bool, device="cuda")
    if case.get("causal", True):
        hidden |= (apart < 0) & (key >= prefix)
    if case["window"]:
        hidden |= (apart.abs() >= case["window"]) & (key >= case["sinks"])
    score = score.masked_fill(hidden, -math.inf)
    return torch.nan_to_num(torch.softmax(score, -1), nan=0.0) @ v


def exact(case, seed):
    s = prepare(case, seed)
    kind, hkv = case["kind"], case["hkv"]
    if kind == "append":
        spans = list(zip(_numbers(case, "new"), _numbers(case, "context")))
        position = torch.cat([torch.arange(c - n, c) for n, c in spans]).cuda()
        k = _turned64(s["k"], position, case) if case["rotary"] else s["k"].double()
        out = {} if "q" not in s else {"q": _turned64(s["q"], position, case)}
        out["k"] = _appended64(k, s["k_cache"], s["k_scales"], s, case)
        out["v"] = _appended64(s["v"].double(), s["v_cache"], s["v_scales"], s, case)
        return out
    if kind == "read":
        both = []
        for name in ("k", "v"):
            parts = []
            for b, (n, c) in enumerate(zip(_numbers(case, "new"), _numbers(case, "context"))):
                where = s["table"][b, :-(-c // case["page"])].long()
                parts.append(_decoded64(s[name + "_cache"], s[name + "_scales"], where, case["block"],
                                        case["codes"])[:, c - n:c])
            both.append(torch.cat(parts, 1))
        return tuple(both)
    hq, at = case["hq"], 0
    group = hq // hkv
    slopes = [float(x) for x in s["slopes"].cpu().double()] if "slopes" in s else [None] * hq
    out = torch.zeros(s["q"].shape[1], hq, case["d"], dtype=torch.float64, device="cuda")
    if kind == "attention":
        q, k, v = s["q"].double(), s["k"].double(), s["v"].double()
        for n in _numbers(case, "lengths"):
            for h in range(hq):
                out[at:at + n, h] = _attend64(q[h, at:at + n], k[h // group, at:at + n], v[h // group, at:at + n], 0,
                                              case, 0, slopes[h])
            at += n
        return out.reshape(out.shape[0], -1)
    prefixes = _prefixes(_numbers(case, "context")) if case["prefix"] else [0] * len(_numbers(case, "new"))
    for b, (n, c) in enumerate(zip(_numbers(case, "new"), _numbers(case, "context"))):
        where = s["table"][b, :-(-c // case["page"])].long()
        for h in range(hkv if c >= n else 0):
            one = slice(h, h + 1)
            if case["codes"] == "none":
                k, v = (t[where, h].reshape(-1, case["d"])[:c].double() for t in (s["k_cache"], s["v_cache"]))
            else:
                k, v = (_decoded64(s[x + "_cache"][:, one], s[x + "_scales"][:, one], where, case["block"],
                                   case["codes"])[0, :c] for x in ("k", "v"))
            for j in range(h * group, (h + 1) * group):
                out[at:at + n, j] = _attend64(s["q"][j, at:at + n].double(), k, v, c - n, case, prefixes[b], slopes[j])
        at += n
    return out.reshape(out.shape[0], -1)
