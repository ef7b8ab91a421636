"""The attention step behind the Q/K/V projections on MI355X: rotary positions, the paged cache that keys and
values are appended to, attention of new tokens over it, and attention without a cache.

Q, K and V come head-major, [heads, tokens, width], as projection_qk_rope and projection_qkv_rope return them (or as a
strided view of a gemm() output: ``y.view(tokens, heads, width).transpose(0, 1)`` is read in place); attention returns
[tokens, heads * width], the activations of the output projection.  Query head h reads key head
h // (heads / kv_heads).  Outputs are fresh tensors; only paged_append writes an argument, the caches.  These are
operators of inference: no gradient flows through them.

Sequences of one call lie behind each other along the token axis: ``query_starts`` int32 [sequences + 1], nondecreasing
from 0, says where each begins.  ``context_lengths`` int32 [sequences] counts the keys of each sequence's cache, its
new tokens included, and ``page_table`` int32 [sequences, width] names the pages that hold them.  All of them stay on
the device: a call reads no length back, so it can be captured into a graph and replayed with other lengths.
Nothing is checked that only the device knows; the kernels stay inside every buffer whatever the values.

A cache may be held in 8 bits: k_cache and v_cache are then codes, uint8 (E4M3) or int8 (in [-127, 127]), and k_scales
and v_scales uint8 [pages, kv_heads, page_size / block] are the exponent bytes of the power-of-two scales (as
quantize's "mxint8" has them) that the codes of `block` tokens of a page and head share: a code stands for
code * 2^(byte - 127), under byte 255 for NaN.  A block is 16 to 128 tokens, a multiple of 16 that divides the page;
heads are 64 or 128 wide.  paged_append writes such a cache, paged_read reads it back, paged_attention attends over it.
"""

from __future__ import annotations

import contextlib
import ctypes
import functools
import math

import torch

from . import _lib, hip

_LAYOUTS = ("half", "interleaved")
_HALF_DTYPES = (torch.float16, torch.bfloat16)
_FLOAT_DTYPES = (torch.float16, torch.bfloat16, torch.float32)
_CODE_MODES = {torch.uint8: _lib.QUANT_FP8, torch.int8: _lib.QUANT_INT8}
HEAD_DIMS = (64, 128)
BLOCK_MAX = 128
_READ_MAX = (1 << 35) - 2048  # values a head of a read, 8 a thread in workgroups of 256, below 2^32 threads
_WINDOW_MAX = (1 << 30) - 1
_F32_LEAST = 2.0 ** -126
_RATIO_MAX = 1e37  # scale / softcap: what a score is multiplied by before the cap's tanh, finite with its log2(e)


def rope_frequencies(rotary_dim, base=10000.0, *, scaling=None, factor=1.0, original_length=None, fast=32.0, slow=1.0,
                     device="cuda"):
    """(frequencies, magnitude) of rotary positions over the first `rotary_dim` channels: float64 radians a position
    of pair j, base ** (-2 j / rotary_dim), and the factor on cosine and sine.

    `scaling` stretches the positions of a model for contexts `factor` (>= 1) times as long:

    * "linear": every frequency divided by factor.
    * "ntk": base * factor ** (d / (d - 2)) in place of base: the lowest frequency is divided by factor, the highest
      stays.
    * "yarn": pairs that turn more than `fast` times over `original_length` positions stay, pairs that turn less than
      `slow` times are divided by factor, between them the two are mixed linearly; magnitude 0.1 ln(factor) + 1.
    """
    if not _lib.is_int(rotary_dim) or rotary_dim <= 0 or rotary_dim % 2:
        raise ValueError("rotary_dim must be a positive even integer")
    for name, v in (("base", base), ("factor", factor), ("fast", fast), ("slow", slow)):
        if not _lib.is_real(v) or not math.isfinite(v) or v <= 0:
            raise ValueError(f"{name} must be a positive finite real scalar")
    if scaling not in (None, "linear", "ntk", "yarn"):
        raise NotImplementedError("scaling must be None, 'linear', 'ntk' or 'yarn'")
    if factor < 1:
        raise ValueError("factor must be at least 1")
    if scaling is None and factor != 1:
        raise ValueError("factor needs a scaling")
    d, base, magnitude = int(rotary_dim), float(base), 1.0
    if scaling == "ntk":
        if d == 2:
            raise ValueError("'ntk' scaling needs more than one pair")
        base *= factor ** (d / (d - 2))
    f = base ** (torch.arange(0, d, 2, dtype=torch.float64) / -d)
    if scaling == "linear":
        f = f / factor
    elif scaling == "yarn":
        if not _lib.is_int(original_length) or original_length <= 0:
            raise ValueError("'yarn' scaling needs original_length, a positive integer")
        if fast <= slow:
            raise ValueError("fast must exceed slow")
        keep = ((original_length * f / (2 * math.pi) - slow) / (fast - slow)).clamp(0.0, 1.0)
        f = (1 - keep) * f / factor + keep * f
        magnitude = 0.1 * math.log(factor) + 1.0
    return f.to(device), magnitude


def _device(first, *named):
    """The device of `first`, which every other tensor has to share."""
    device = first.device
    for t, name in named:
        if t is not None and t.device != device:
            raise ValueError(f"{name} is on {t.device}, not on {device}")
    return device


def _on(device):
    """Launches go to the tensors' device, whatever the current one is."""
    if device.index == torch.cuda.current_device():
        return contextlib.nullcontext()
    return torch.cuda.device(device)


def _strides(t):
    """Strides in elements, 0 along axes of one entry (torch gives those any value)."""
    return [0 if n == 1 else s for n, s in zip(t.shape, t.stride())]


def _rows(t, name, aligned=True):
    """`t` where its last axis is contiguous and, if asked, its rows start at multiples of 16 bytes; else a copy."""
    if not t.is_cuda:
        raise ValueError(f"{name} must be a ROCm device tensor (got {t.device}); there is no CPU path")
    unit = 16 // t.element_size()
    if t.shape[-1] > 1 and t.stride(-1) != 1:
        return _lib.aligned_device_tensor(t, name)
    if aligned and (t.data_ptr() % 16 or any(s % unit for s in _strides(t)[:-1])):
        return _lib.aligned_device_tensor(t, name)
    return t


def _apart(t):
    """`t` [heads, keys, width], copied where its rows overlap or lie further apart than the kernel's windows reach."""
    if t.shape[1] > 1 and not t.shape[2] <= t.stride(1) <= 1 << 23:
        return t.contiguous()
    return t


def _heads_tensor(t, name, dtypes):
    if not isinstance(t, torch.Tensor) or t.dim() != 3:
        raise ValueError(f"{name} must be a [heads, tokens, width] tensor")
    if t.dtype not in dtypes:
        raise ValueError(f"{name} dtype must be " + ", ".join(str(d).removeprefix("torch.") for d in dtypes))
    if not t.shape[0] or not t.shape[2]:
        raise ValueError(f"{name} must have at least one head and one channel")
    return t.shape


def _int_vector(t, n, name):
    if not isinstance(t, torch.Tensor) or t.dtype != torch.int32 or tuple(t.shape) != (n,):
        raise ValueError(f"{name} must be an int32 vector of length {n}")
    return _lib.device_tensor(t, name)


def _positive(v, name):
    if not _lib.is_real(v) or not math.isfinite(v) or not 0 < v < 1e30:
        raise ValueError(f"{name} must be a positive finite real scalar")
    return float(v)


def _normal(v, name):
    """A positive scalar that FP32, in which the kernels take it, has a normal number for."""
    v = _positive(v, name)
    if v < _F32_LEAST:
        raise ValueError(f"{name} must be at least 2^-126")
    return v


def _rotation(frequencies, layout, magnitude, width):
    if layout not in _LAYOUTS:
        raise ValueError("layout must be 'half' or 'interleaved'")
    if not isinstance(frequencies, torch.Tensor) or frequencies.dtype != torch.float64 or frequencies.dim() != 1:
        raise ValueError("frequencies must be a float64 vector")
    if not 1 <= frequencies.shape[0] <= width // 2:
        raise ValueError("frequencies must hold 1 to width / 2 pairs")
    return _lib.device_tensor(frequencies, "frequencies"), _positive(magnitude, "magnitude")


def rope(x, positions, frequencies, *, layout="half", magnitude=1.0):
    """x [heads, tokens, width] with pair j of its first 2 * len(frequencies) channels turned by
    positions[token] * frequencies[j] radians (the product reduced in 64 bits: far positions stay exact) and scaled by
    `magnitude`; the other channels are copied.  Pair j is channels (j, j + pairs) with layout "half", (2j, 2j + 1) with
    "interleaved".  x float16, bfloat16 or float32 in any strides, positions int32 [tokens], frequencies float64
    [pairs] (rope_frequencies).  Computed in FP32 and rounded once; returns a contiguous tensor of x's dtype."""
    fast = hip._fast
    if fast is not None:
        y = fast.rope(x, positions, frequencies, layout, magnitude)
        if y is not None:
            return y
    heads, tokens, width = _heads_tensor(x, "x", _FLOAT_DTYPES)
    frequencies, magnitude = _rotation(frequencies, layout, magnitude, width)
    positions = _int_vector(positions, tokens, "positions")
    device = _device(x, (positions, "positions"), (frequencies, "frequencies"))
    x = _rows(x, "x", aligned=False)
    y = torch.empty((heads, tokens, width), dtype=x.dtype, device=device)
    if tokens == 0:
        return y
    xs = _strides(x)
    with _on(device):
        _lib.call("m5k_rope", _lib.ptr(x), _lib.dtype_code(x), tokens, heads, width, xs[0], xs[1], _lib.ptr(positions),
                  _lib.ptr(frequencies), frequencies.shape[0], int(layout == "interleaved"), magnitude, _lib.ptr(y),
                  _lib.stream_of(x))
    return y


def _cache(t, name, dtype, kv_heads, width):
    if not isinstance(t, torch.Tensor) or t.dim() != 4 or t.dtype != dtype:
        raise ValueError(f"{name} must be a [pages, kv_heads, page_size, width] tensor of {dtype}")
    if t.shape[1] != kv_heads or t.shape[3] != width or not all(t.shape):
        raise ValueError(f"{name} must have nonempty shape [pages, {kv_heads}, page_size, {width}]")
    if not t.is_cuda:
        raise ValueError(f"{name} must be a ROCm device tensor (got {t.device}); there is no CPU path")
    s = _strides(t)
    if t.stride(3) != 1:
        raise ValueError(f"{name} channels must be contiguous")
    return s


def _aligned_rows(t, s, name):
    unit = 16 // t.element_size()
    if t.data_ptr() % 16 or any(x % unit for x in s[:3]):
        raise ValueError(f"{name} rows must start at multiples of 16 bytes")


def _codes(k_cache, v_cache, k_scales, v_scales):
    """Of a cache in 8 bits: its mode, block and scales' strides, checked; None for one in 16 or 32."""
    if k_scales is None and v_scales is None:
        return None
    for t, scales, name in ((k_cache, k_scales, "k"), (v_cache, v_scales, "v")):
        if not isinstance(t, torch.Tensor) or t.dim() != 4 or t.dtype not in _CODE_MODES or not all(t.shape):
            raise ValueError(f"{name}_cache with scales must be a nonempty [pages, kv_heads, page_size, width] tensor "
                             "of uint8 or int8 codes")
        if not isinstance(scales, torch.Tensor) or scales.dim() != 3 or scales.dtype != torch.uint8:
            raise ValueError(f"{name}_scales must be a uint8 [pages, kv_heads, page_size / block] tensor")
    if k_scales.shape != v_scales.shape or k_scales.shape[:2] != k_cache.shape[:2] or not k_scales.shape[2]:
        raise ValueError("k_scales and v_scales must have the same shape, with the caches' pages and heads")
    page_size, blocks = k_cache.shape[2], k_scales.shape[2]
    if page_size % blocks:
        raise ValueError("the blocks that the scales count must divide the page")
    if page_size // blocks % 16 or page_size // blocks > BLOCK_MAX:
        raise NotImplementedError(f"a block must be 16 to {BLOCK_MAX} tokens, a multiple of 16")
    if k_cache.shape[3] not in HEAD_DIMS:
        raise NotImplementedError("a cache in 8 bits has heads of 64 or 128 channels")
    for scales, name in ((k_scales, "k_scales"), (v_scales, "v_scales")):
        if not scales.is_cuda:
            raise ValueError(f"{name} must be a ROCm device tensor (got {scales.device}); there is no CPU path")
        if blocks > 1 and scales.stride(2) != 1:
            raise ValueError(f"{name} of a page must be contiguous")
    return _CODE_MODES[k_cache.dtype], page_size // blocks, _strides(k_scales), _strides(v_scales)


def _paged(k_cache, v_cache, page_table, query_starts, context_lengths):
    if k_cache.shape != v_cache.shape:
        raise ValueError("k_cache and v_cache must have the same shape")
    if not isinstance(page_table, torch.Tensor) or page_table.dim() != 2 or page_table.dtype != torch.int32:
        raise ValueError("page_table must be an int32 [sequences, width] tensor")
    sequences, width = page_table.shape
    if not sequences or not width:
        raise ValueError("page_table must be nonempty")
    if k_cache.shape[2] > 1 << 20 or width * k_cache.shape[2] > 1 << 30:
        raise NotImplementedError("a sequence may have up to 2^30 keys, in pages of up to 2^20")
    return (_lib.device_tensor(page_table, "page_table"), _int_vector(query_starts, sequences + 1, "query_starts"),
            _int_vector(context_lengths, sequences, "context_lengths"))


def paged_append(k, v, k_cache, v_cache, page_table, query_starts, context_lengths, *, q=None, frequencies=None,
                 layout="half", magnitude=1.0, k_scales=None, v_scales=None):
    """Write new keys and values into a paged cache, the keys turned to their positions on the way.

    k, v [kv_heads, tokens, width] (float16, bfloat16 or float32, any strides); k_cache, v_cache
    [pages, kv_heads, page_size, width] of the same dtype, written in place.  Token i of the n new ones of sequence b
    has position context_lengths[b] - n + i.  With `frequencies` keys are turned as by rope(); without, they are stored
    as they are (those of projection_qk_rope are turned already).  `q` [heads, tokens, width] is turned by the same
    launch and returned (contiguous; rows behind the last sequence are 0); otherwise None is returned.

    A token whose position is negative (an idle slot: context_lengths 0) or lies behind the table, or whose table entry
    names no page, is not stored.  Where two tokens of one call name the same place, what lies there is unspecified:
    each channel of each head is one token's or the other's, in the keys and the values by themselves.

    With `k_scales` and `v_scales` the caches are codes, and they and the scales are written.  A block's scale is the
    least power of two 2^e with max |x| <= 448 * 2^e (E4M3; INT8: 127 * 2^e) over its tokens of this call, or, where it
    holds older tokens (positions below context_lengths[b] - n), the scale that it has, if that is larger; a code is
    x / 2^e to the nearest, ties to even.  Where the scale grows, the older tokens' codes are rounded again under it.
    Slots behind the context stay as they are.  A block that gets an infinity or NaN reads as NaN until it is written
    from its first slot on.  Keys are turned in 64 bits, and their codes rounded from that; one turned beyond FP32's
    range counts as an infinity.  Where two sequences of a call write into one block, its codes are unspecified."""
    fast = hip._fast
    if fast is not None:
        done = fast.paged_append(k, v, k_cache, v_cache, page_table, query_starts, context_lengths, q, frequencies,
                                 layout, magnitude, k_scales, v_scales)
        if done is not None:
            return None if done is True else done
    kv_heads, tokens, width = _heads_tensor(k, "k", _FLOAT_DTYPES)
    if not isinstance(v, torch.Tensor) or v.shape != k.shape or v.dtype != k.dtype:
        raise ValueError("k and v must have the same shape and dtype")
    codes = _codes(k_cache, v_cache, k_scales, v_scales)
    ks = _cache(k_cache, "k_cache", k_cache.dtype if codes else k.dtype, kv_heads, width)
    vs = _cache(v_cache, "v_cache", k_cache.dtype if codes else k.dtype, kv_heads, width)
    for t, name in ((k_cache, "k_cache"), (v_cache, "v_cache"), (k_scales, "k_scales"), (v_scales, "v_scales")):
        if t is not None and any(n > 1 and s == 0 for n, s in zip(t.shape, t.stride())):
            raise ValueError(f"{name} must not be an expanded view: it is written")
    if codes:
        _aligned_rows(k_cache, ks, "k_cache")
        _aligned_rows(v_cache, vs, "v_cache")
    page_table, query_starts, context_lengths = _paged(k_cache, v_cache, page_table, query_starts, context_lengths)
    pairs, heads, q_out, qs = 0, 0, None, (0, 0)
    if frequencies is not None:
        frequencies, magnitude = _rotation(frequencies, layout, magnitude, width)
        pairs = frequencies.shape[0]
    elif q is not None:
        raise ValueError("q is only turned: it needs frequencies")
    elif layout not in _LAYOUTS:
        raise ValueError("layout must be 'half' or 'interleaved'")
    if q is not None:
        heads, q_tokens, q_width = _heads_tensor(q, "q", (k.dtype,))
        if q_tokens != tokens or q_width != width:
            raise ValueError("q must have k's tokens and width")
    device = _device(k, (v, "v"), (k_cache, "k_cache"), (v_cache, "v_cache"), (page_table, "page_table"),
                     (query_starts, "query_starts"), (context_lengths, "context_lengths"), (q, "q"),
                     (frequencies, "frequencies"), (k_scales, "k_scales"), (v_scales, "v_scales"))
    aligned = codes is not None
    if q is not None:
        q = _rows(q, "q", aligned)
        qs = _strides(q)
        q_out = torch.empty((heads, tokens, width), dtype=k.dtype, device=device)
    k, v = _rows(k, "k", aligned), _rows(v, "v", aligned)
    if tokens == 0:
        return q_out
    kr, vr = _strides(k), _strides(v)
    if codes:
        mode, block, ke, ve = codes
        with _on(device):
            _lib.call(
                "m5k_paged_append_codes64", _lib.ptr(k), kr[0], kr[1], _lib.ptr(v), vr[0], vr[1], _lib.dtype_code(k),
                tokens, kv_heads, width, mode, _lib.ptr(k_cache), ks[0], ks[1], ks[2], _lib.ptr(k_scales), ke[0], ke[1],
                _lib.ptr(v_cache), vs[0], vs[1], vs[2], _lib.ptr(v_scales), ve[0], ve[1], block, k_cache.shape[0],
                k_cache.shape[2], _lib.ptr(page_table), page_table.shape[1], page_table.shape[0],
                _lib.ptr(query_starts), _lib.ptr(context_lengths), _lib.ptr(q), heads, qs[0], qs[1], _lib.ptr(q_out),
                _lib.ptr(frequencies), pairs, int(layout == "interleaved"), float(magnitude), _lib.stream_of(k))
        return q_out
    with _on(device):
        _lib.call(
            "m5k_paged_append", _lib.ptr(k), kr[0], kr[1], _lib.ptr(v), vr[0], vr[1], _lib.dtype_code(k), tokens,
            kv_heads, width, _lib.ptr(k_cache), ks[0], ks[1], ks[2], _lib.ptr(v_cache), vs[0], vs[1], vs[2],
            k_cache.shape[0], k_cache.shape[2], _lib.ptr(page_table), page_table.shape[1], page_table.shape[0],
            _lib.ptr(query_starts), _lib.ptr(context_lengths), _lib.ptr(q), heads, qs[0], qs[1], _lib.ptr(q_out),
            _lib.ptr(frequencies), pairs, int(layout == "interleaved"), float(magnitude), _lib.stream_of(k))
    return q_out


def paged_read(k_cache, v_cache, page_table, query_starts, context_lengths, tokens, *, k_scales, v_scales,
               dtype=torch.bfloat16):
    """Keys and values of a cache in 8 bits as (k, v), fresh [kv_heads, tokens, width] tensors of `dtype` (bfloat16,
    float16 or float32).

    Arguments are paged_append's: of sequence b the last n = query_starts[b + 1] - query_starts[b] of its
    context_lengths[b] keys, so that the call with paged_append's arguments gives what that call stored.  `tokens` is
    how many rows come back: query_starts[-1], or more where the host does not know it (rows behind it are 0), 2^28 at
    most and fewer than 2^28 - 15 of 128 channels.  Rows that paged_append would not store are 0 too.  Values are exact
    in float32 and bfloat16 down to their subnormals and rounded in float16; above a type's range they are
    infinities."""
    fast = hip._fast
    if fast is not None:
        done = fast.paged_read(k_cache, v_cache, page_table, query_starts, context_lengths, tokens, k_scales, v_scales,
                               dtype)
        if done is not None:
            return done
    if k_scales is None or v_scales is None:
        raise ValueError("paged_read reads caches in 8 bits: it needs k_scales and v_scales")
    mode, block, ke, ve = _codes(k_cache, v_cache, k_scales, v_scales)
    kv_heads, width = k_cache.shape[1], k_cache.shape[3]
    ks = _cache(k_cache, "k_cache", k_cache.dtype, kv_heads, width)
    vs = _cache(v_cache, "v_cache", k_cache.dtype, kv_heads, width)
    _aligned_rows(k_cache, ks, "k_cache")
    _aligned_rows(v_cache, vs, "v_cache")
    if dtype not in _FLOAT_DTYPES:
        raise ValueError("dtype must be bfloat16, float16 or float32")
    if not _lib.is_int(tokens) or tokens < 0:
        raise ValueError("tokens must be a nonnegative integer")
    if tokens > 1 << 28 or tokens * width > _READ_MAX:
        raise NotImplementedError("paged_read supports up to 2^28 tokens, and 2^35 - 2048 values a head")
    page_table, query_starts, context_lengths = _paged(k_cache, v_cache, page_table, query_starts, context_lengths)
    device = _device(k_cache, (v_cache, "v_cache"), (k_scales, "k_scales"), (v_scales, "v_scales"),
                     (page_table, "page_table"), (query_starts, "query_starts"), (context_lengths, "context_lengths"))
    k, v = (torch.empty((kv_heads, tokens, width), dtype=dtype, device=device) for _ in range(2))
    if tokens == 0:
        return k, v
    with _on(device):
        _lib.call(
            "m5k_paged_read", mode, _lib.ptr(k_cache), ks[0], ks[1], ks[2], _lib.ptr(k_scales), ke[0], ke[1],
            _lib.ptr(v_cache), vs[0], vs[1], vs[2], _lib.ptr(v_scales), ve[0], ve[1], block, k_cache.shape[0],
            k_cache.shape[2], kv_heads, width, _lib.ptr(page_table), page_table.shape[1], page_table.shape[0],
            _lib.ptr(query_starts), _lib.ptr(context_lengths), tokens, _lib.ptr(k), _lib.ptr(v), _lib.dtype_code(k),
            _lib.stream_of(k))
    return k, v


@functools.lru_cache(maxsize=4096)
def _plan(paged, tokens, heads, kv_heads, sequences, keys, cus):
    """(key splits, whether waves share rows) of a call (m5k_attention_plan; host only)."""
    n, few = ctypes.c_int(0), ctypes.c_int(0)
    _lib.call("m5k_attention_plan", paged, tokens, heads, kv_heads, sequences, keys, cus, ctypes.byref(n),
              ctypes.byref(few))
    return n.value, bool(few.value)


def _coded_plan(mode, width, modified):
    """What m5k_attention_plan calls a cache of codes."""
    return (2 if mode == _lib.QUANT_FP8 else 4) + 8 * (width == 128) + 16 * modified


def _first_keys(sinks, window):
    if sinks is None:
        return 0
    if not _lib.is_int(sinks) or sinks <= 0:
        raise ValueError("sinks must be a positive integer")
    if window is None:
        raise ValueError("sinks need a window")
    return min(int(sinks), _WINDOW_MAX)


def _reach(keys, window, sinks, causal):
    """Keys that the plan counts a row to see."""
    return min(keys, (1 if causal else 2) * window + sinks + 64) if sinks else keys


def _scores(q, heads, width, scale, softcap, window, slopes):
    scale = 1.0 / math.sqrt(width) if scale is None else _normal(scale, "scale")
    if softcap is None:
        softcap = 0.0
    else:
        softcap = _normal(softcap, "softcap")
        if scale / softcap > _RATIO_MAX:
            raise ValueError(f"scale / softcap must be at most {_RATIO_MAX:g}")
    if window is None:
        window = 0
    elif not _lib.is_int(window) or window <= 0:
        raise ValueError("window must be a positive integer")
    if slopes is not None:
        if not isinstance(slopes, torch.Tensor) or slopes.dtype != torch.float32 or tuple(slopes.shape) != (heads,):
            raise ValueError(f"slopes must be a float32 vector of length {heads}")
        slopes = _lib.device_tensor(slopes, "slopes")
    return scale, softcap, min(int(window), _WINDOW_MAX), slopes


def _query(q, kv_heads, width, dtype):
    heads, tokens, q_width = _heads_tensor(q, "q", _HALF_DTYPES)
    if q_width != width or q.dtype != dtype or heads % kv_heads:
        raise ValueError("q must have the keys' width and dtype, and a multiple of their heads")
    if width not in HEAD_DIMS:
        raise NotImplementedError("attention supports heads of 64 and 128 channels")
    if tokens > 1 << 24 or heads > 1 << 16 or tokens * heads >= 1 << 30:
        raise NotImplementedError("attention supports up to 2^24 tokens, and 2^30 rows over all heads")
    return heads, tokens


def _workspace(splits, tokens, heads, width, device):
    """Sums, maxima and totals of the key splits, or none."""
    if splits == 1:
        return None, 0
    n = splits * tokens * heads * (width + 2)
    return torch.empty((n,), dtype=torch.float32, device=device), n


def paged_attention(q, k_cache, v_cache, page_table, query_starts, context_lengths, *, scale=None, window=None,
                    softcap=None, slopes=None, prefix_lengths=None, sinks=None, k_scales=None, v_scales=None):
    """Attention of new tokens, single ones or chunks, over a paged cache that holds their keys and values already.

    q [heads, tokens, width] (bfloat16 or float16, width 64 or 128); caches [pages, kv_heads, page_size, width] of the
    same dtype, any page_size, channels contiguous and rows at multiples of 16 bytes.  The n new tokens of sequence b
    are the last n of its context_lengths[b] keys; a token at position p sees keys j <= p, of them with `window` those
    with p - j < window and with `sinks` (a number; it needs a window) the sequence's first ones too, j < sinks, and
    with `prefix_lengths` (int32 [sequences]) also every j below the prefix.  Scores are
    scale * q . k (scale defaults to width ** -0.5); `softcap` c turns s into c * tanh(s / c); `slopes` (float32
    [heads]) then adds -slopes[h] * (distance of j from p).  Scores are FP32 numbers of any size; scale and c are normal
    ones, scale / c at most 1e37.  Returns
    [tokens, heads * width]; rows that see no key, and rows behind the last sequence, are 0; rows that see only keys of
    score -inf are NaN.  Keys on pages that a table entry outside [0, pages) would name are left out.

    With `k_scales` and `v_scales` the caches are codes; keys and values are taken in q's dtype, as paged_read gives
    them."""
    fast = hip._fast
    if fast is not None:
        out = fast.paged_attention(q, k_cache, v_cache, page_table, query_starts, context_lengths, scale, window,
                                   softcap, slopes, prefix_lengths, sinks, k_scales, v_scales)
        if out is not None:
            return out
    if prefix_lengths is not None and window is not None:
        raise NotImplementedError("a window and a prefix cannot be combined")
    if not isinstance(k_cache, torch.Tensor) or k_cache.dim() != 4:
        raise ValueError("k_cache must be a [pages, kv_heads, page_size, width] tensor")
    kv_heads, width = k_cache.shape[1], k_cache.shape[3]
    codes = _codes(k_cache, v_cache, k_scales, v_scales)
    ks = _cache(k_cache, "k_cache", k_cache.dtype, kv_heads, width)
    vs = _cache(v_cache, "v_cache", k_cache.dtype, kv_heads, width)
    _aligned_rows(k_cache, ks, "k_cache")
    _aligned_rows(v_cache, vs, "v_cache")
    if codes and k_cache.shape[2] > 1 and not all(width <= s[2] <= 1 << 23 for s in (ks, vs)):
        raise NotImplementedError("rows of codes must be width to 2^23 bytes apart")
    heads, tokens = _query(q, kv_heads, width, k_cache.dtype if codes is None else getattr(q, "dtype", None))
    page_table, query_starts, context_lengths = _paged(k_cache, v_cache, page_table, query_starts, context_lengths)
    sequences, table_width = page_table.shape
    sinks = _first_keys(sinks, window)
    scale, softcap, window, slopes = _scores(q, heads, width, scale, softcap, window, slopes)
    if prefix_lengths is not None:
        prefix_lengths = _int_vector(prefix_lengths, sequences, "prefix_lengths")
    device = _device(q, (k_cache, "k_cache"), (v_cache, "v_cache"), (page_table, "page_table"),
                     (query_starts, "query_starts"), (context_lengths, "context_lengths"), (slopes, "slopes"),
                     (prefix_lengths, "prefix_lengths"), (k_scales, "k_scales"), (v_scales, "v_scales"))
    out = torch.empty((tokens, heads * width), dtype=q.dtype, device=device)
    if tokens == 0:
        return out
    q = _rows(q, "q")
    qs = _strides(q)
    pages, page_size = k_cache.shape[0], k_cache.shape[2]
    kind = _coded_plan(codes[0], width, softcap > 0 or slopes is not None) if codes else 1
    splits, _ = _plan(kind, tokens, heads, kv_heads, sequences, _reach(table_width * page_size, window, sinks, True),
                      hip._cu_count_of(device.index))
    workspace, n = _workspace(splits, tokens, heads, width, device)
    name, mode, k_more, v_more = "m5k_paged_attention_sinks", (), (), ()
    if codes:
        mode, block, ke, ve = codes
        name, mode = "m5k_paged_attention_codes", (mode,)
        k_more, v_more = (_lib.ptr(k_scales), ke[0], ke[1]), (_lib.ptr(v_scales), ve[0], ve[1], block)
    with _on(device):
        _lib.call(
            name, _lib.ptr(q), _lib.dtype_code(q), tokens, heads, width, qs[0], qs[1], *mode, _lib.ptr(k_cache), ks[0],
            ks[1], ks[2], *k_more, _lib.ptr(v_cache), vs[0], vs[1], vs[2], *v_more, pages, page_size, kv_heads,
            _lib.ptr(page_table), table_width, sequences, _lib.ptr(query_starts), _lib.ptr(context_lengths), scale,
            window, sinks, softcap, _lib.ptr(slopes), _lib.ptr(prefix_lengths), _lib.ptr(out), splits,
            _lib.ptr(workspace), n, _lib.stream_of(q))
    return out


def attention(q, k, v, *, causal=False, window=None, document_starts=None, prefix_lengths=None, softcap=None,
              slopes=None, scale=None, sinks=None):
    """softmax(scores) V of q [heads, tokens, width] over k, v [kv_heads, keys, width] (bfloat16 or float16, width 64 or
    128, any strides): [tokens, heads * width].

    Token i stands at key position p = i + keys - tokens.  `causal` shows it keys j <= p; `window` those with
    p - j < window (and, without causal, j - p < window), and with `sinks` (a number; it needs a window) the first ones
    of the row's document, or of all keys, too.  `document_starts` (int32 [documents + 1], nondecreasing from
    0, as many keys as tokens) confines it to its own document.  `prefix_lengths` (int32 [documents], or [1]; with
    causal, without window) shows every token of a document that many of its first keys too.  Scores as in
    paged_attention.  A row that sees no key, and a row behind the last document, is 0."""
    fast = hip._fast
    if fast is not None:
        out = fast.attention(q, k, v, causal, window, document_starts, prefix_lengths, softcap, slopes, scale, sinks)
        if out is not None:
            return out
    if prefix_lengths is not None and window is not None:
        raise NotImplementedError("a window and a prefix cannot be combined")
    kv_heads, keys, width = _heads_tensor(k, "k", _HALF_DTYPES)
    if not isinstance(v, torch.Tensor) or v.shape != k.shape or v.dtype != k.dtype:
        raise ValueError("k and v must have the same shape and dtype")
    heads, tokens = _query(q, kv_heads, width, k.dtype)
    if keys > 1 << 24:
        raise NotImplementedError("attention supports up to 2^24 keys")
    if not isinstance(causal, bool):
        raise ValueError("causal must be a boolean")
    sinks = _first_keys(sinks, window)
    scale, softcap, window, slopes = _scores(q, heads, width, scale, softcap, window, slopes)
    documents = 0
    if document_starts is not None:
        if not isinstance(document_starts, torch.Tensor) or document_starts.dim() != 1 or document_starts.numel() < 2:
            raise ValueError("document_starts must be an int32 vector of at least 2 entries")
        if tokens != keys:
            raise ValueError("documents need as many keys as tokens")
        documents = document_starts.shape[0] - 1
        document_starts = _int_vector(document_starts, documents + 1, "document_starts")
    if prefix_lengths is not None:
        if not causal:
            raise ValueError("a prefix needs a causal mask")
        prefix_lengths = _int_vector(prefix_lengths, max(documents, 1), "prefix_lengths")
    device = _device(q, (k, "k"), (v, "v"), (document_starts, "document_starts"), (slopes, "slopes"),
                     (prefix_lengths, "prefix_lengths"))
    out = torch.empty((tokens, heads * width), dtype=q.dtype, device=device)
    if tokens == 0:
        return out
    q, k, v = _rows(q, "q"), _apart(_rows(k, "k")), _apart(_rows(v, "v"))
    qs, ks, vs = _strides(q), _strides(k), _strides(v)
    splits, _ = _plan(0, tokens, heads, kv_heads, documents, _reach(keys, window, sinks, causal),
                      hip._cu_count_of(device.index))
    workspace, n = _workspace(splits, tokens, heads, width, device)
    with _on(device):
        _lib.call(
            "m5k_attention_sinks", _lib.ptr(q), _lib.dtype_code(q), tokens, heads, width, qs[0], qs[1], _lib.ptr(k),
            ks[0], ks[1], _lib.ptr(v), vs[0], vs[1], keys, kv_heads, scale, int(causal), window, sinks, softcap,
            _lib.ptr(slopes), _lib.ptr(document_starts), documents, _lib.ptr(prefix_lengths), _lib.ptr(out), splits,
            _lib.ptr(workspace), n, _lib.stream_of(q))
    return out
