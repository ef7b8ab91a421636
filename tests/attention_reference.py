"""Attention, rotation and the paged cache in 64 bits on the CPU, one row at a time in spirit: every mask is
written as its condition on (position, key), none of the intervals that the kernels work with."""

from __future__ import annotations

import math

import torch


def rotate(x, positions, frequencies, layout="half", magnitude=1.0):
    """x [heads, tokens, width] in float64."""
    angle = torch.outer(positions.double(), frequencies)
    c, s = magnitude * torch.cos(angle), magnitude * torch.sin(angle)
    y, r = x.double().clone(), frequencies.shape[0]
    a, b = (slice(0, r), slice(r, 2 * r)) if layout == "half" else (slice(0, 2 * r, 2), slice(1, 2 * r, 2))
    x1, x2 = y[..., a].clone(), y[..., b].clone()
    y[..., a], y[..., b] = x1 * c - x2 * s, x2 * c + x1 * s
    return y


def attend(q, k, v, visible, position, scale, softcap=None, slopes=None):
    """q [heads, rows, D], k and v [kv_heads, keys, D], visible [rows, keys], position [rows]: (out, slack) in float64,
    [rows, heads, D].  What no row sees is taken out of k and v first.

    slack bounds what the kernel may be off by, apart from the output's own rounding: the probabilities' rounding to
    the inputs' type (half a step each, so half a step of the weighted sum of |v|), and the FP32 scores and sums.
    A dot product of D terms is off by at most D 2^-24 of its sum of magnitudes, in the exponent; a sum of n terms by
    n 2^-24 of itself; the exponential, the cap's tanh and the bias by a few units, counted as 2^-20 of their size."""
    dtype, group, d, n = q.dtype, q.shape[0] // k.shape[0], q.shape[2], k.shape[1]
    rows = q.shape[1]
    out = torch.zeros(rows, q.shape[0], d, dtype=torch.float64)
    slack = torch.zeros_like(out)
    if n == 0 or rows == 0:
        return out, slack
    half = torch.finfo(dtype).eps / 2
    for h in range(q.shape[0]):
        kh, vh, qh = k[h // group].double(), v[h // group].double(), q[h].double()
        score = torch.where(visible, qh @ torch.where(visible.any(0)[:, None], kh, 0.0).T, 0.0) * scale
        size = (qh.abs() @ torch.where(visible.any(0)[:, None], kh, 0.0).abs().T * scale).amax()
        off = (d + 8) * 2.0 ** -24 * size + n * 2.0 ** -24 + 2.0 ** -20 * (1 + score.abs().amax())
        if softcap is not None:
            score = softcap * torch.tanh(score / softcap)
            off = off + 2.0 ** -20 * softcap
        if slopes is not None:
            bias = slopes[h].double() * (position[:, None] - torch.arange(n)[None, :]).abs()
            score = score - bias
            off = off + 2.0 ** -22 * torch.where(visible, bias, 0.0).abs().amax()
        score = score.masked_fill(~visible, -math.inf)
        top = score.amax(1, keepdim=True)
        p = torch.exp(score - torch.where(top == -math.inf, 0.0, top))
        p = p / p.sum(1, keepdim=True).clamp_min(1e-300)
        clean = torch.where(visible.any(0)[:, None], vh, 0.0)
        out[:, h] = p @ clean
        tiny = n * 2.0 ** -25 if dtype == torch.float16 else 0.0  # probabilities below float16's normal range
        slack[:, h] = (half + 2 * off) * (p @ clean.abs()) + tiny * clean.abs().amax()
    return out, slack


def mask(rows_position, keys, causal, window=None, prefix=0):
    p, j = rows_position[:, None], torch.arange(keys)[None, :]
    m = torch.ones(p.shape[0], keys, dtype=torch.bool)
    if causal:
        m &= (j <= p) | (j < prefix)
    if window is not None:
        m &= (p - j < window) & (causal | (j - p < window))
    return m


def dense(q, k, v, *, causal=False, window=None, document_starts=None, prefix_lengths=None, softcap=None, slopes=None,
          scale=None):
    """(out, slack) of attention(), float64 [tokens, heads * D]; arguments on the CPU."""
    tokens, keys, d = q.shape[1], k.shape[1], q.shape[2]
    scale = 1 / math.sqrt(d) if scale is None else scale
    position = torch.arange(tokens) + keys - tokens
    if document_starts is None:
        visible = mask(position, keys, causal, window, 0 if prefix_lengths is None else int(prefix_lengths[0]))
    else:
        visible = torch.zeros(tokens, keys, dtype=torch.bool)
        starts = document_starts.tolist()
        for i, (s, e) in enumerate(zip(starts[:-1], starts[1:])):
            prefix = 0 if prefix_lengths is None else int(prefix_lengths[i])
            visible[s:e, s:e] = mask(torch.arange(e - s), e - s, causal, window, prefix)
    out, slack = attend(q, k, v, visible, position, scale, softcap, slopes)
    return out.reshape(tokens, -1), slack.reshape(tokens, -1)


def gather(cache, table, keys, page):
    """Keys 0..keys of one sequence, [kv_heads, keys, D], and which of them lie on a page that the cache has."""
    j = torch.arange(keys)
    ids = table.long()[j // page]
    has = (ids >= 0) & (ids < cache.shape[0])
    rows = cache[ids.clamp(0, cache.shape[0] - 1), :, j % page]
    return rows.transpose(0, 1), has


def paged(q, k_cache, v_cache, table, starts, context, *, window=None, prefix_lengths=None, softcap=None, slopes=None,
          scale=None):
    """(out, slack) of paged_attention(), float64 [tokens, heads * D]; arguments on the CPU."""
    heads, tokens, d = q.shape
    scale = 1 / math.sqrt(d) if scale is None else scale
    out, slack = (torch.zeros(tokens, heads, d, dtype=torch.float64) for _ in range(2))
    for b in range(table.shape[0]):
        s, e, keys = int(starts[b]), int(starts[b + 1]), max(int(context[b]), 0)
        position = torch.arange(e - s) + int(context[b]) - (e - s)
        k, has = gather(k_cache, table[b], keys, k_cache.shape[2])
        v, _ = gather(v_cache, table[b], keys, k_cache.shape[2])
        visible = mask(position, keys, True, window, 0 if prefix_lengths is None else int(prefix_lengths[b])) & has
        out[s:e], slack[s:e] = attend(q[:, s:e], k, v, visible, position, scale, softcap, slopes)
    return out.reshape(tokens, -1), slack.reshape(tokens, -1)


def close(got, out, slack):
    """The largest excess of |got - out| over slack and half a step of the output's type; <= 0 is within bounds."""
    eps = torch.finfo(got.dtype).eps / 2
    tiny = torch.finfo(got.dtype).smallest_normal * torch.finfo(got.dtype).eps
    got = got.cpu().double()
    assert torch.isfinite(got).all()
    return float((got - out).abs().sub(slack).sub(eps * (out.abs() + slack) + tiny).max()) if out.numel() else 0.0
