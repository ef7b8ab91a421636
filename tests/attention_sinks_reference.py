"""Attention with a window and first keys that stay visible, in 64 bits on the CPU (see attention_reference.py)."""

from __future__ import annotations

import math

import torch

import attention_reference as ref


def mask(position, keys, causal, window=None, prefix=0, sinks=None):
    m = ref.mask(position, keys, causal, window, prefix)
    if sinks is not None:
        p, j = position[:, None], torch.arange(keys)[None, :]
        m |= (j < sinks) & ((j <= p) | (not causal))
    return m


def dense(q, k, v, *, causal=False, window=None, document_starts=None, softcap=None, slopes=None, scale=None,
          sinks=None):
    """(out, slack) of attention(), float64 [tokens, heads * D]; arguments on the CPU."""
    tokens, keys, d = q.shape[1], k.shape[1], q.shape[2]
    scale = 1 / math.sqrt(d) if scale is None else scale
    position = torch.arange(tokens) + keys - tokens
    if document_starts is None:
        visible = mask(position, keys, causal, window, 0, sinks)
    else:
        visible = torch.zeros(tokens, keys, dtype=torch.bool)
        starts = document_starts.tolist()
        for s, e in zip(starts[:-1], starts[1:]):
            visible[s:e, s:e] = mask(torch.arange(e - s), e - s, causal, window, 0, sinks)
    out, slack = ref.attend(q, k, v, visible, position, scale, softcap, slopes)
    return out.reshape(tokens, -1), slack.reshape(tokens, -1)


def paged(q, k_cache, v_cache, table, starts, context, *, window=None, prefix_lengths=None, softcap=None, slopes=None,
          scale=None, sinks=None):
    """(out, slack) of paged_attention(), float64 [tokens, heads * D]; arguments on the CPU."""
    heads, tokens, d = q.shape
    scale = 1 / math.sqrt(d) if scale is None else scale
    out, slack = (torch.zeros(tokens, heads, d, dtype=torch.float64) for _ in range(2))
    for b in range(table.shape[0]):
        s, e, keys = int(starts[b]), int(starts[b + 1]), max(int(context[b]), 0)
        position = torch.arange(e - s) + int(context[b]) - (e - s)
        k, has = ref.gather(k_cache, table[b], keys, k_cache.shape[2])
        v, _ = ref.gather(v_cache, table[b], keys, k_cache.shape[2])
        prefix = 0 if prefix_lengths is None else int(prefix_lengths[b])
        visible = mask(position, keys, True, window, prefix, sinks) & has
        out[s:e], slack[s:e] = ref.attend(q[:, s:e], k, v, visible, position, scale, softcap, slopes)
    return out.reshape(tokens, -1), slack.reshape(tokens, -1)
