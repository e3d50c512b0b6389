"""Attention of a batch whose rows share a long prefix (a system prompt, a document, a common history).

The prefix's keys and values exist once.  Each query attends over ``[prefix ; the row's own keys]`` with
one softmax; the prefix is read once for the whole batch instead of once per row.
"""

from __future__ import annotations

import math

import torch

from ..ops._ext import require


def shared_prefix_attention(q: torch.Tensor, prefix_k: torch.Tensor, prefix_v: torch.Tensor, k: torch.Tensor,
                            v: torch.Tensor, lengths: torch.Tensor, heads: int, kv_heads: int, head_dim: int, *,
                            prefix_lengths: torch.Tensor | None = None, scale: float | None = None,
                            return_lse: bool = False):
    """``q`` ``[B, T, H D]``: the last ``T`` tokens of every row (``T = 1``: a decode step).  ``prefix_k`` /
    ``prefix_v`` ``[P, >= Hkv D]``: keys (post-rotary) and values that every row shares.  ``k`` / ``v``
    ``[B, capacity, >= Hkv D]``: the rows' own, of which the first ``lengths[b]`` (int32, these ``T`` tokens
    included, clamped to the capacity) are valid.  Token ``t`` of row ``b`` sees the first
    ``prefix_lengths[b]`` prefix keys (int32; all ``P`` by default) and own keys
    ``0 .. lengths[b] - T + t``.

    Returns ``[B, T, H D]`` (and, with ``return_lse``, the fp32 natural-log sums ``[B, H, T]``); a query that
    sees no key gives 0 and ``-inf``.  bf16, head dim 64 or 128; every view with contiguous rows,
    16-byte aligned, and a batch stride of ``k`` and ``v`` that is a multiple of their row stride.  Keys and
    values that no query sees are never used, whatever they hold; a value that one query sees and
    another does not must be finite (its weight is 0 there).  Scores, maxima and sums are fp32; each softmax weight
    is rounded to bf16 where it meets its value.  No gradients.
    """
    out, lse = require().shared_prefix_attention(q, prefix_k, prefix_v, k, v, lengths, heads, kv_heads, head_dim,
                                                 prefix_lengths, 1.0 / math.sqrt(head_dim) if scale is None else scale,
                                                 return_lse, False)
    return (out, lse) if return_lse else out


def shared_prefix_partials(q: torch.Tensor, prefix_k: torch.Tensor, prefix_v: torch.Tensor, k: torch.Tensor,
                           v: torch.Tensor, lengths: torch.Tensor, heads: int, kv_heads: int, head_dim: int, *,
                           prefix_lengths: torch.Tensor | None = None, scale: float | None = None):
    """``shared_prefix_attention`` before the division: fp32 ``(sums [B T, H, 1, D], (max, sum)
    [B T, H, 1, 2])``, the sums relative to the maximum.  For queries that attend over further keys
    elsewhere; ``merge_attention_partials`` joins both."""
    return tuple(require().shared_prefix_attention(q, prefix_k, prefix_v, k, v, lengths, heads, kv_heads, head_dim,
                                                   prefix_lengths,
                                                   1.0 / math.sqrt(head_dim) if scale is None else scale, False, True))


def merge_attention_partials(partials, more=None, *, batch: int, return_lse: bool = False):
    """One softmax from one or two sets of partials of the same queries: ``[batch, T, H D]`` bf16 (and the
    log sums ``[batch, H, T]``).  A part with maximum ``-inf`` counts as empty and is not read."""
    more_o, more_ml = more if more is not None else (None, None)
    out, lse = require().merge_attention_partials(*partials, more_o, more_ml, batch, return_lse)
    return (out, lse) if return_lse else out
