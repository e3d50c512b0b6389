"""Rotary positions: half and interleaved layouts, part of the head, scaled tables.

``rotary`` rotates queries and keys in one launch and carries gradients (the backward is the
transposed rotation); ``rotary_cache`` is the serving form, which takes a fused ``[q | k | v]``
projection and leaves rotated keys and plain values in their cache rows.  Angles come from a
``RotaryTable``: fp32 cosines and sines of angles computed in 64 bits.
"""

from __future__ import annotations

import math
from dataclasses import dataclass

import torch

from ._ext import require


@dataclass(frozen=True)
class RotaryTable:
    """``cos`` / ``sin`` ``[positions, rotary_dim / 2]`` fp32; ``interleaved`` pairs elements
    ``(2i, 2i + 1)``, the half layout ``(i, i + rotary_dim / 2)``."""

    cos: torch.Tensor
    sin: torch.Tensor
    interleaved: bool = False

    @property
    def rotary_dim(self) -> int:
        return 2 * self.cos.shape[1]


def rotary_frequencies(rotary_dim: int, theta: float = 10000.0, scaling: dict | None = None,
                       max_positions: int | None = None) -> tuple[torch.Tensor, float]:
    """Angle per position of every pair (fp64 ``[rotary_dim / 2]``) and the factor on cosines and
    sines.  ``scaling`` (``rope_type`` or ``type``, and its numbers) stretches the positions a
    model was trained on:

    * ``linear``: every angle divided by ``factor``;
    * ``ntk``: the base raised to ``theta * factor^(d / (d - 2))``; ``dynamic``: the same with the
      factor grown with ``max_positions`` over ``original_max_position_embeddings``: the angles of a
      sequence of that length (``rotary_angles`` takes sequences of several lengths);
    * ``llama3``: wavelengths over ``original / low_freq_factor`` divided by ``factor``, those under
      ``original / high_freq_factor`` kept, a linear blend between;
    * ``yarn``: pairs that turn less than ``beta_slow`` times over the original window are divided by
      ``factor``, those over ``beta_fast`` kept, a linear ramp between; cosines and sines times
      ``attention_factor`` (``0.1 ln(factor) + 1`` unless given).
    """
    if rotary_dim <= 0 or rotary_dim % 2:
        raise ValueError("rotary_dim must be a positive even number")
    pair = torch.arange(0, rotary_dim // 2, dtype=torch.float64) / (rotary_dim // 2)
    freq = 1.0 / float(theta) ** pair
    if not scaling:
        return freq, 1.0
    kind = scaling.get("rope_type", scaling.get("type", "default"))
    if kind == "default":
        return freq, 1.0
    if kind not in ("linear", "ntk", "dynamic", "llama3", "yarn"):
        raise ValueError(f"unknown rotary scaling {kind!r} (linear, ntk, dynamic, llama3, yarn)")
    factor = float(scaling.get("factor", 1.0))
    if not factor >= 1.0:
        raise ValueError("rotary scaling needs a factor of at least 1")
    if kind == "linear":
        return freq / factor, 1.0
    original = scaling.get("original_max_position_embeddings")
    if kind != "ntk" and not original:
        raise ValueError(f"rotary scaling {kind!r} needs original_max_position_embeddings")
    if kind in ("ntk", "dynamic"):
        if rotary_dim == 2:
            return freq, 1.0  # the single pair's angle does not depend on the base
        if kind == "dynamic":
            length = max(int(max_positions or original), int(original))
            factor = factor * length / original - (factor - 1.0)
        return (float(theta) * factor ** (rotary_dim / (rotary_dim - 2))) ** -pair, 1.0
    if kind == "llama3":
        low, high = float(scaling.get("low_freq_factor", 1.0)), float(scaling.get("high_freq_factor", 4.0))
        if not high > low:
            raise ValueError("llama3 scaling needs high_freq_factor > low_freq_factor")
        turns = original * freq / (2 * math.pi)  # full turns over the original window
        keep = ((turns - low) / (high - low)).clamp(0.0, 1.0)
        return freq * keep + freq / factor * (1 - keep), 1.0
    fast, slow = float(scaling.get("beta_fast", 32.0)), float(scaling.get("beta_slow", 1.0))

    def pair_of(turns: float) -> float:  # the pair index that makes this many turns over the window
        return rotary_dim * math.log(original / (turns * 2 * math.pi)) / (2 * math.log(theta))

    first, last = pair_of(fast), pair_of(slow)
    if scaling.get("truncate", True):
        first, last = math.floor(first), math.ceil(last)
    first, last = max(first, 0), min(last, rotary_dim - 1)
    ramp = ((torch.arange(rotary_dim // 2, dtype=torch.float64) - first) / max(last - first, 1e-3)).clamp(0.0, 1.0)
    scale = scaling.get("attention_factor")
    if scale is None:
        def mscale(m: float) -> float:
            return 0.1 * m * math.log(factor) + 1.0 if factor > 1.0 else 1.0

        m, m_all = scaling.get("mscale"), scaling.get("mscale_all_dim")
        scale = mscale(float(m)) / mscale(float(m_all)) if m and m_all else mscale(1.0)
    return freq * (1 - ramp) + freq / factor * ramp, float(scale)


def dynamic_window(scaling: dict | None) -> int | None:
    """The window of ``dynamic`` scaling, past which angles go by the length of the sequence; ``None`` for others."""
    if not scaling or scaling.get("rope_type", scaling.get("type")) != "dynamic":
        return None
    return int(scaling["original_max_position_embeddings"])


def rotary_angles(positions: torch.Tensor, rotary_dim: int, theta: float = 10000.0, scaling: dict | None = None,
                  lengths: torch.Tensor | int | None = None) -> tuple[torch.Tensor, float]:
    """fp64 angles ``[..., rotary_dim / 2]`` of integer ``positions`` ``[...]`` and the factor on cosines and
    sines.  ``lengths`` (broadcast against ``positions``): the length of the sequence that a position is rotated
    in, which only ``dynamic`` scaling goes by; by default the sequence ends at the position, as in a decode
    step."""
    freq, scale = rotary_frequencies(rotary_dim, theta, scaling)
    window = dynamic_window(scaling)
    positions = positions.to(torch.float64)[..., None]
    if window is None or rotary_dim == 2:
        return positions * freq.to(positions.device), scale
    if lengths is None:
        lengths = positions + 1
    else:
        lengths = torch.as_tensor(lengths, device=positions.device).to(torch.float64)[..., None]
    factor = float(scaling.get("factor", 1.0))
    grown = factor * lengths.clamp(min=window) / window - (factor - 1.0)
    pair = torch.arange(0, rotary_dim // 2, dtype=torch.float64, device=positions.device) / (rotary_dim // 2)
    return positions * (float(theta) * grown ** (rotary_dim / (rotary_dim - 2))) ** -pair, scale


def rotary_table(rotary_dim: int, max_positions: int, *, theta: float = 10000.0, scaling: dict | None = None,
                 interleaved: bool = False, device="cuda") -> RotaryTable:
    """The table of positions ``0 .. max_positions - 1`` (angles in 64 bits, entries rounded once)."""
    freq, scale = rotary_frequencies(rotary_dim, theta, scaling, max_positions)
    angle = torch.arange(max_positions, dtype=torch.float64)[:, None] * freq
    return RotaryTable((angle.cos() * scale).float().to(device), (angle.sin() * scale).float().to(device), interleaved)


def rotary(q: torch.Tensor, k: torch.Tensor | None, positions: torch.Tensor, table: RotaryTable):
    """``q`` ``[..., H, D]`` and ``k`` ``[..., Hkv, D]`` (bf16, fp16 or fp32; the same leading
    dimensions; strided views are read in place) rotated by ``positions`` ``[...]`` (int32 or
    int64).  Returns new contiguous tensors ``(q', k')`` (``k'`` is ``None`` without ``k``), with
    gradients for ``q`` and ``k`` (of any order; none for the table and none in forward mode, which are
    refused; a backward pass captured into a CUDA graph needs, as
    with every operator, that no eager graph of the same leaves is alive).  Elements behind
    ``table.rotary_dim`` pass through; a position outside the table gives NaN in the rotated part of its
    token."""
    return tuple(require().rotary(q, k, positions, table.cos, table.sin, table.interleaved, False))


def rotary_cache(qkv: torch.Tensor, heads: int, kv_heads: int, head_dim: int, positions: torch.Tensor,
                 table: RotaryTable, k_cache: torch.Tensor, v_cache: torch.Tensor, slots: torch.Tensor) -> torch.Tensor:
    """Serving form, one launch, no gradients: token ``m`` of ``qkv`` ``[M, (H + 2 Hkv) D]`` leaves its
    rotated keys and its values in row ``slots[m]`` (int32) of ``k_cache`` / ``v_cache``
    ``[rows, >= Hkv D]``, and its rotated queries in the returned ``[M, H D]``.  A slot outside the
    cache (-1 for padding) writes nothing; slots of one call must differ."""
    return require().rotary_cache(qkv, heads, kv_heads, head_dim, positions, table.cos, table.sin, table.interleaved,
                                  k_cache, v_cache, slots)
