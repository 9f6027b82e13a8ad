"""Rotary positions of queries and keys.

The reference's attention takes queries and keys that are already turned (its
hook sits after RoPE, eval/perplexity_eval.py:366-395); these are the turns
themselves, on tensors here and on the way into a paged cache in
`paged_cache.append_paged`.
"""

from __future__ import annotations

import math
from dataclasses import dataclass
from typing import Dict, Optional

import torch

from ._ops import ops


@dataclass(frozen=True)
class RotaryTable:
    """Radians per position of every pair, float64 (rotary_dim // 2,) on the
    GPU, and the factor that turned rows are scaled by."""
    inv_freq: torch.Tensor
    scale: float = 1.0

    @property
    def rotary_dim(self) -> int:
        return 2 * self.inv_freq.shape[0]


def rotary_table(rotary_dim: int, base: float = 10000.0, *, scaling: Optional[Dict] = None, scale: float = 1.0,
                 device="cuda") -> RotaryTable:
    """inv_freq[i] = base^(-2 i / rotary_dim), for long contexts changed by
    scaling = {"type": ...}:

    "linear"  factor: every frequency / factor.
    "ntk"     factor: base times factor^(rotary_dim / (rotary_dim - 2)), which
              divides the lowest frequency by factor and keeps the highest.
    "ramp"    factor, low, high, original: a pair that turns r = original *
              inv_freq / (2 pi) times over the original context keeps its
              frequency for r > high, has it / factor for r < low, and a linear
              mixture by (r - low) / (high - low) between.

    Any other frequencies (a model's own) go straight into RotaryTable."""
    if rotary_dim < 2 or rotary_dim % 2:
        raise ValueError(f"rotary_dim {rotary_dim} must be even and positive")
    if not base > 0:
        raise ValueError(f"base {base} must be positive")
    kind = None if scaling is None else scaling.get("type")
    factor = 1.0 if scaling is None else float(scaling["factor"])
    if not factor > 0:
        raise ValueError(f"scaling factor {factor} must be positive")
    if kind == "ntk":
        if rotary_dim == 2:
            raise ValueError("ntk scaling needs rotary_dim > 2")
        base = base * factor ** (rotary_dim / (rotary_dim - 2))
    f = [base ** (-2.0 * i / rotary_dim) for i in range(rotary_dim // 2)]
    if kind == "linear":
        f = [x / factor for x in f]
    elif kind == "ramp":
        low, high, n = float(scaling["low"]), float(scaling["high"]), float(scaling["original"])
        if not low < high:
            raise ValueError(f"ramp scaling needs low < high, got {low}, {high}")
        keep = [min(max((n * x / (2 * math.pi) - low) / (high - low), 0.0), 1.0) for x in f]
        f = [g * x + (1.0 - g) * x / factor for g, x in zip(keep, f)]
    elif kind not in (None, "ntk"):
        raise ValueError(f"unknown scaling type {kind!r} (linear, ntk, ramp)")
    return RotaryTable(torch.tensor(f, dtype=torch.float64, device=device), float(scale))


def apply_rotary(q: torch.Tensor, k: Optional[torch.Tensor], positions: torch.Tensor, table: RotaryTable, *,
                 layout: str = "half", backward: bool = False, inplace: bool = False):
    """q (and k) turned by their positions (oc_apply_rotary).

    q, k: (batch, heads, tokens, head_dim), or (tokens, heads, head_dim), in
    float32, float16 or bfloat16, any strides but a contiguous last
    dimension; k may be None.  positions: int32 or int64 (tokens,) or (batch,
    tokens).  layout: "half" pairs column i with i + rotary_dim / 2,
    "interleaved" 2 i with 2 i + 1; columns from rotary_dim on are kept.
    Angles are formed in float64, the rest in float32, rounded once.
    backward: the transposed rotation, which takes the gradients of the turned
    tensors to those of q and k.  inplace: into q and k themselves, which must
    share no elements.

    Returns q' (and k', as a pair, when k is given)."""
    return ops().apply_rotary(q, k, positions, table.inv_freq, table.scale, layout, backward, inplace)
