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

from . import _launch as X
from . import _native as N

LAYOUTS = ("half", "interleaved")


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


def check_table(table: Optional[RotaryTable], head_dim: int, layout: str, device: torch.device) -> int:
    """The columns that `table` turns (0 without one)."""
    if layout not in LAYOUTS:
        raise ValueError(f"layout must be one of {LAYOUTS}, got {layout!r}")
    if table is None:
        return 0
    f = table.inv_freq
    if f.dtype != torch.float64 or f.dim() != 1 or not f.is_contiguous() or f.device != device:
        raise ValueError(f"inv_freq must be a contiguous float64 vector on {device}")
    if table.rotary_dim > head_dim:
        raise ValueError(f"the table turns {table.rotary_dim} columns, head_dim is {head_dim}")
    return table.rotary_dim


def check_positions(positions: torch.Tensor, device: torch.device) -> torch.Tensor:
    if positions.dtype not in (torch.int32, torch.int64):
        raise TypeError(f"positions must be int32 or int64, got {positions.dtype}")
    if positions.device != device:
        raise RuntimeError(f"orthocache_gpu: positions on {positions.device}, the rest on {device}")
    return positions if positions.shape[-1] <= 1 or positions.stride(-1) == 1 else positions.contiguous()


def no_grad_needed(what: str, *tensors: Optional[torch.Tensor]) -> None:
    """These operators record no gradient: an input that wants one is refused
    rather than cut off silently."""
    for t in tensors:
        if t is not None and t.requires_grad and torch.is_grad_enabled():
            raise RuntimeError(f"{what} records no gradient: call it under torch.no_grad(), or detach its inputs")


def overlaps(t: torch.Tensor) -> bool:
    """Whether elements of t may share memory (an expanded view, say)."""
    if t.is_contiguous():
        return False
    reach = 0  # of the elements along the dimensions of smaller strides
    for st, n in sorted((abs(s), n) for s, n in zip(t.stride(), t.shape) if n > 1):
        if st <= reach:
            return True
        reach += st * (n - 1)
    return False


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
    tensors to those of q and k.  inplace: into q and k themselves.

    Returns q' (and k', as a pair, when k is given)."""
    no_grad_needed("apply_rotary", q, k)
    device = X.require_gpu(q, k, positions, table.inv_freq)
    if q.dim() not in (3, 4):
        raise ValueError(f"q must be (tokens, heads, d) or (batch, heads, tokens, d), got {tuple(q.shape)}")
    dt = X.dtype_code(q.dtype, "q", allow_fp8=False)
    d = q.shape[-1]
    rot = check_table(table, d, layout, device)
    xs = [q] if k is None else [q, k]
    if k is not None:
        same = (0, 2) if q.dim() == 3 else (0, 2, 3)
        if k.dim() != q.dim() or any(k.shape[i] != q.shape[i] for i in same):
            raise ValueError(f"k {tuple(k.shape)} does not match q {tuple(q.shape)}")
        if k.dtype != q.dtype:
            raise TypeError(f"q and k must share a dtype ({q.dtype}, {k.dtype})")
    tokens = q.shape[0] if q.dim() == 3 else q.shape[2]
    batch = 1 if q.dim() == 3 else q.shape[0]
    if tuple(positions.shape) not in ((tokens,), (batch, tokens)):
        raise ValueError(f"positions must be ({tokens},) or ({batch}, {tokens}), got {tuple(positions.shape)}")
    positions = check_positions(positions, device)
    ys, ptrs, heads = [], [], []
    for x in xs:
        if inplace:
            if (x.stride(-1) != 1 and d > 1) or overlaps(x):
                raise ValueError("in place, the last dimension must be contiguous and no elements may share memory")
            y = x
        else:
            if x.stride(-1) != 1:
                x = x.contiguous()
            y = torch.empty_like(x)
            if y.stride(-1) != 1:
                y = torch.empty(x.shape, dtype=x.dtype, device=device)
        ys.append(y)
        xst, yst = x.stride(), y.stride()
        if len(xst) == 3:  # (tokens, heads, d)
            xst, yst = (0, xst[1], xst[0]), (0, yst[1], yst[0])
        ptrs.append((x.data_ptr(), y.data_ptr(), *xst[:3], *yst[:3]))
        heads.append(x.shape[1])
    if k is None:
        ptrs.append((None, None, 0, 0, 0, 0, 0, 0))
        heads.append(0)
    elif inplace and q.data_ptr() == k.data_ptr() and q.numel() and k.numel():
        raise ValueError("in place, q and k must be different tensors")
    p = N.OcRotaryParams(
        *zip(*ptrs), tuple(heads), dt, batch, tokens, d, rot, layout == "interleaved", backward,
        positions.dtype == torch.int64, positions.data_ptr(),
        positions.stride(0) if positions.dim() == 2 and batch > 1 else 0, table.inv_freq.data_ptr(), table.scale)
    X.launch("oc_apply_rotary", p, device)
    return ys[0] if k is None else tuple(ys)
