"""Operators on a paged cache: new tokens into their pages, and forks, ends,
room and evicted tiles of sequences in the block tables.

A cache is (num_blocks, num_kv_heads, block_size, head_dim), K and V alike, as
`fused_orthocache_attention_paged` takes it (paged_eviction.py:323-445); the
reference fills it by hand and has no operator that changes a block table.
"""

from __future__ import annotations

import ctypes
from dataclasses import dataclass
from typing import Optional, Tuple, Union

import torch

from . import _launch as X
from . import _native as N
from .rotary import RotaryTable, check_positions, check_table, no_grad_needed, overlaps

MAX_SEQS = 4096  # sequences and children of a fork


class OutOfPages(RuntimeError):
    """A call needs more free blocks than the cache has."""


def index_tensor(t: torch.Tensor, shape: Tuple[int, ...], what: str, device: torch.device) -> torch.Tensor:
    """An int32 tensor of the shape (-1: any size) with a contiguous last dimension."""
    if t.dtype != torch.int32:
        raise TypeError(f"{what} must be int32, got {t.dtype}")
    if t.device != device:
        raise RuntimeError(f"orthocache_gpu: {what} on {t.device}, the rest on {device}")
    got = t.shape
    if got != shape:
        if len(got) != len(shape) or any(n not in (-1, m) for n, m in zip(shape, got)):
            raise ValueError(f"{what} must be {shape}, got {tuple(got)}")
    return t if t.is_contiguous() or got[-1] <= 1 or t.stride(-1) == 1 else t.contiguous()


def check_caches(k_cache: torch.Tensor, v_cache: torch.Tensor, dims: Tuple[int, ...]) -> None:
    if k_cache.dim() not in dims or v_cache.shape != k_cache.shape:
        raise ValueError(f"k_cache and v_cache must be {' or '.join(str(n) + '-D' for n in dims)} of one shape, got "
                         f"{tuple(k_cache.shape)} and {tuple(v_cache.shape)}")
    if k_cache.dtype != v_cache.dtype:
        raise TypeError(f"k_cache and v_cache must share a dtype ({k_cache.dtype}, {v_cache.dtype})")
    X.dtype_code(k_cache.dtype, "cache")
    bs = k_cache.shape[-2]
    if bs < 1 or bs & (bs - 1):
        raise ValueError(f"block_size ({bs}) must be a power of 2")
    if k_cache.shape[-1] > 1 and (k_cache.stride(-1) != 1 or v_cache.stride(-1) != 1):
        raise ValueError("cache rows must be contiguous along head_dim")


def written_caches(k_cache: torch.Tensor, v_cache: torch.Tensor) -> None:
    if overlaps(k_cache) or overlaps(v_cache):
        raise ValueError("elements of a cache that is written may not share memory")


def cache_scales(dtype: torch.dtype, *scales: float) -> None:
    for s in scales:
        if isinstance(s, torch.Tensor):
            raise TypeError("k_scale and v_scale are numbers here")
        if not (s > 0 and s < float("inf")):
            raise ValueError(f"scales must be positive and finite, got {s}")
        if s != 1.0 and dtype != torch.float8_e4m3fn:
            raise ValueError(f"k_scale and v_scale are for float8_e4m3fn caches, not {dtype}")


def append_paged(k: torch.Tensor, v: torch.Tensor, k_cache: torch.Tensor, v_cache: torch.Tensor,
                 block_tables: torch.Tensor, context_lens: torch.Tensor, *, q: Optional[torch.Tensor] = None,
                 cu_seqlens: Optional[torch.Tensor] = None, positions: Optional[torch.Tensor] = None,
                 table: Optional[RotaryTable] = None, layout: str = "half", k_scale: float = 1.0,
                 v_scale: float = 1.0, sync: bool = True) -> Optional[torch.Tensor]:
    """New tokens of every sequence: their keys turned by their positions and
    written, with their values, to the tokens' slots in the cache
    (oc_append_paged); with q the queries turned alike, which it returns.

    k, v (and q): (tokens, heads, head_dim) in float32, float16 or bfloat16.
    Rows cu_seqlens[b] .. cu_seqlens[b + 1) (int32, (num_seqs + 1,), not
    decreasing) are sequence b's; without it row b is.  context_lens: int32
    (num_seqs,) tokens that were cached before; they are not changed here.  A
    sequence of negative length takes part without tokens, and rows outside
    every sequence are padding: neither writes to the cache, and their turned
    queries are zeros.  positions: int32 or int64 (tokens,), by default the
    tokens' places in their sequences (they differ once tiles were evicted).
    table None: nothing is turned.  The cache may have another type; float8
    takes x / k_scale and x / v_scale, at most 448 in size.

    Sequences of one call must not share the blocks that they write
    (`fork_pages` sees to that).  With sync, a block id outside [0, num_blocks)
    and a table too short for a token raise ValueError; without, such tokens
    are left out."""
    no_grad_needed("append_paged", q, k, v)
    device = X.require_gpu(k, v, k_cache, v_cache, block_tables, context_lens, q)
    check_caches(k_cache, v_cache, (4,))
    written_caches(k_cache, v_cache)
    nb, hkv, bs, d = k_cache.shape
    tokens = k.shape[0]
    if k.shape != (tokens, hkv, d) or v.shape != k.shape:
        raise ValueError(f"k and v must be (tokens, {hkv}, {d}), got {tuple(k.shape)} and {tuple(v.shape)}")
    if q is not None and (q.dim() != 3 or q.shape[0] != tokens or q.shape[2] != d):
        raise ValueError(f"q must be ({tokens}, heads, {d}), got {tuple(q.shape)}")
    if v.dtype != k.dtype or (q is not None and q.dtype != k.dtype):
        raise TypeError("q, k and v must share a dtype")
    cache_scales(k_cache.dtype, k_scale, v_scale)
    n = context_lens.shape[0] if context_lens.dim() == 1 else -1
    context_lens = index_tensor(context_lens, (n,), "context_lens", device)
    block_tables = index_tensor(block_tables, (n, -1), "block_tables", device)
    if cu_seqlens is not None:
        cu_seqlens = index_tensor(cu_seqlens, (n + 1,), "cu_seqlens", device)
    elif tokens != n:
        raise ValueError(f"{tokens} tokens for {n} sequences need cu_seqlens")
    rot = check_table(table, d, layout, device)
    dt = X.dtype_code(k.dtype, "k", allow_fp8=False)
    if positions is not None:
        if positions.shape != (tokens,):
            raise ValueError(f"positions must be ({tokens},), got {tuple(positions.shape)}")
        positions = check_positions(positions, device)
    if k.stride(-1) != 1:
        k = k.contiguous()
    if v.stride(-1) != 1:
        v = v.contiguous()
    out, qp, op, hq = None, None, None, 0
    qs = os = (0, 0)
    if q is not None:
        if q.stride(-1) != 1:
            q = q.contiguous()
        out = torch.empty(q.shape, dtype=q.dtype, device=device)
        if n == 0:
            out.zero_()
        qp, op, hq, qs, os = q.data_ptr(), out.data_ptr(), q.shape[1], q.stride(), out.stride()
    ks, vs, kcs, vcs = k.stride(), v.stride(), k_cache.stride(), v_cache.stride()
    flag = torch.zeros(1, dtype=torch.int32, device=device) if sync else None
    p = N.OcAppendParams(
        qp, k.data_ptr(), v.data_ptr(), op, qs[0], qs[1], ks[0], ks[1], vs[0], vs[1], os[0], os[1],
        k_cache.data_ptr(), v_cache.data_ptr(), kcs[0], kcs[1], kcs[2], vcs[0], vcs[1], vcs[2],
        dt, X.dtype_code(k_cache.dtype, "cache"), tokens, n, hq, hkv, d, rot, bs, block_tables.shape[1], nb,
        block_tables.data_ptr(), block_tables.stride(0), context_lens.data_ptr(), X._ptr(cu_seqlens), X._ptr(positions),
        positions is not None and positions.dtype == torch.int64, layout == "interleaved",
        None if table is None else table.inv_freq.data_ptr(), 1.0 if table is None else table.scale, k_scale, v_scale,
        X._ptr(flag))
    X.launch("oc_append_paged", p, device)
    if flag is not None and int(flag.item()):
        raise ValueError("block_tables holds no block in [0, num_blocks) for some of the tokens")
    return out


@dataclass
class PageTables:
    """Block tables int32 (num_seqs, max_blocks), -1 past a sequence's blocks;
    context_lens int32 (num_seqs,); ref_counts int32 (num_blocks,), the
    holders of every block; status int32 (1,), 0 where the call was carried
    out (bits _native.OC_PAGES_*)."""
    block_tables: torch.Tensor
    context_lens: torch.Tensor
    ref_counts: torch.Tensor
    status: torch.Tensor

    def check(self) -> "PageTables":
        """Waits for the call and raises what its status says."""
        s = int(self.status.item())
        if s & N.OC_PAGES_BAD_PARENT:
            raise ValueError("parents must be -1 or a sequence's number")
        if s & N.OC_PAGES_BAD_BLOCK:
            raise ValueError("block_tables holds a block id outside [0, num_blocks) among a sequence's blocks")
        if s & N.OC_PAGES_TOO_LONG:
            raise ValueError("a sequence needs more blocks than its table has columns")
        if s & N.OC_PAGES_NO_ROOM:
            raise OutOfPages("the cache has fewer free blocks than the call needs")
        return self


def _out_tables(out: Optional[PageTables], rows: int, cols: int, blocks: int, device: torch.device, *inputs) -> PageTables:
    if out is None:
        # one allocation: the tables, the lengths, the counts and the status
        flat = torch.empty(rows * cols + rows + blocks + 1, dtype=torch.int32, device=device)
        t, l, r, s = flat.split((rows * cols, rows, blocks, 1))
        return PageTables(t.view(rows, cols), l, r, s)
    for t, shape, what in ((out.block_tables, (rows, cols), "block_tables"), (out.context_lens, (rows,), "context_lens"),
                           (out.ref_counts, (blocks,), "ref_counts"), (out.status, (1,), "status")):
        if t.dtype != torch.int32 or tuple(t.shape) != shape or t.device != device or not t.is_contiguous():
            raise ValueError(f"out.{what} must be a contiguous int32 {shape} tensor on {device}")
        lo, hi = t.data_ptr(), t.data_ptr() + 4 * t.numel()
        for i in inputs:
            if i is not None and i.numel() and t.numel():
                reach = i.element_size() * (1 + sum((m - 1) * s for m, s in zip(i.shape, i.stride())))
                if i.data_ptr() < hi and lo < i.data_ptr() + reach:
                    raise ValueError(f"out.{what} overlaps an input: the old tables must stay")
    return out


def fork_pages(k_cache: torch.Tensor, v_cache: torch.Tensor, block_tables: torch.Tensor, context_lens: torch.Tensor,
               ref_counts: torch.Tensor, *, parents: Optional[torch.Tensor] = None,
               new_tokens: Union[int, torch.Tensor] = 0, max_blocks: Optional[int] = None, sync: bool = True,
               out: Optional[PageTables] = None) -> PageTables:
    """New tables in which sequence i continues sequence parents[i]
    (oc_fork_pages): beams reordered, prompts shared, sequences ended and
    started, and room for their next tokens.

    parents: int32 (num_children,), -1 for an empty sequence without blocks (a
    later call can go on with it); a sequence that is no one's parent ends.  None: every sequence goes on.  new_tokens: how
    many tokens each child shall have room for past its own (a number, or int32
    (num_children,)).  Children share their parent's full blocks; a last block
    that is not full stays with the first child if no one else holds it, and
    the others get a copy of its tokens, in every layer: caches are
    (num_blocks, num_kv_heads, block_size, head_dim), or with layers in front.

    A child's row holds exactly the blocks that its tokens and new_tokens need,
    then -1; blocks that an earlier call made room with and that hold no token
    are given back.  Fresh blocks are those of ref_counts 0 before the call,
    lowest first, in the order of the children (what the call frees is not
    used by it).  max_blocks: columns of the new tables (the old ones' by
    default).  The inputs stay as they are; out takes the results in tensors of
    the caller's, for captured graphs.

    With sync, raises OutOfPages, or ValueError for a parent that is no
    sequence's number, a block id outside the cache or a table too narrow;
    without, the result's status says so.  Then nothing is copied and the new
    tables are empty."""
    device = X.require_gpu(k_cache, v_cache, block_tables, context_lens, ref_counts, parents)
    check_caches(k_cache, v_cache, (4, 5))
    written_caches(k_cache, v_cache)
    if k_cache.dim() == 4:
        k_cache, v_cache = k_cache.unsqueeze(0), v_cache.unsqueeze(0)
    layers, nb, hkv, bs, d = k_cache.shape
    n = context_lens.shape[0] if context_lens.dim() == 1 else -1
    context_lens = index_tensor(context_lens, (n,), "context_lens", device)
    block_tables = index_tensor(block_tables, (n, -1), "block_tables", device)
    ref_counts = index_tensor(ref_counts, (nb,), "ref_counts", device)
    children = n
    if parents is not None:
        parents = index_tensor(parents, (-1,), "parents", device)
        children = parents.shape[0]
    if max(n, children) > MAX_SEQS:
        raise NotImplementedError(f"at most {MAX_SEQS} sequences and children, got {n} and {children}")
    if isinstance(new_tokens, torch.Tensor):
        new_tokens = index_tensor(new_tokens, (children,), "new_tokens", device)
    else:
        if new_tokens < 0:
            raise ValueError(f"new_tokens {new_tokens} is negative")
        new_tokens = None if new_tokens == 0 else torch.full((children,), int(new_tokens), dtype=torch.int32, device=device)
    cols = block_tables.shape[1] if max_blocks is None else int(max_blocks)
    if cols < 0:
        raise ValueError(f"max_blocks {cols} is negative")
    res = _out_tables(out, children, cols, nb, device, block_tables, context_lens, ref_counts, parents, new_tokens)
    ks, vs = k_cache.stride(), v_cache.stride()
    p = N.OcForkParams(
        k_cache.data_ptr(), v_cache.data_ptr(), ks[0], ks[1], ks[2], ks[3], vs[0], vs[1], vs[2], vs[3],
        X.dtype_code(k_cache.dtype, "cache"), layers if nb else 0, hkv, d, bs, n, children, block_tables.shape[1], cols, nb,
        block_tables.data_ptr(), block_tables.stride(0), context_lens.data_ptr(), ref_counts.data_ptr(), X._ptr(parents),
        X._ptr(new_tokens), res.block_tables.data_ptr(), res.block_tables.stride(0), res.context_lens.data_ptr(),
        res.ref_counts.data_ptr(), res.status.data_ptr())
    need = N.lib().oc_fork_pages_workspace_size(ctypes.byref(p))
    ws = torch.empty(need, dtype=torch.uint8, device=device)
    p.workspace, p.workspace_bytes = ws.data_ptr(), need
    X.launch("oc_fork_pages", p, device)
    return res.check() if sync else res


def evict_pages(block_tables: torch.Tensor, context_lens: torch.Tensor, ref_counts: torch.Tensor,
                evict_mask: torch.Tensor, *, block_size: int, sync: bool = True, out: Optional[PageTables] = None
                ) -> Tuple[PageTables, torch.Tensor]:
    """New tables without the evicted 64-token tiles (oc_evict_pages): the
    complete tiles that every kv head evicts leave their sequences, the others
    close up in order, and the blocks lose a holder.

    evict_mask: bool or uint8 (num_seqs, num_kv_heads, tiles) or (num_seqs,
    tiles), nonzero = evicted; tiles past its columns stay, and a partial last
    tile does.  block_size divides 64.  Blocks past a sequence's tokens are
    given back.  The inputs stay as they are (out: as in fork_pages).

    Returns the tables and the tile map, int32 (num_seqs, ceil(max_blocks *
    block_size / 64)): the old tile of every new one, -1 past the last -- what
    moves a score cache's columns along.  Places in the cache are no longer
    positions then: append_paged takes the positions of the next tokens, while
    the window, the prefix and the distance of attend_paged count cached
    tokens.  With sync, a block id outside the cache raises ValueError."""
    device = X.require_gpu(block_tables, context_lens, ref_counts, evict_mask)
    n = context_lens.shape[0] if context_lens.dim() == 1 else -1
    context_lens = index_tensor(context_lens, (n,), "context_lens", device)
    block_tables = index_tensor(block_tables, (n, -1), "block_tables", device)
    ref_counts = index_tensor(ref_counts, (-1,), "ref_counts", device)
    if block_size < 1 or X.TILE_SIZE % block_size:
        raise ValueError(f"block_size ({block_size}) must divide a tile of {X.TILE_SIZE} tokens")
    evict_mask = tile_flags(evict_mask.unsqueeze(1) if evict_mask.dim() == 2 else evict_mask, n, -1, device)
    cols, nb = block_tables.shape[1], ref_counts.shape[0]
    tiles = -(-cols * block_size // X.TILE_SIZE)
    res = _out_tables(out, n, cols, nb, device, block_tables, context_lens, ref_counts, evict_mask)
    tile_map = torch.empty((n, tiles), dtype=torch.int32, device=device)
    p = N.OcEvictParams(
        n, evict_mask.shape[1], block_size, cols, nb, block_tables.data_ptr(), block_tables.stride(0), context_lens.data_ptr(),
        ref_counts.data_ptr(), evict_mask.data_ptr(), evict_mask.stride(0), evict_mask.stride(1), evict_mask.shape[2], tiles,
        res.block_tables.data_ptr(), res.block_tables.stride(0), res.context_lens.data_ptr(), res.ref_counts.data_ptr(),
        tile_map.data_ptr(), res.status.data_ptr())
    X.launch("oc_evict_pages", p, device)
    return (res.check() if sync else res), tile_map


def tile_flags(mask: torch.Tensor, batch: int, heads: int, device: torch.device) -> torch.Tensor:
    """A (batch, heads, tiles) bool or uint8 mask with a contiguous last dimension (heads -1: any, at least one)."""
    if mask.dtype not in (torch.bool, torch.uint8):
        raise TypeError(f"evict_mask must be bool or uint8, got {mask.dtype}")
    if mask.device != device:
        raise RuntimeError(f"orthocache_gpu: evict_mask on {mask.device}, the rest on {device}")
    if mask.dim() != 3 or mask.shape[0] != batch or (mask.shape[1] != heads if heads >= 0 else mask.shape[1] < 1):
        raise ValueError(f"evict_mask must be ({batch}, {heads if heads >= 0 else 'heads'}, tiles), got {tuple(mask.shape)}")
    return mask if mask.shape[2] <= 1 or mask.stride(2) == 1 else mask.contiguous()
