"""Operators on a paged cache: new tokens into their pages, and forks, ends,
room and evicted tiles of sequences in the block tables.

A cache is (num_blocks, num_kv_heads, block_size, head_dim), K and V alike, as
`fused_orthocache_attention_paged` takes it (paged_eviction.py:323-445); the
reference fills it by hand and has no operator that changes a block table.
"""

from __future__ import annotations

from dataclasses import dataclass
from typing import Optional, Tuple, Union

import torch

from . import _native as N
from ._ops import number, ops
from .rotary import RotaryTable


class OutOfPages(RuntimeError):
    """A call needs more free blocks than the cache has."""


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
    (`fork_pages` sees to that), and k_cache and v_cache are different memory.
    With sync, a block id outside [0, num_blocks) and a table too short for a
    token raise ValueError; without (as in a captured graph), such tokens are
    left out."""
    freq, scale = (None, 1.0) if table is None else (table.inv_freq, table.scale)
    return ops().append_paged(k, v, k_cache, v_cache, block_tables, context_lens, q, cu_seqlens, positions, freq, scale,
                              layout, number(k_scale, "k_scale"), number(v_scale, "v_scale"), sync)


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


def _parts(out: Optional[PageTables]):
    return None if out is None else (out.block_tables, out.context_lens, out.ref_counts, out.status)


def fork_pages(k_cache: torch.Tensor, v_cache: torch.Tensor, block_tables: torch.Tensor, context_lens: torch.Tensor,
               ref_counts: torch.Tensor, *, parents: Optional[torch.Tensor] = None,
               new_tokens: Union[int, torch.Tensor] = 0, max_blocks: Optional[int] = None, sync: bool = True,
               out: Optional[PageTables] = None) -> PageTables:
    """New tables in which sequence i continues sequence parents[i]
    (oc_fork_pages): beams reordered, prompts shared, sequences ended and
    started, and room for their next tokens.

    parents: int32 (num_children,), -1 for an empty sequence without blocks (a
    later call can go on with it); a sequence that is no one's parent ends.
    None: every sequence goes on.  new_tokens: how many tokens each child shall
    have room for past its own (a number, or int32 (num_children,)).  Children share their parent's full blocks; a last block
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
    each, every = (new_tokens, 0) if isinstance(new_tokens, torch.Tensor) else (None, new_tokens)
    res = PageTables(*ops().fork_pages(k_cache, v_cache, block_tables, context_lens, ref_counts, parents, each, every,
                                       max_blocks, _parts(out)))
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
    *tables, tile_map = ops().evict_pages(block_tables, context_lens, ref_counts, evict_mask, block_size, _parts(out))
    res = PageTables(*tables)
    return (res.check() if sync else res), tile_map
