"""Attention whose scores are changed before the softmax: capped by a tanh,
biased by distance, in a window, behind a prefix, between documents; for one
new token per sequence over a paged cache, and for whole prompts.

The reference attends by q.k / sqrt(d) and a causal mask alone
(paged_eviction.py:323-445, eval/perplexity_eval.py:399-545); evicted tiles are
left out here as there.

For the query at place i and the key at place j, in this order:

    z = scale * q.k
    z = softcap * tanh(z / softcap)         softcap > 0
    z = z - alibi_slopes[head] * |i - j|    alibi_slopes
    seen: (j <= i and (window <= 0 or i - j < window)) or j < prefix_lens[b],
          of the same document, in no evicted tile

A query that sees nothing gets zeros, and keys and values that are not seen
have no effect whatever they hold.
"""

from __future__ import annotations

from typing import Optional

import torch

from ._ops import number, ops


def _optional(scale: Optional[float]) -> Optional[float]:
    return None if scale is None else number(scale, "scale")


def attend_paged(q: torch.Tensor, k_cache: torch.Tensor, v_cache: torch.Tensor, block_tables: torch.Tensor,
                 context_lens: torch.Tensor, *, scale: Optional[float] = None, softcap: float = 0.0,
                 alibi_slopes: Optional[torch.Tensor] = None, window: int = 0,
                 prefix_lens: Optional[torch.Tensor] = None, k_scale: float = 1.0, v_scale: float = 1.0,
                 evict_mask: Optional[torch.Tensor] = None, num_splits: Optional[int] = None, sync: bool = True,
                 out: Optional[torch.Tensor] = None, portable: bool = False) -> torch.Tensor:
    """One new token per sequence, the last cached one, over its pages
    (oc_attend_paged): (num_seqs, num_heads, head_dim) in q's type.

    q (num_seqs, num_heads, head_dim) in float32, float16 or bfloat16; caches
    (num_blocks, num_kv_heads, block_size, head_dim) in q's type, or
    float8_e4m3fn, whose values count k_scale and v_scale times; head_dim a
    multiple of 8 up to 512, block_size a power of two.  block_tables int32
    (num_seqs, max_blocks); context_lens int32 (num_seqs,), the query's token
    included, clamped to 0 .. max_blocks * block_size.  evict_mask: bool or
    uint8 (num_seqs, num_kv_heads, tiles), nonzero = the complete 64-token tile
    is left out.  num_splits: parts of each sequence (chosen by default, 1024 at
    most).  out: may be q, but share no other memory with the inputs.  The
    score changes are this module's.  portable: the kernel that takes every
    shape, whatever the shape.

    With sync, a block id outside [0, num_blocks) where a seen token needs one
    raises ValueError; without (as in a captured graph), such tokens are left
    out."""
    return ops().attend_paged(q, k_cache, v_cache, block_tables, context_lens, _optional(scale), number(softcap, "softcap"),
                              alibi_slopes, window, prefix_lens, number(k_scale, "k_scale"), number(v_scale, "v_scale"),
                              evict_mask, num_splits, sync, out, portable)


def attend_prompt(q: torch.Tensor, k: torch.Tensor, v: torch.Tensor, *, scale: Optional[float] = None,
                  softcap: float = 0.0, alibi_slopes: Optional[torch.Tensor] = None, window: int = 0,
                  prefix_lens: Optional[torch.Tensor] = None, documents: Optional[torch.Tensor] = None,
                  evict_mask: Optional[torch.Tensor] = None) -> torch.Tensor:
    """Attention of whole prompts (oc_attend_prompt): (batch, num_heads, q_len,
    head_dim) in q's type, for q of that shape over k, v (batch, num_kv_heads,
    kv_len, head_dim) in float32, float16 or bfloat16, head_dim 64 or 128.

    Query s is at place s + kv_len - q_len.  documents: int32 (batch, kv_len)
    or (kv_len,), the document of every place: others' keys are not seen, and a
    negative one is seen by no one and sees nothing (padding).  evict_mask:
    bool or uint8 (batch, num_kv_heads, tiles), nonzero = the complete 64-token
    tile is left out.  The score changes are this module's."""
    return ops().attend_prompt(q, k, v, _optional(scale), number(softcap, "softcap"), alibi_slopes, window, prefix_lens,
                               documents, evict_mask)
