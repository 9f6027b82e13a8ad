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

import ctypes
import math
from typing import Optional

import torch

from . import _launch as X
from . import _native as N
from .paged_cache import cache_scales, check_caches, index_tensor, tile_flags
from .rotary import no_grad_needed


def _mods(scale, softcap, slopes, window, prefix, evict, batch, hq, hkv, d, device):
    """The score changes as the library's block, and the tensors it points to."""
    scale = 1.0 / math.sqrt(d) if scale is None else float(scale)
    if not math.isfinite(scale):
        raise ValueError(f"scale {scale} must be finite")
    if not (softcap >= 0 and math.isfinite(softcap)):
        raise ValueError(f"softcap {softcap} must be 0 (none) or positive")
    if window < 0:
        raise ValueError(f"window {window} must be 0 (none) or positive")
    ptrs = [None, None, None]
    sb = sh = cols = 0
    if slopes is not None:
        if slopes.dtype != torch.float32 or slopes.shape != (hq,) or slopes.device != device:
            raise ValueError(f"alibi_slopes must be float32 ({hq},) on {device}")
        slopes = slopes.contiguous()
        ptrs[0] = slopes.data_ptr()
    if prefix is not None:
        prefix = index_tensor(prefix, (batch,), "prefix_lens", device)
        ptrs[1] = prefix.data_ptr()
    if evict is not None:
        evict = tile_flags(evict, batch, hkv, device)
        ptrs[2], (sb, sh), cols = evict.data_ptr(), evict.stride()[:2], evict.shape[2]
    return (N.OcScoreMods(scale, softcap, *ptrs, sb, sh, cols, min(int(window), 2 ** 31 - 1)), (slopes, prefix, evict))


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
    is left out.  num_splits: parts of each sequence (chosen by default).  The
    score changes are this module's.  portable: the kernel that takes every
    shape, whatever the shape.

    With sync, a block id outside [0, num_blocks) where a seen token needs one
    raises ValueError; without, such tokens are left out."""
    no_grad_needed("attend_paged", q, k_cache, v_cache, alibi_slopes)
    device = X.require_gpu(q, k_cache, v_cache, block_tables, context_lens, alibi_slopes, prefix_lens, evict_mask)
    check_caches(k_cache, v_cache, (4,))
    nb, hkv, bs, d = k_cache.shape
    if q.dim() != 3 or q.shape[2] != d:
        raise ValueError(f"q must be (num_seqs, heads, {d}), got {tuple(q.shape)}")
    n, hq, _ = q.shape
    if hkv == 0 or hq % hkv:
        raise ValueError(f"{hq} query heads on {hkv} kv heads")
    dt = X.dtype_code(q.dtype, "q", allow_fp8=False)
    if k_cache.dtype not in (q.dtype, torch.float8_e4m3fn):
        raise TypeError(f"the cache must have q's dtype ({q.dtype}) or float8_e4m3fn, got {k_cache.dtype}")
    cache_scales(k_cache.dtype, k_scale, v_scale)
    block_tables = index_tensor(block_tables, (n, -1), "block_tables", device)
    context_lens = index_tensor(context_lens, (n,), "context_lens", device)
    if num_splits is not None and num_splits < 1:
        raise ValueError(f"num_splits ({num_splits}) must be positive")
    if out is None:
        out = torch.empty((n, hq, d), dtype=q.dtype, device=device)
    elif out.shape != (n, hq, d) or out.dtype != q.dtype or out.device != device or (d > 1 and out.stride(2) != 1):
        raise ValueError(f"out must be a ({n}, {hq}, {d}) {q.dtype} tensor on {device} with a contiguous last dim")
    q = X.ready16(q)
    mods, held = _mods(scale, softcap, alibi_slopes, window, prefix_lens, evict_mask, n, hq, hkv, d, device)
    flag = torch.zeros(1, dtype=torch.int32, device=device) if sync else None
    qs, ks, vs, os = q.stride(), k_cache.stride(), v_cache.stride(), out.stride()
    p = N.OcAttendPagedParams(
        q.data_ptr(), qs[0], qs[1], k_cache.data_ptr(), v_cache.data_ptr(), ks[0], ks[1], ks[2], vs[0], vs[1], vs[2],
        block_tables.data_ptr(), block_tables.stride(0), nb, context_lens.data_ptr(), block_tables.shape[1], bs, dt,
        X.dtype_code(k_cache.dtype, "cache"), n, hq, hkv, d, k_scale, v_scale, mods, num_splits or 0, bool(portable),
        out.data_ptr(), os[0], os[1], X._ptr(flag))
    need = N.lib().oc_attend_paged_workspace_size(ctypes.byref(p))
    if need:
        # a buffer of the call's own: two captured graphs replayed at once share nothing
        ws = torch.empty(need, dtype=torch.uint8, device=device)
        p.workspace, p.workspace_bytes = ws.data_ptr(), need
    X.launch("oc_attend_paged", p, device)
    if flag is not None and int(flag.item()):
        raise ValueError("block_tables holds a block id outside [0, num_blocks)")
    return out


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
    no_grad_needed("attend_prompt", q, k, v, alibi_slopes)
    device = X.check_prefill(q, k, v)
    X.require_gpu(q, alibi_slopes, prefix_lens, documents, evict_mask)
    B, hq, sq, d = q.shape
    hkv, skv = k.shape[1], k.shape[2]
    dt = X.dtype_code(q.dtype, "q", allow_fp8=False)
    if d not in (64, 128):
        raise NotImplementedError(f"head_dim {d} is not supported (64 or 128)")
    mods, held = _mods(scale, softcap, alibi_slopes, window, prefix_lens, evict_mask, B, hq, hkv, d, device)
    docs, docs_sb = None, 0
    if documents is not None:
        if documents.dim() == 1:
            documents = documents.unsqueeze(0).expand(B, -1)
        documents = index_tensor(documents, (B, skv), "documents", device)
        docs, docs_sb = documents.data_ptr(), documents.stride(0)
    q, k, v = X.ready16(q), X.ready16(k, 2), X.ready16(v, 2)
    out = torch.empty((B, hq, sq, d), dtype=q.dtype, device=device)
    p = N.OcAttendPromptParams(
        q.data_ptr(), *q.stride()[:3], k.data_ptr(), *k.stride()[:3], v.data_ptr(), *v.stride()[:3], out.data_ptr(),
        *out.stride()[:3], dt, B, hq, hkv, sq, skv, d, docs, docs_sb, mods)
    if docs is not None:
        need = N.lib().oc_attend_prompt_workspace_size(ctypes.byref(p))
        ws = torch.empty(need, dtype=torch.uint8, device=device)
        p.workspace, p.workspace_bytes = ws.data_ptr(), need
    X.launch("oc_attend_prompt", p, device)
    return out
