"""CPU tests of the paged operators' boundary: exported symbols, struct layout, and what the library and the
entry points refuse before any launch."""

import ctypes
import os
import re

import pytest
import torch

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
HEADER = os.path.join(ROOT, "include", "orthocache_paged.h")


def test_symbols_and_layout():
    from orthocache_gpu import _native as N
    text = re.sub(r"/\*.*?\*/", "", open(HEADER).read(), flags=re.S)
    names = sorted(set(re.findall(r"\b(oc_[a-z0-9_]+)\s*\(", text)))
    assert len(names) == 10
    for n in names:
        assert hasattr(N.lib(), n) and n in N.SIGNATURES, n
    sizes = (ctypes.c_size_t * 6)()
    N.lib().oc_paged_params_bytes(sizes)
    assert list(sizes) == [ctypes.sizeof(s) for s in (N.OcRotaryParams, N.OcAppendParams, N.OcAttendPagedParams,
                                                      N.OcAttendPromptParams, N.OcForkParams, N.OcEvictParams)]


def _refused(fn, p, code, text):
    from orthocache_gpu import _native as N
    assert getattr(N.lib(), fn)(ctypes.byref(p), None) == code, N.lib().oc_last_error()
    assert text in N.lib().oc_last_error(), N.lib().oc_last_error()


def test_rotary_and_append():
    from orthocache_gpu import _native as N
    p = N.OcRotaryParams()
    p.dtype, p.batch, p.tokens, p.head_dim, p.rotary_dim, p.heads[0] = N.OC_BF16, 1, 4, 64, 66, 2
    _refused("oc_apply_rotary", p, N.OC_ERR_INVALID, b"rotary_dim")
    p.rotary_dim = 64
    _refused("oc_apply_rotary", p, N.OC_ERR_INVALID, b"NULL")
    p.head_dim = 1024
    _refused("oc_apply_rotary", p, N.OC_ERR_UNSUPPORTED, b"head_dim")
    p.head_dim, p.dtype = 64, N.OC_FP8_E4M3FN
    _refused("oc_apply_rotary", p, N.OC_ERR_INVALID, b"dtype")
    p.dtype, p.tokens = N.OC_BF16, 0
    assert N.lib().oc_apply_rotary(ctypes.byref(p), None) == N.OC_OK
    a = N.OcAppendParams()
    a.dtype, a.cache_dtype, a.tokens, a.num_seqs, a.num_kv_heads, a.head_dim, a.block_size = N.OC_BF16, N.OC_BF16, 3, 2, 1, 64, 16
    _refused("oc_append_paged", a, N.OC_ERR_INVALID, b"cu_seqlens")
    a.num_seqs = 3
    _refused("oc_append_paged", a, N.OC_ERR_INVALID, b"NULL")
    a.block_size = 24
    _refused("oc_append_paged", a, N.OC_ERR_INVALID, b"power of two")
    a.block_size, a.cache_dtype = 16, 9
    _refused("oc_append_paged", a, N.OC_ERR_INVALID, b"cache dtype")


def test_attention():
    from orthocache_gpu import _native as N
    p = N.OcAttendPagedParams()
    p.dtype, p.cache_dtype, p.head_dim, p.block_size = N.OC_BF16, N.OC_F16, 64, 16
    p.num_seqs, p.num_q_heads, p.num_kv_heads = 1, 4, 2
    _refused("oc_attend_paged", p, N.OC_ERR_UNSUPPORTED, b"cache dtype")
    p.cache_dtype, p.head_dim = N.OC_BF16, 60
    _refused("oc_attend_paged", p, N.OC_ERR_UNSUPPORTED, b"head_dim")
    p.head_dim, p.num_q_heads = 64, 5
    _refused("oc_attend_paged", p, N.OC_ERR_INVALID, b"query heads")
    p.num_q_heads, p.max_blocks = 4, 1 << 21
    _refused("oc_attend_paged", p, N.OC_ERR_UNSUPPORTED, b"2^24")
    p.max_blocks, p.mods.softcap = 4, float("nan")
    _refused("oc_attend_paged", p, N.OC_ERR_INVALID, b"softcap")
    p.mods.softcap, p.mods.window = 0.0, -1
    _refused("oc_attend_paged", p, N.OC_ERR_INVALID, b"window")
    p.mods.window = 0
    _refused("oc_attend_paged", p, N.OC_ERR_INVALID, b"NULL")
    r = N.OcAttendPromptParams()
    r.dtype, r.batch, r.num_q_heads, r.num_kv_heads, r.q_len, r.kv_len, r.head_dim = N.OC_F16, 1, 4, 2, 8, 8, 96
    _refused("oc_attend_prompt", r, N.OC_ERR_UNSUPPORTED, b"head_dim")
    r.head_dim, r.kv_len = 64, (1 << 24) + 1
    _refused("oc_attend_prompt", r, N.OC_ERR_UNSUPPORTED, b"2^24")
    r.kv_len = 8
    _refused("oc_attend_prompt", r, N.OC_ERR_INVALID, b"NULL")
    r.documents = 4096
    assert N.lib().oc_attend_prompt_workspace_size(ctypes.byref(r)) == 8
    r.q = r.k = r.v = r.out = 4096
    r.k_stride_s = r.v_stride_s = 64
    _refused("oc_attend_prompt", r, N.OC_ERR_WORKSPACE, b"workspace")
    r.k_stride_s = 32
    _refused("oc_attend_prompt", r, N.OC_ERR_INVALID, b"token stride")
    r.k_stride_s = 68
    _refused("oc_attend_prompt", r, N.OC_ERR_INVALID, b"multiples of 16")


def test_pages():
    from orthocache_gpu import _native as N
    p = N.OcForkParams()
    p.cache_dtype, p.block_size, p.num_seqs, p.num_children = N.OC_BF16, 16, 2, 3
    _refused("oc_fork_pages", p, N.OC_ERR_INVALID, b"parents")
    p.num_children = 5000
    _refused("oc_fork_pages", p, N.OC_ERR_UNSUPPORTED, b"4096")
    p.num_children, p.max_blocks = 2, (1 << 20) + 1
    _refused("oc_fork_pages", p, N.OC_ERR_UNSUPPORTED, b"2^20")
    p.max_blocks, p.block_size = 4, 0
    _refused("oc_fork_pages", p, N.OC_ERR_INVALID, b"power of two")
    p.block_size = 16
    _refused("oc_fork_pages", p, N.OC_ERR_INVALID, b"NULL")
    e = N.OcEvictParams()
    e.num_seqs, e.num_kv_heads, e.block_size, e.max_blocks = 1, 1, 128, 4
    _refused("oc_evict_pages", e, N.OC_ERR_INVALID, b"divide")
    e.block_size = 16
    _refused("oc_evict_pages", e, N.OC_ERR_INVALID, b"tile_map")
    e.tile_map_cols = 1
    _refused("oc_evict_pages", e, N.OC_ERR_INVALID, b"NULL")


def test_limits():
    from orthocache_gpu import _native as N
    p = N.OcForkParams()
    p.cache_dtype, p.block_size, p.num_seqs, p.num_children, p.num_kv_heads, p.head_dim = N.OC_BF16, 1 << 22, 1, 1, 2, 128
    _refused("oc_fork_pages", p, N.OC_ERR_UNSUPPORTED, b"2^30 bytes")
    r = N.OcAttendPromptParams()
    r.dtype, r.batch, r.num_q_heads, r.num_kv_heads, r.q_len, r.kv_len, r.head_dim = N.OC_F16, 1, 4, 2, 8, 4096, 64
    r.mods.scale, r.mods.softcap = 1e20, 1e-20
    _refused("oc_attend_prompt", r, N.OC_ERR_INVALID, b"over softcap")
    r.mods.softcap = 0.0
    size = N.lib().oc_attend_prompt_workspace_size(ctypes.byref(r))
    assert size % (4 * 8 * (64 + 2) * 4) == 0 and size > 0  # a whole number of shares of 4 heads of 8 queries
    r.num_q_heads = r.num_kv_heads = 1
    for r.q_len, r.kv_len in ((65408, 32768), (64, 1 << 24), (30000, 40000), (2 ** 23, 64)):  # shares' sums stay small
        assert N.lib().oc_attend_prompt_workspace_size(ctypes.byref(r)) < 2 ** 27
    r.num_q_heads, r.num_kv_heads, r.q_len, r.kv_len = 4, 2, 8, 4096
    r.q = r.k = r.v = r.out = 4096
    r.k_stride_s = r.v_stride_s = 64
    r.workspace, r.workspace_bytes = 4104, size
    _refused("oc_attend_prompt", r, N.OC_ERR_INVALID, b"16-byte")


def test_entry_points_need_a_gpu():
    import orthocache_gpu as oc
    x = torch.zeros((2, 2, 64))
    i = torch.zeros(2, dtype=torch.int32)
    t = torch.zeros((2, 1), dtype=torch.int32)
    c = torch.zeros((3, 2, 16, 64))
    with pytest.raises(RuntimeError, match="GPU only"):
        oc.apply_rotary(x, None, i, oc.rotary_table(64, device="cpu"))
    with pytest.raises(RuntimeError, match="GPU only"):
        oc.append_paged(x, x, c, c, t, i)
    with pytest.raises(RuntimeError, match="GPU only"):
        oc.attend_paged(x, c, c, t, i)
    with pytest.raises(RuntimeError, match="GPU only"):
        oc.attend_prompt(x[None], x[None], x[None])
    with pytest.raises(RuntimeError, match="GPU only"):
        oc.fork_pages(c, c, t, i, i)
    with pytest.raises(RuntimeError, match="GPU only"):
        oc.evict_pages(t, i, i, torch.zeros((2, 1), dtype=torch.bool), block_size=16)


def test_rotary_table_arguments():
    import orthocache_gpu as oc
    for kw, text in ((dict(rotary_dim=3), "even"), (dict(rotary_dim=4, base=0.0), "base"),
                     (dict(rotary_dim=4, scaling={"type": "other", "factor": 2}), "unknown"),
                     (dict(rotary_dim=4, scaling={"type": "linear", "factor": 0}), "factor"),
                     (dict(rotary_dim=2, scaling={"type": "ntk", "factor": 2}), "ntk"),
                     (dict(rotary_dim=4, scaling={"type": "ramp", "factor": 2, "low": 4, "high": 4, "original": 9}), "low < high")):
        with pytest.raises(ValueError, match=text):
            oc.rotary_table(device="cpu", **kw)


def test_overlaps():
    from orthocache_gpu._ops import ops
    overlaps = ops().overlaps
    x = torch.zeros((4, 6, 8))
    assert not overlaps(x) and not overlaps(x.transpose(0, 2)) and not overlaps(x[:, ::2, 3:]) and not overlaps(x[:, :1])
    assert overlaps(x[:, :1].expand(4, 6, 8)) and overlaps(torch.as_strided(x, (3, 4), (2, 1)))
