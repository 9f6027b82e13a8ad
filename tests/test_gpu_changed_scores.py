"""Attention with changed scores, over paged caches and over whole prompts,
against float64 with bounds from the roundings (tests/paged_oracle.py)."""

import math

import pytest
import torch

from tests import paged_oracle as O

pytestmark = pytest.mark.gpu
DEV = "cuda"
DTYPES = [torch.float32, torch.float16, torch.bfloat16]
FP8 = torch.float8_e4m3fn
INF, NAN = float("inf"), float("nan")


@pytest.fixture(scope="module", autouse=True)
def _gpu():
    if not torch.cuda.is_available():
        pytest.skip("no GPU")
    import orthocache_gpu._native as N
    N.lib()
    yield


def _randn(shape, dt, seed):
    g = torch.Generator().manual_seed(seed)
    return torch.randn(shape, generator=g).to(dt).to(DEV)


def _slopes(h):
    return torch.tensor([2.0 ** (-8.0 * (i + 1) / h) for i in range(h)], device=DEV)


# what the kernels round: the prompt kernel its 16-bit probabilities, which run up to 2^8 relative to the row's
# reference of at least the largest one / 2^8; float16 ones below 2^-14 are subnormal (2^-25 each)
def _p_step(dt):
    return 0.0 if dt == torch.float32 else O.half_step(dt)


# ------------------------------------------------------------ paged

def _paged(lens, hkv, d, bs, dt, seed, transposed=False):
    """A pool of random values with every sequence's blocks in random order; tables -1 past them."""
    pages = [-(-n // bs) for n in lens]
    nb, cols = sum(pages) + 3, max(pages + [1])
    g = torch.Generator().manual_seed(seed)
    order = torch.randperm(nb, generator=g).tolist()
    t, at = [], 0
    for n in pages:
        t.append(order[at:at + n] + [-1] * (cols - n))
        at += n
    shape = (nb, bs, hkv, d) if transposed else (nb, hkv, bs, d)
    kc, vc = (torch.randn(shape, generator=g).to(dt).to(DEV) for _ in range(2))
    if transposed:
        kc, vc = kc.transpose(1, 2), vc.transpose(1, 2)
    return kc, vc, torch.tensor(t, dtype=torch.int32, device=DEV)


def _row(cache, table, b, h, n, bs):
    ids = table[b, :-(-n // bs)].long()
    c = cache[:, h].contiguous()
    c = c.view(torch.uint8)[ids].view(c.dtype) if c.dtype == FP8 else c[ids]
    return c.double().reshape(-1, c.shape[-1])[:n]


def _check_paged(out, q, kc, vc, table, lens, *, scale=None, softcap=0.0, slopes=None, window=0, prefix=None, ks=1.0,
                 vs=1.0, evict=None, what="", p_step=0.0):
    n, hq, d = q.shape
    hkv, bs = kc.shape[1], kc.shape[2]
    scale = 1.0 / math.sqrt(d) if scale is None else scale
    for b in range(n):
        m = lens[b]
        for h in range(hq):
            kv = h // (hq // hkv)
            k, v = _row(kc, table, b, kv, m, bs) * ks, _row(vc, table, b, kv, m, bs) * vs
            more = None
            if evict is not None:
                j = torch.arange(m, device=DEV)
                t = j // 64
                cols = evict.shape[2]
                gone = (t < m // 64) & (t < cols) & (evict[b, kv][t.clamp(max=max(cols - 1, 0))] if cols else False)
                more = ~gone[None, :]
            o, bound = O.attention(q[b, h:h + 1], k, v, torch.tensor([m - 1], device=DEV), scale=scale, softcap=softcap,
                                   slopes=None if slopes is None else float(slopes[h]), window=window,
                                   prefix=0 if prefix is None else int(prefix[b]), seen_more=more, p_step=p_step,
                                   p_tiny=2.0 ** -24 if q.dtype == torch.float16 and p_step else 0.0)
            O.check_out(out[b, h], o[0], bound[0], f"{what} sequence {b} head {h}")


CHANGES = [dict(), dict(softcap=20.0), dict(slopes=True), dict(window=70), dict(softcap=5.0, slopes=True, window=200, prefix=[0, 1, 64, 70, 3, 500, 1]),
           dict(window=1, prefix=[130, 0, 5, 1, 64, 63, 0]), dict(evict=0.5), dict(evict=0.7, window=300, prefix=[70] * 7), dict(evict=1.0, softcap=3.0)]


@pytest.mark.parametrize("portable", [False, True], ids=["tuned", "portable"])
@pytest.mark.parametrize("change", range(len(CHANGES)))
@pytest.mark.parametrize("dt,cache,d,g,bs", [(torch.float32, torch.float32, 128, 2, 16), (torch.float16, torch.float16, 64, 8, 16),
                                             (torch.bfloat16, torch.bfloat16, 128, 4, 32), (torch.bfloat16, FP8, 128, 8, 64),
                                             (torch.float16, FP8, 64, 3, 16), (torch.bfloat16, torch.bfloat16, 256, 5, 128),
                                             (torch.bfloat16, FP8, 256, 1, 16)], ids=str)
def test_paged(dt, cache, d, g, bs, change, portable):
    import orthocache_gpu as oc
    c = dict(CHANGES[change])
    lens, hkv = [0, 1, 63, 64, 65, 700, 1037], 2
    kc, vc, t = _paged(lens, hkv, d, bs, cache, change)
    q = _randn((len(lens), hkv * g, d), dt, 99)
    ks, vs = (1.5, 0.75) if cache == FP8 else (1.0, 1.0)
    slopes = _slopes(hkv * g) if c.pop("slopes", False) else None
    prefix = c.pop("prefix", None)
    evict = None
    if "evict" in c:
        evict = torch.rand((len(lens), hkv, 17), generator=torch.Generator().manual_seed(change)).to(DEV) < c.pop("evict")
    p32 = None if prefix is None else torch.tensor(prefix, dtype=torch.int32, device=DEV)
    l32 = torch.tensor(lens, dtype=torch.int32, device=DEV)
    for splits in (None, 1, 7):
        out = oc.attend_paged(q, kc, vc, t, l32, alibi_slopes=slopes, prefix_lens=p32, k_scale=ks, v_scale=vs, evict_mask=evict,
                              num_splits=splits, portable=portable, **c)
        _check_paged(out, q, kc, vc, t, lens, slopes=slopes, prefix=prefix, ks=ks, vs=vs, evict=evict, p_step=_p_step(dt),
                     what=f"splits {splits}", **c)


@pytest.mark.parametrize("d", [64, 128, 256])
@pytest.mark.parametrize("cache", [torch.bfloat16, FP8], ids=str)
def test_paged_blocks(d, cache):
    """Blocks of 8 to 1024 tokens (four to a unit of the tuned kernel's, and a unit in a part of one), more query
    heads to a kv head than one workgroup takes."""
    import orthocache_gpu as oc
    for bs, g in ((8, 17), (16, 33), (512, 2), (1024, 16)):
        lens = [29, 1100, 2500]
        kc, vc, t = _paged(lens, 1, d, bs, cache, bs, transposed=bs == 8)
        q = _randn((3, g, d), torch.bfloat16, 1)
        l32 = torch.tensor(lens, dtype=torch.int32, device=DEV)
        p32 = torch.tensor([3, 100, 41], dtype=torch.int32, device=DEV)
        out = oc.attend_paged(q, kc, vc, t, l32, window=901, prefix_lens=p32, alibi_slopes=_slopes(g))
        _check_paged(out, q, kc, vc, t, lens, window=901, prefix=[3, 100, 41], slopes=_slopes(g), what=f"block {bs}", p_step=_p_step(torch.bfloat16))


@pytest.mark.parametrize("d", [8, 24, 80, 96, 192, 512])
@pytest.mark.parametrize("dt,cache", [(torch.float32, torch.float32), (torch.bfloat16, torch.bfloat16), (torch.float16, FP8)], ids=str)
def test_paged_head_dims(d, dt, cache):
    """Head dims of the portable kernel, blocks of 1 and 4 tokens, caches whose heads lie behind their slots."""
    import orthocache_gpu as oc
    for bs in (1, 4, 256):
        lens = [5, 130]
        kc, vc, t = _paged(lens, 2, d, bs, cache, d, transposed=True)
        q = _randn((2, 6, d), dt, 1)
        l32 = torch.tensor(lens, dtype=torch.int32, device=DEV)
        out = oc.attend_paged(q, kc, vc, t, l32, softcap=10.0, scale=0.3)
        _check_paged(out, q, kc, vc, t, lens, softcap=10.0, scale=0.3, what=f"block {bs}", p_step=_p_step(dt))


@pytest.mark.parametrize("dt,cache,d", [(torch.bfloat16, torch.bfloat16, 128), (torch.float16, FP8, 64),
                                        (torch.float32, torch.float32, 64), (torch.bfloat16, FP8, 256)], ids=str)
def test_paged_unseen_values_have_no_effect(dt, cache, d):
    """NaN and infinities behind the length, outside the window, in evicted tiles and in blocks of no one; an infinite
    value that is seen shows."""
    import orthocache_gpu as oc
    bs, lens, hkv, g = 16, [100, 333], 1, 4
    kc, vc, t = _paged(lens, hkv, d, bs, cache, 3)
    q = _randn((2, g, d), dt, 4)
    l32 = torch.tensor(lens, dtype=torch.int32, device=DEV)
    evict = torch.tensor([[[0] * 6], [[0, 0, 1, 1, 0, 0]]], dtype=torch.uint8, device=DEV)
    kw = dict(window=150, prefix_lens=torch.tensor([0, 7], dtype=torch.int32, device=DEV), evict_mask=evict)
    want = oc.attend_paged(q, kc, vc, t, l32, **kw)
    bad = {torch.bfloat16: [NAN, INF, -INF, -3.3e38], torch.float16: [NAN, INF, -INF, -65504.0],
           torch.float32: [NAN, INF, -INF, -3.4e38], FP8: [NAN, NAN, NAN, -448.0]}[cache]
    seen = torch.zeros((kc.shape[0], bs), dtype=torch.bool)
    for b, n in enumerate(lens):
        for j in range(n):
            if (j >= n - 150 or j < (0, 7)[b]) and not (j // 64 < n // 64 and int(evict[b, 0, j // 64])):
                seen[int(t[b, j // bs]), j % bs] = True
    for value in bad:
        k2, v2 = kc.clone(), vc.clone()
        for c in (k2, v2):
            f = c.float()
            f[:, 0][~seen.to(DEV)] = value
            c.copy_(f.to(cache))
        got = oc.attend_paged(q, k2, v2, t, l32, **kw)
        assert torch.equal(got, want), f"{value} had an effect"
    v2 = vc.clone().float()
    v2[int(t[1, 332 // bs]), 0, 332 % bs, 5] = NAN
    got = oc.attend_paged(q, kc, v2.to(cache), t, l32, **kw)
    assert bool(torch.isnan(got[1, :, 5]).all()) and not bool(torch.isnan(got[0]).any())
    assert int(torch.isnan(got).sum()) == g


def test_paged_long_context_and_offsets():
    """A pool of more than 2^32 bytes, read at its end, and a long sequence."""
    import orthocache_gpu as oc
    nb, hkv, bs, d = 140000, 2, 64, 128
    kc = torch.empty((nb, hkv, bs, d), dtype=torch.bfloat16, device=DEV)
    vc = torch.empty_like(kc)
    lens = [70001, 3]
    ids = torch.arange(nb - 1100, nb, dtype=torch.int32, device=DEV)
    t = torch.full((2, 1100), -1, dtype=torch.int32, device=DEV)
    t[0, :1094] = ids[:1094].flip(0)
    t[1, 0] = ids[1099]
    for s, c in enumerate((kc, vc)):
        c[nb - 1100:] = torch.randn((1100, hkv, bs, d), generator=torch.Generator().manual_seed(s)).to(torch.bfloat16).to(DEV)
    q = _randn((2, 8, d), torch.bfloat16, 1)
    l32 = torch.tensor(lens, dtype=torch.int32, device=DEV)
    slopes = _slopes(8) * 0.001
    out = oc.attend_paged(q, kc, vc, t, l32, alibi_slopes=slopes, softcap=30.0)
    _check_paged(out, q, kc, vc, t, lens, slopes=slopes, softcap=30.0, p_step=_p_step(torch.bfloat16))


def test_paged_large_slopes_and_scores():
    """Scores far below and above zero: a bias of 1e10, and q.k up to 1e4."""
    import orthocache_gpu as oc
    kc, vc, t = _paged([900], 1, 64, 16, torch.bfloat16, 1)
    l32 = torch.tensor([900], dtype=torch.int32, device=DEV)
    q = _randn((1, 2, 64), torch.bfloat16, 2)
    slopes = torch.tensor([1e10, 0.0], device=DEV)
    out = oc.attend_paged(q, kc, vc, t, l32, alibi_slopes=slopes, portable=True)
    v = _row(vc, t, 0, 0, 900, 16)
    assert float((out[0, 0].double() - v[-1]).abs().max()) <= 2.0 ** -7 * float(v[-1].abs().max())
    # only tokens at distance 3 and more remain: the best is far below zero and still wins
    evict = torch.zeros((1, 1, 14), dtype=torch.bool, device=DEV)
    evict[0, 0, 5:] = True
    l2 = torch.tensor([896], dtype=torch.int32, device=DEV)
    out = oc.attend_paged(q, kc, vc, t, l2, alibi_slopes=slopes, evict_mask=evict)
    assert float((out[0, 0].double() - v[319]).abs().max()) <= 2.0 ** -7 * float(v[319].abs().max())
    big = (q * 2000).contiguous()
    out = oc.attend_paged(big, kc, vc, t, l32)
    _check_paged(out, big, kc, vc, t, [900], p_step=_p_step(torch.bfloat16))


def test_paged_errors_and_refusals():
    import orthocache_gpu as oc
    kc, vc, t = _paged([40, 5], 2, 64, 16, torch.bfloat16, 1)
    q = _randn((2, 4, 64), torch.bfloat16, 2)
    l32 = torch.tensor([40, 5], dtype=torch.int32, device=DEV)
    for bad in (-1, kc.shape[0], 2 ** 31 - 1):
        b = t.clone()
        b[0, 1] = bad
        with pytest.raises(ValueError, match="outside"):
            oc.attend_paged(q, kc, vc, b, l32)
        got = oc.attend_paged(q, kc, vc, b, l32, sync=False)  # the bad block's tokens are left out
        assert bool(torch.isfinite(got).all())
        oc.attend_paged(q, kc, vc, b, torch.tensor([16, 5], dtype=torch.int32, device=DEV))  # not needed
    # lengths past the table and below zero are clamped
    over = oc.attend_paged(q, kc, vc, t[:, :1].contiguous(), torch.tensor([4000, -3], dtype=torch.int32, device=DEV))
    same = oc.attend_paged(q, kc, vc, t[:, :1].contiguous(), torch.tensor([16, 0], dtype=torch.int32, device=DEV))
    assert torch.equal(over, same) and float(same[1].abs().max()) == 0.0
    with pytest.raises(ValueError, match="softcap"):
        oc.attend_paged(q, kc, vc, t, l32, softcap=-1.0)
    with pytest.raises(ValueError, match="window"):
        oc.attend_paged(q, kc, vc, t, l32, window=-1)
    with pytest.raises(ValueError, match="alibi_slopes"):
        oc.attend_paged(q, kc, vc, t, l32, alibi_slopes=torch.ones(2, device=DEV))
    with pytest.raises(ValueError, match="query heads"):
        oc.attend_paged(q[:, :3], kc, vc, t, l32)
    with pytest.raises(TypeError, match="dtype"):
        oc.attend_paged(q.half(), kc, vc, t, l32)
    with pytest.raises(TypeError, match="int32"):
        oc.attend_paged(q, kc, vc, t, l32.long())
    with pytest.raises(TypeError, match="bool or uint8"):
        oc.attend_paged(q, kc, vc, t, l32, evict_mask=torch.zeros((2, 2, 1), device=DEV))
    with pytest.raises(ValueError, match="num_splits"):
        oc.attend_paged(q, kc, vc, t, l32, num_splits=0)
    with pytest.raises(RuntimeError, match="no gradient"):
        oc.attend_paged(q.clone().requires_grad_(), kc, vc, t, l32)
    out = torch.full((2, 8, 64), 7.0, dtype=torch.bfloat16, device=DEV)
    r = oc.attend_paged(q, kc, vc, t, l32, out=out[:, ::2])
    assert torch.equal(out[:, ::2], oc.attend_paged(q, kc, vc, t, l32)) and bool((out[:, 1::2] == 7.0).all()) and r.data_ptr() == out.data_ptr()
    assert oc.attend_paged(q[:0], kc, vc, t[:0], l32[:0]).shape == (0, 4, 64)


def test_paged_in_two_graphs():
    """Two captured calls of different sizes, replayed on two streams at once with eager calls between."""
    import orthocache_gpu as oc
    sets = []
    for s, lens in enumerate(([3000, 17], [900])):
        kc, vc, t = _paged(lens, 2, 128, 16, torch.bfloat16, s)
        q = _randn((len(lens), 8, 128), torch.bfloat16, s + 5)
        sets.append((q, kc, vc, t, torch.tensor(lens, dtype=torch.int32, device=DEV)))
    want = [oc.attend_paged(*x, softcap=9.0) for x in sets]
    graphs, outs, streams = [], [], [torch.cuda.Stream(), torch.cuda.Stream()]
    for x in sets:
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            outs.append(oc.attend_paged(*x, softcap=9.0, sync=False))
        graphs.append(g)
    for _ in range(4):
        for o in outs:
            o.zero_()
        torch.cuda.synchronize()
        for g, st in zip(graphs, streams):
            with torch.cuda.stream(st):
                g.replay()
        oc.attend_paged(*sets[0], sync=False)
        torch.cuda.synchronize()
        for o, w in zip(outs, want):
            assert torch.equal(o, w)


# ------------------------------------------------------------ prompts

def _check_prompt(out, q, k, v, *, scale=None, softcap=0.0, slopes=None, window=0, prefix=None, docs=None, evict=None, what=""):
    B, hq, sq, d = q.shape
    hkv, skv = k.shape[1], k.shape[2]
    scale = 1.0 / math.sqrt(d) if scale is None else scale
    place = torch.arange(sq, device=DEV) + skv - sq
    j = torch.arange(skv, device=DEV)
    for b in range(B):
        for h in range(hq):
            kv = h // (hq // hkv)
            more = torch.ones((sq, skv), dtype=torch.bool, device=DEV)
            if docs is not None:
                dd = docs if docs.dim() == 1 else docs[b]
                mine = torch.where(place >= 0, dd[place.clamp(min=0)], -1) if skv else place
                more &= (mine[:, None] == dd[None, :]) & (mine[:, None] >= 0)
            if evict is not None and evict.shape[2]:
                t = j // 64
                gone = (t < skv // 64) & (t < evict.shape[2]) & (evict[b, kv][t.clamp(max=evict.shape[2] - 1)] != 0)
                more &= ~gone[None, :]
            o, bound = O.attention(q[b, h], k[b, kv], v[b, kv], place, scale=scale, softcap=softcap,
                                   slopes=None if slopes is None else float(slopes[h]), window=window,
                                   prefix=0 if prefix is None else int(prefix[b]), seen_more=more, p_step=_p_step(q.dtype),
                                   p_tiny=2.0 ** -24 if q.dtype == torch.float16 else 0.0)
            O.check_out(out[b, h], o, bound, f"{what} batch {b} head {h}")


PROMPTS = [dict(), dict(softcap=20.0), dict(slopes=True), dict(window=1), dict(window=70, prefix=True), dict(prefix=True),
           dict(docs=3), dict(docs=2, prefix=True, softcap=5.0, slopes=True), dict(evict=0.5, window=200), dict(docs=-1, slopes=True)]


@pytest.mark.parametrize("change", range(len(PROMPTS)))
@pytest.mark.parametrize("sq,skv", [(1, 1), (63, 63), (65, 65), (130, 300), (257, 257), (200, 100), (1, 513), (5, 0)])
@pytest.mark.parametrize("dt,d", [(torch.float32, 64), (torch.float32, 128), (torch.float16, 128), (torch.bfloat16, 64), (torch.bfloat16, 128)], ids=str)
def test_prompt(dt, d, sq, skv, change):
    import orthocache_gpu as oc
    c = dict(PROMPTS[change])
    B, hq, hkv = 2, 4, 2
    q = _randn((B, sq, hq, d), dt, 1).transpose(1, 2)
    k, v = (_randn((B, skv, hkv, d), dt, s).transpose(1, 2) for s in (2, 3))
    slopes = _slopes(hq) if c.pop("slopes", False) else None
    prefix = torch.tensor([7, max(0, skv // 2)], dtype=torch.int32, device=DEV) if c.pop("prefix", False) else None
    docs, evict = c.pop("docs", None), c.pop("evict", None)
    if docs is not None:
        g = torch.Generator().manual_seed(skv + change)
        if docs < 0:  # documents in any order, some places of none
            docs = torch.randint(-1, 3, (B, skv), generator=g).to(torch.int32).to(DEV)
        else:
            docs = torch.sort(torch.randint(0, docs, (B, skv), generator=g), 1).values.to(torch.int32).to(DEV)
    if evict is not None:
        evict = torch.rand((B, hkv, skv // 64 + 1), generator=torch.Generator().manual_seed(9)).to(DEV) < evict
    out = oc.attend_prompt(q, k, v, alibi_slopes=slopes, prefix_lens=prefix, documents=docs, evict_mask=evict, **c)
    _check_prompt(out, q, k, v, slopes=slopes, prefix=prefix, docs=docs, evict=evict, **c)


@pytest.mark.parametrize("dt", [torch.float16, torch.bfloat16], ids=str)
def test_prompt_many_tiles(dt):
    """More than 64 tiles (several words of them), documents of all lengths, several query blocks per head."""
    import orthocache_gpu as oc
    n, d = 4400, 128
    q, k, v = _randn((1, 2, n, d), dt, 1), _randn((1, 1, n, d), dt, 2), _randn((1, 1, n, d), dt, 3)
    cuts = [0, 3, 64, 70, 700, 701, 2900, 4399, n]
    docs = torch.cat([torch.full((b - a,), i, dtype=torch.int32) for i, (a, b) in enumerate(zip(cuts, cuts[1:]))]).to(DEV)
    slopes = _slopes(2)
    out = oc.attend_prompt(q, k, v, documents=docs, alibi_slopes=slopes)
    _check_prompt(out, q, k, v, docs=docs, slopes=slopes)
    out = oc.attend_prompt(q, k, v, softcap=8.0, window=1500, prefix_lens=torch.tensor([4300], dtype=torch.int32, device=DEV))
    _check_prompt(out, q, k, v, softcap=8.0, window=1500, prefix=[4300])


@pytest.mark.parametrize("dt,d", [(torch.float32, 64), (torch.float32, 128), (torch.float16, 64), (torch.bfloat16, 128)], ids=str)
def test_prompt_unseen_values_have_no_effect(dt, d):
    """Values that are not finite: in the future, behind the window, in other documents, in padding; a row that sees
    one shows it, the others are as without it."""
    import orthocache_gpu as oc
    n = 300
    q, k, v = _randn((1, 2, n, d), dt, 1), _randn((1, 1, n, d), dt, 2), _randn((1, 1, n, d), dt, 3)
    docs = torch.tensor([0] * 100 + [-1] * 30 + [1] * 170, dtype=torch.int32, device=DEV)
    want = oc.attend_prompt(q, k, v, documents=docs)
    for value in (NAN, INF, -INF):
        k2, v2 = k.clone(), v.clone()
        k2[:, :, 100:130], v2[:, :, 100:130] = value, value
        assert torch.equal(oc.attend_prompt(q, k2, v2, documents=docs), want)
        v3 = v2.clone()
        v3[0, 0, 210, 7] = value  # seen by the rows from 210 on of its document
        got = oc.attend_prompt(q, k2, v3, documents=docs)
        _check_prompt(got, q, k2, v3, docs=docs, what=str(value))
    for kw in (dict(window=60), dict(prefix_lens=torch.tensor([5], dtype=torch.int32, device=DEV)), dict()):
        k2, v2 = k.clone(), v.clone()
        v2[0, 0, 150, 3], v2[0, 0, 151, 3], v2[0, 0, 160, 9] = INF, -INF, NAN
        k2[0, 0, 200] = NAN
        got = oc.attend_prompt(q, k2, v2, **kw)
        check = {("prefix" if a == "prefix_lens" else a): b for a, b in kw.items()}
        ok = torch.arange(n, device=DEV) < 200
        if "window" in kw:
            ok |= torch.arange(n, device=DEV) >= 260
        assert bool(torch.isnan(got[0, :, ~ok]).all())
        k3 = k2.clone()
        k3[0, 0, 200] = 0.0
        B = oc.attend_prompt(q, k3, v2, **kw)
        assert torch.equal(B[0, :, ok].nan_to_num(1.0, 2.0, 3.0), got[0, :, ok].nan_to_num(1.0, 2.0, 3.0))
        _check_prompt(B, q, k3, v2, what=str(kw), **check)


SHARES = [dict(), dict(softcap=20.0, slopes=True), dict(window=700), dict(window=70, prefix=True), dict(docs=5), dict(evict=0.5, docs=-1)]


@pytest.mark.parametrize("change", range(len(SHARES)))
@pytest.mark.parametrize("sq,skv", [(1, 4097), (130, 2000), (1341, 1341), (1500, 1400)])
@pytest.mark.parametrize("dt,d", [(torch.float32, 64), (torch.float32, 128), (torch.float16, 128), (torch.bfloat16, 64)], ids=str)
def test_prompt_shares(dt, d, sq, skv, change):
    """Few queries on a long context: tiles in shares, some of which see nothing, some rows nothing at all."""
    import orthocache_gpu as oc
    c = dict(SHARES[change])
    B, hq, hkv = 2, 2, 1
    q, k, v = _randn((B, hq, sq, d), dt, 1), _randn((B, hkv, skv, d), dt, 2), _randn((B, hkv, skv, d), dt, 3)
    slopes = _slopes(hq) if c.pop("slopes", False) else None
    prefix = torch.tensor([900, 0], dtype=torch.int32, device=DEV) if c.pop("prefix", False) else None
    docs, evict = c.pop("docs", None), c.pop("evict", None)
    g = torch.Generator().manual_seed(skv + change)
    if docs is not None:
        docs = torch.randint(-1, 2, (B, skv), generator=g) if docs < 0 else torch.sort(torch.randint(0, docs, (B, skv), generator=g), 1).values
        docs = docs.to(torch.int32).to(DEV)
    if evict is not None:
        evict = torch.rand((B, hkv, skv // 64), generator=g) < evict
        evict[0] = True  # nothing but the last tile, where it is not a whole one
        evict = evict.to(DEV)
    out = oc.attend_prompt(q, k, v, alibi_slopes=slopes, prefix_lens=prefix, documents=docs, evict_mask=evict, **c)
    _check_prompt(out, q, k, v, slopes=slopes, prefix=prefix, docs=docs, evict=evict, **c)


@pytest.mark.parametrize("dt", [torch.float32, torch.bfloat16], ids=str)
def test_prompt_shares_not_finite(dt):
    """A NaN in one share makes its rows NaN, an infinite V shows in its column, and what is not seen has no effect."""
    import orthocache_gpu as oc
    n, m, d = 20, 3000, 128
    q, k, v = _randn((1, 2, n, d), dt, 1), _randn((1, 1, m, d), dt, 2), _randn((1, 1, m, d), dt, 3)
    docs = torch.zeros(m, dtype=torch.int32, device=DEV)
    docs[500:900] = -1
    want = oc.attend_prompt(q, k, v, documents=docs)
    _check_prompt(want, q, k, v, docs=docs)
    k2, v2 = k.clone(), v.clone()
    k2[:, :, 500:900], v2[:, :, 500:900] = NAN, INF
    assert torch.equal(oc.attend_prompt(q, k2, v2, documents=docs), want)
    k3 = k2.clone()
    k3[0, 0, m - 5] = NAN  # seen by the last five queries, in the last share
    got = oc.attend_prompt(q, k3, v2, documents=docs)
    assert bool(torch.isnan(got[:, :, -5:]).all()) and torch.equal(got[:, :, :-5], want[:, :, :-5])
    k3 = k2.clone()
    k3[0, 0, 70] = NAN  # by all, in the first
    assert bool(torch.isnan(oc.attend_prompt(q, k3, v2, documents=docs)).all())


def test_prompt_shares_in_two_graphs():
    """Two captured calls with shares, replayed at once: each has a workspace of its own."""
    import orthocache_gpu as oc
    sets = [tuple(_randn((1, h, n, 128), torch.float16, s + i) for i, (h, n) in enumerate(((4, 40), (2, 2500), (2, 2500)))) for s in (1, 9)]
    want = [oc.attend_prompt(*x, softcap=3.0) for x in sets]
    graphs, outs, streams = [], [], [torch.cuda.Stream(), torch.cuda.Stream()]
    for x in sets:
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            outs.append(oc.attend_prompt(*x, softcap=3.0))
        graphs.append(g)
    for _ in range(4):
        for o in outs:
            o.zero_()
        torch.cuda.synchronize()
        for g, st in zip(graphs, streams):
            with torch.cuda.stream(st):
                g.replay()
        oc.attend_prompt(*sets[0])
        torch.cuda.synchronize()
        for o, w in zip(outs, want):
            assert torch.equal(o, w)


def test_prompt_large_bias():
    """Scores far below zero, past -1e9: the nearest key that is left wins."""
    import orthocache_gpu as oc
    n = 256
    q, k, v = _randn((1, 1, n, 64), torch.bfloat16, 1), _randn((1, 1, n, 64), torch.bfloat16, 2), _randn((1, 1, n, 64), torch.bfloat16, 3)
    evict = torch.tensor([[[0, 1, 1, 1]]], dtype=torch.uint8, device=DEV)
    out = oc.attend_prompt(q, k, v, alibi_slopes=torch.tensor([1e10], device=DEV), evict_mask=evict)
    assert float((out[0, 0, 200].double() - v[0, 0, 63].double()).abs().max()) <= 2.0 ** -7 * float(v[0, 0, 63].abs().max())


def test_prompt_strides_streams_and_graphs():
    import orthocache_gpu as oc
    big = _randn((2, 6, 150, 3 * 64 + 8), torch.bfloat16, 1)
    q, k, v = big[..., :64], big[:, ::3, :, 64:128], big[:, ::3, :, 128:192]
    want = oc.attend_prompt(q.contiguous(), k.contiguous(), v.contiguous(), softcap=4.0)
    assert torch.equal(oc.attend_prompt(q, k, v, softcap=4.0), want)
    one = k[:, :, :1].expand(2, 2, 150, 64)  # tokens that share memory
    assert torch.equal(oc.attend_prompt(q, one, v), oc.attend_prompt(q, one.contiguous(), v))
    docs = torch.arange(150, device=DEV, dtype=torch.int32) // 40
    eager = oc.attend_prompt(q, k, v, documents=docs)
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        other = oc.attend_prompt(q, k, v, documents=docs)
    s.synchronize()
    assert torch.equal(other, eager)
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        out = oc.attend_prompt(q, k, v, documents=docs)
    for shift in (0, 13, 40):
        docs.copy_((torch.arange(150, device=DEV, dtype=torch.int32) + shift) // 40)
        g.replay()
        assert torch.equal(out.clone(), oc.attend_prompt(q, k, v, documents=docs))


def test_prompt_refusals():
    import orthocache_gpu as oc
    q = _randn((1, 4, 8, 64), torch.bfloat16, 1)
    k = _randn((1, 2, 8, 64), torch.bfloat16, 2)
    with pytest.raises(NotImplementedError, match="head_dim"):
        oc.attend_prompt(q[..., :32], k[..., :32], k[..., :32])
    with pytest.raises(TypeError, match="int32"):
        oc.attend_prompt(q, k, k, documents=torch.zeros(8, device=DEV, dtype=torch.int64))
    with pytest.raises(ValueError, match="documents"):
        oc.attend_prompt(q, k, k, documents=torch.zeros(7, device=DEV, dtype=torch.int32))
    with pytest.raises(ValueError, match="scale"):
        oc.attend_prompt(q, k, k, scale=NAN)
    with pytest.raises(RuntimeError, match="no gradient"):
        oc.attend_prompt(q.clone().requires_grad_(), k, k)
    with pytest.raises(RuntimeError, match="GPU"):
        oc.attend_prompt(q, k, k, alibi_slopes=torch.ones(4))
    assert oc.attend_prompt(q[:, :, :0], k, k).shape == (1, 4, 0, 64)


# ------------------------------------------------------------ a run of them together

@pytest.mark.parametrize("cache", [torch.bfloat16, FP8], ids=str)
def test_serving_run(cache):
    """Two prompts are prefilled and stored, forked into beams with one ended, decoded step by step with their
    distance bias, their evicted tiles dropped, and decoded again: every output against float64 over the sequences'
    own tokens, kept on the side."""
    import orthocache_gpu as oc
    torch.manual_seed(0)
    dt, hq, hkv, d, bs, nb, cols = torch.bfloat16, 4, 2, 64, 16, 200, 24
    table = oc.rotary_table(d, device=DEV)
    slopes = _slopes(hq) * 0.1
    ks, vs = (0.02, 0.02) if cache == FP8 else (1.0, 1.0)
    kc, vc = (torch.zeros((2, nb, hkv, bs, d), dtype=dt, device=DEV).to(cache) for _ in range(2))
    t = torch.full((2, cols), -1, dtype=torch.int32, device=DEV)
    lens, refs = torch.zeros(2, dtype=torch.int32, device=DEV), torch.zeros(nb, dtype=torch.int32, device=DEV)
    fresh = [150, 75]
    st = oc.fork_pages(kc, vc, t, lens, refs, new_tokens=torch.tensor(fresh, dtype=torch.int32, device=DEV))
    cu = torch.tensor([0, 150, 225], dtype=torch.int32, device=DEV)
    q, k, v = (torch.randn((225, h, d), device=DEV).to(dt) for h in (hq, hkv, hkv))
    q2 = oc.append_paged(k, v, kc[1], vc[1], st.block_tables, st.context_lens, q=q, cu_seqlens=cu, table=table, k_scale=ks, v_scale=vs)
    docs = torch.tensor([0] * 150 + [1] * 75, dtype=torch.int32, device=DEV)
    pos = torch.cat([torch.arange(150), torch.arange(75)]).to(DEV)
    qr, kr = oc.apply_rotary(q, k, pos, table)
    assert torch.equal(qr, q2)
    packed = [x.transpose(0, 1).unsqueeze(0) for x in (qr, kr, v)]
    out = oc.attend_prompt(*packed, documents=docs, alibi_slopes=slopes)
    _check_prompt(out, *packed, docs=docs, slopes=slopes)

    def in_cache(c, i, n0, n1, x, scale):
        """What the cache holds of sequence i's tokens n0 .. n1: x, rounded by at most one step of an 8-bit type
        (the queries' type rounds x here before, the kernel does not)."""
        j = torch.arange(n0, n1, device=DEV)
        page = st.block_tables[i, j // bs].long()
        got = c[1].view(torch.uint8)[page, :, j % bs].view(c.dtype) if c.dtype == FP8 else c[1][page, :, j % bs]
        if c.dtype != FP8:
            assert torch.equal(got, x)
            return got.double()
        got = got.double()
        want = x.double() / scale
        assert bool(((got - want).abs() <= 2.0 ** -3 * want.abs() + 2.0 ** -9).all())
        return got * scale
    held = [(in_cache(kc, i, 0, b - a, kr[a:b], ks), in_cache(vc, i, 0, b - a, v[a:b], vs))
            for i, (a, b) in enumerate(((0, 150), (150, 225)))]
    lens = st.context_lens + torch.tensor(fresh, dtype=torch.int32, device=DEV)
    places = [150, 75]  # positions of the next tokens
    parents = [0, 1, 0, 0]
    st = oc.fork_pages(kc, vc, st.block_tables, lens, st.ref_counts, parents=torch.tensor(parents, dtype=torch.int32, device=DEV), new_tokens=4)
    held = [held[p] for p in parents]
    places = [places[p] for p in parents]
    lens = st.context_lens

    def step():
        nonlocal lens, st
        n = len(held)
        # room for one more token each (an empty sequence that a parent of -1 left gets its first block here)
        st = oc.fork_pages(kc, vc, st.block_tables, lens, st.ref_counts, new_tokens=1)
        q, k, v = (torch.randn((n, h, d), device=DEV).to(dt) for h in (hq, hkv, hkv))
        p = torch.tensor(places, device=DEV)
        q2 = oc.append_paged(k, v, kc[1], vc[1], st.block_tables, lens, q=q, positions=p, table=table, k_scale=ks, v_scale=vs)
        _, kr = oc.apply_rotary(q, k, p, table)
        lens = lens + 1
        for i in range(n):
            m = int(lens[i])
            new = (in_cache(kc, i, m - 1, m, kr[i:i + 1], ks), in_cache(vc, i, m - 1, m, v[i:i + 1], vs))
            held[i] = tuple(torch.cat([x, y]) for x, y in zip(held[i], new))
            places[i] += 1
        out = oc.attend_paged(q2, kc[1], vc[1], st.block_tables, lens, alibi_slopes=slopes, softcap=25.0, k_scale=ks, v_scale=vs)
        for i in range(n):
            assert int(lens[i]) == held[i][0].shape[0]
            for h in range(hq):
                o, bound = O.attention(q2[i, h:h + 1], held[i][0][:, h // 2], held[i][1][:, h // 2],
                                       torch.tensor([held[i][0].shape[0] - 1], device=DEV), scale=d ** -0.5, softcap=25.0,
                                       slopes=float(slopes[h]), p_step=_p_step(dt))
                O.check_out(out[i, h], o[0], bound[0], f"step: sequence {i} head {h}")
    for _ in range(3):
        step()
    mask = torch.zeros((4, hkv, 3), dtype=torch.bool, device=DEV)
    mask[0, :, 0] = mask[2, :, 1] = mask[3, 0, 0] = mask[1, :, 0] = True  # (sequence 3: one head alone)
    before = lens.tolist()
    st, tile_map = oc.evict_pages(st.block_tables, lens, st.ref_counts, mask, block_size=bs)
    lens = st.context_lens
    assert lens.tolist() == [before[0] - 64, before[1] - 64, before[2] - 64, before[3]]
    for i, m in enumerate(tile_map.tolist()):
        at = [j for x in m if x >= 0 for j in range(64 * x, min(64 * x + 64, before[i]))]
        held[i] = (held[i][0][at], held[i][1][at])
    st = oc.fork_pages(kc, vc, st.block_tables, lens, st.ref_counts, parents=torch.tensor([3, 0, -1, 1], dtype=torch.int32, device=DEV))
    lens = st.context_lens
    assert lens.tolist()[2] == 0
    held = [held[3], held[0], (held[0][0][:0], held[0][1][:0]), held[1]]
    places = [places[3], places[0], 0, places[1]]
    step()
    step()
    used = set()
    for row in st.block_tables.tolist():
        used |= {b for b in row if b >= 0}
    assert [b for b, r in enumerate(st.ref_counts.tolist()) if r > 0] == sorted(used)
