"""Rotary positions on tensors and into paged caches, against float64."""

import pytest
import torch

from tests import paged_oracle as O

pytestmark = pytest.mark.gpu
DEV = "cuda"
DTYPES = [torch.float32, torch.float16, torch.bfloat16]


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


def _check(got, x, positions, table, layout, backward=False):
    y = O.turn(x.double(), positions, table.inv_freq, table.scale, layout, backward)
    bound = O.turn_bound(x.double(), y, x.dtype, table.rotary_dim, layout, table.scale)
    over = ((got.double() - y).abs() - bound).max()
    assert float(over) <= 0.0, f"{float(over):.3g} over the bound"
    assert torch.equal(got[..., table.rotary_dim:], x[..., table.rotary_dim:])


@pytest.mark.parametrize("dt", DTYPES, ids=str)
@pytest.mark.parametrize("layout", ["half", "interleaved"])
@pytest.mark.parametrize("d,rot", [(128, 128), (128, 64), (64, 64), (80, 20), (96, 96), (48, 2), (512, 512), (10, 6)])
def test_turns(dt, layout, d, rot):
    import orthocache_gpu as oc
    table = oc.rotary_table(rot, 500000.0, device=DEV)
    q, k = _randn((2, 5, 7, d), dt, 1), _randn((2, 3, 7, d), dt, 2)
    pos = torch.tensor([[0, 1, 2, 3, 1000, 131071, 2 ** 24 + 3], [7, 6, 5, 4, 3, 2, 10 ** 6]], device=DEV, dtype=torch.int64)
    for backward in (False, True):
        a, b = oc.apply_rotary(q, k, pos, table, layout=layout, backward=backward)
        _check(a, q, pos[:, None], table, layout, backward)
        _check(b, k, pos[:, None], table, layout, backward)


@pytest.mark.parametrize("tokens", [1, 4, 2047, 2048, 2051])
def test_lengths_and_strides(tokens):
    """One to many tokens; heads and tokens swapped in memory; k absent; int32 positions shared by the batch."""
    import orthocache_gpu as oc
    table = oc.rotary_table(64, device=DEV, scale=1.25)
    base = _randn((2, tokens, 4, 64), torch.bfloat16, 3)
    q = base.transpose(1, 2)
    pos = torch.arange(tokens, device=DEV, dtype=torch.int32) + 11
    got = oc.apply_rotary(q, None, pos, table)
    assert got.shape == q.shape
    _check(got, q, pos, table, "half")
    rows = base[0]  # (tokens, heads, d)
    got3 = oc.apply_rotary(rows, None, pos, table)
    assert torch.equal(got3.transpose(0, 1), got[0])
    odd = _randn((1, 2, tokens, 67), torch.float16, 4)[..., 1:65]  # rows that no 16-byte load fits
    _check(oc.apply_rotary(odd, None, pos, table), odd, pos, table, "half")


@pytest.mark.parametrize("layout", ["half", "interleaved"])
def test_in_place_and_back(layout):
    import orthocache_gpu as oc
    table = oc.rotary_table(128, device=DEV)
    q, k = _randn((1, 4, 33, 128), torch.float32, 5), _randn((1, 2, 33, 128), torch.float32, 6)
    pos = torch.arange(33, device=DEV)
    a, b = oc.apply_rotary(q, k, pos, table, layout=layout)
    q2, k2 = q.clone(), k.clone()
    r = oc.apply_rotary(q2, k2, pos, table, layout=layout, inplace=True)
    assert r[0] is q2 and torch.equal(q2, a) and torch.equal(k2, b)
    back, _ = oc.apply_rotary(a, b, pos, table, layout=layout, backward=True)
    # two turns of float32 pairs: twice turn_bound's 2^-20 of the pair, whose size is at most 2 max |x|
    assert float((back - q).abs().max()) <= 2 * 2.0 ** -20 * 2 * float(q.abs().max()) * 1.01


def test_gradient_by_differences():
    """backward=True is the transpose: sum w . turn(x) changes by backward(w) . dx."""
    import orthocache_gpu as oc
    for layout in ("half", "interleaved"):
        table = oc.rotary_table(32, device=DEV, scale=1.5)
        pos = torch.tensor([3, 100000], device=DEV)
        x, w, dx = (_randn((1, 2, 2, 40), torch.float32, s) for s in (7, 8, 9))
        grad = oc.apply_rotary(w, None, pos, table, layout=layout, backward=True).double()

        def f(t):
            return (w.double() * O.turn(t.double(), pos, table.inv_freq, 1.5, layout)).sum()
        diff = f(x.double() + 0.5 * dx.double()) - f(x.double() - 0.5 * dx.double())  # linear: exact
        # 160 products, each off by turn_bound's float32 part
        assert abs(float(diff - (grad * dx.double()).sum())) <= 160 * 2.0 ** -19 * 1.5 * float(w.abs().max() * dx.abs().max())


def test_scalings():
    import orthocache_gpu as oc
    f = oc.rotary_table(8, 100.0, device=DEV).inv_freq.cpu()
    want = torch.tensor([100.0 ** (-i / 4) for i in range(4)], dtype=torch.float64)
    assert torch.allclose(f, want, rtol=1e-15, atol=0)
    assert torch.allclose(oc.rotary_table(8, 100.0, scaling={"type": "linear", "factor": 4}, device=DEV).inv_freq.cpu(),
                          want / 4, rtol=1e-15, atol=0)
    ntk = oc.rotary_table(8, 100.0, scaling={"type": "ntk", "factor": 4}, device=DEV).inv_freq.cpu()
    assert float(ntk[0]) == 1.0 and abs(float(ntk[3] / want[3]) - 0.25) < 1e-14
    ramp = oc.rotary_table(8, 100.0, scaling={"type": "ramp", "factor": 8, "low": 1, "high": 4, "original": 40},
                           device=DEV).inv_freq.cpu()
    turns = 40 * want / (2 * torch.pi)
    g = ((turns - 1) / 3).clamp(0, 1)
    assert torch.allclose(ramp, g * want + (1 - g) * want / 8, rtol=1e-15, atol=0)
    assert float(ramp[0]) == 1.0 and abs(float(ramp[3] * 8 / want[3]) - 1) < 1e-14


def test_refusals():
    import orthocache_gpu as oc
    table = oc.rotary_table(64, device=DEV)
    q, pos = _randn((1, 2, 3, 64), torch.float32, 1), torch.arange(3, device=DEV)
    with pytest.raises(ValueError, match="positions"):
        oc.apply_rotary(q, None, pos[:2], table)
    with pytest.raises(TypeError, match="int32 or int64"):
        oc.apply_rotary(q, None, pos.float(), table)
    with pytest.raises(ValueError, match="layout"):
        oc.apply_rotary(q, None, pos, table, layout="whole")
    with pytest.raises(ValueError, match="turns 64 columns"):
        oc.apply_rotary(q[..., :32], None, pos, table)
    with pytest.raises(ValueError, match="share memory"):
        oc.apply_rotary(q[:, :1].expand(1, 2, 3, 64), None, pos, table, inplace=True)
    with pytest.raises(ValueError, match="different tensors"):
        oc.apply_rotary(q, q, pos, table, inplace=True)
    with pytest.raises(RuntimeError, match="no gradient"):
        oc.apply_rotary(q.clone().requires_grad_(), None, pos, table)
    with pytest.raises(TypeError, match="dtype"):
        oc.apply_rotary(q, q.half(), pos, table)
    with pytest.raises(TypeError, match="unsupported"):
        oc.apply_rotary(q.double(), None, pos, table)
    assert oc.apply_rotary(q[:, :, :0], None, pos[:0], table).shape == (1, 2, 0, 64)
    k = oc.apply_rotary(q, q[:, :0], pos, table)[1]
    assert k.shape == (1, 0, 3, 64)


# ------------------------------------------------------------ append

def _tables(pages, num_blocks, cols, seed):
    g = torch.Generator().manual_seed(seed)
    order = torch.randperm(num_blocks, generator=g).tolist()
    t, at = [], 0
    for n in pages:
        t.append(order[at:at + n] + [-1] * (cols - n))
        at += n
    return torch.tensor(t, dtype=torch.int32)


@pytest.mark.parametrize("dt,cache", [(torch.float32, torch.float32), (torch.float16, torch.float16),
                                      (torch.bfloat16, torch.bfloat16), (torch.bfloat16, torch.float8_e4m3fn),
                                      (torch.float32, torch.float8_e4m3fn), (torch.float16, torch.float32),
                                      (torch.float32, torch.bfloat16)], ids=str)
@pytest.mark.parametrize("d,rot,layout,bs", [(128, 128, "half", 16), (64, 32, "interleaved", 8), (72, 20, "half", 1),
                                             (40, 40, "interleaved", 64)])
def test_append(dt, cache, d, rot, layout, bs):
    """Ragged chunks (one empty, one of an idle sequence), padding rows on both
    sides, explicit positions; every slot that no token owns stays as it was."""
    import orthocache_gpu as oc
    hq, hkv = 6, 2
    cached, fresh = [0, 5, 130, -1, 63, 64], [3, 0, 70, 2, 1, 9]
    pages = [-(-max(c, 0) // bs) + -(-f // bs) + 1 for c, f in zip(cached, fresh)]
    cols, nb = max(pages), sum(pages) + 3
    tables = _tables(pages, nb, cols, 1)
    lead, tail = 2, 3
    cu = [lead]
    for f in fresh:
        cu.append(cu[-1] + f)
    total = cu[-1] + tail
    q, k, v = (_randn((total, h, d), dt, s) for h, s in ((hq, 2), (hkv, 3), (hkv, 4)))
    pos = torch.randint(0, 200000, (total,), generator=torch.Generator().manual_seed(5)).to(DEV)
    kc, vc = (_randn((nb, hkv, bs, d), torch.float32, s).to(cache) for s in (6, 7))
    k0, v0 = kc.clone(), vc.clone()
    table = oc.rotary_table(rot, device=DEV, scale=1.1)
    ks, vs = (0.01, 0.02) if cache == torch.float8_e4m3fn else (1.0, 1.0)
    ints = [torch.tensor(x, dtype=torch.int32, device=DEV) for x in (cached, cu)]
    out = oc.append_paged(k, v, kc, vc, tables.to(DEV), ints[0], q=q, cu_seqlens=ints[1], positions=pos, table=table,
                          layout=layout, k_scale=ks, v_scale=vs)
    turned = {n: O.turn(x.double().transpose(0, 1), pos, table.inv_freq, 1.1, layout).transpose(0, 1) for n, x in (("q", q), ("k", k))}
    real, owned = torch.zeros(total, dtype=torch.bool), torch.zeros((nb, bs), dtype=torch.bool)
    for b, f in enumerate(fresh):
        for i in range(f):
            if cached[b] < 0:
                continue
            r, n = cu[b] + i, cached[b] + i
            page, slot = int(tables[b, n // bs]), n % bs
            real[r], owned[page, slot] = True, True
            kw, vw = turned["k"][r] / ks, v[r].float().cpu() / vs
            if cache == torch.float8_e4m3fn:
                vw = vw.clamp(-448, 448)
                kw = kw.clamp(-448, 448)
                # half a step (2^-4 of the value, 2^-10 below the normal range), and the turn's own error
                tol = 2.0 ** -4 * kw.abs() + 2.0 ** -10 + 2.0 ** -19 * 1.1 * 2 * k[r].double().abs().amax() / ks
            else:
                tol = O.half_step(cache) * kw.abs() + 2.0 ** -20 * 1.1 * 2 * k[r].double().abs().amax() + 1e-7
            assert bool(((kc[page, :, slot].double() - kw).abs() <= tol).all())
            assert torch.equal(vc[page, :, slot].float().cpu(), vw.to(cache).float())
    real = real.to(DEV)
    assert float(out[~real].abs().max()) == 0.0
    y = turned["q"]
    bound = O.turn_bound(q.double(), y, dt, rot, layout, 1.1)
    assert float(((out.double() - y).abs() - bound)[real].max()) <= 0.0
    keep = ~owned.to(DEV)
    for now, before in ((kc, k0), (vc, v0)):
        w = torch.uint8
        assert torch.equal(now.view(w).transpose(1, 2)[keep], before.view(w).transpose(1, 2)[keep])


@pytest.mark.parametrize("n", [1, 5, 300, 3000])
def test_append_step(n):
    """One token per sequence, default positions, no queries, caches whose heads lie behind their slots; then the
    same as chunks of many sequences (the search for a row's sequence)."""
    import orthocache_gpu as oc
    d, hkv, bs = 64, 2, 16
    g = torch.Generator().manual_seed(n)
    lens = torch.randint(0, 40, (n,), generator=g)
    tables = torch.randperm(3 * n, generator=g).view(n, 3).to(torch.int32).to(DEV)
    k, v = _randn((n, hkv, d), torch.bfloat16, 1), _randn((n, hkv, d), torch.bfloat16, 2)
    kc, vc = (torch.zeros((3 * n, bs, hkv, d), dtype=torch.bfloat16, device=DEV).transpose(1, 2) for _ in range(2))
    table = oc.rotary_table(d, device=DEV)
    l32 = lens.to(torch.int32).to(DEV)
    assert oc.append_paged(k, v, kc, vc, tables, l32, table=table) is None
    page = tables[torch.arange(n), (lens // bs).to(DEV)].long()
    slot = (lens % bs).to(DEV)
    got = kc[page, :, slot]
    _check(got.transpose(0, 1), k.transpose(0, 1), lens.to(DEV), table, "half")
    assert torch.equal(vc[page, :, slot], v)
    k2, v2 = torch.zeros_like(kc), torch.zeros_like(vc)
    cu = torch.arange(n + 1, dtype=torch.int32, device=DEV)
    oc.append_paged(k, v, k2, v2, tables, l32, table=table, cu_seqlens=cu, sync=False)
    assert torch.equal(k2, kc) and torch.equal(v2, vc)


def test_append_special_values_and_bad_blocks():
    import orthocache_gpu as oc
    inf, nan = float("inf"), float("nan")
    k = torch.tensor([1e9, -1e9, inf, -inf, nan, 448.0, 464.1, 0.0], device=DEV).repeat(1, 1, 1)
    kc, vc = (torch.zeros((2, 1, 16, 8), device=DEV).to(torch.float8_e4m3fn) for _ in range(2))
    t = torch.tensor([[1]], dtype=torch.int32, device=DEV)
    lens = torch.tensor([3], dtype=torch.int32, device=DEV)
    oc.append_paged(k, k, kc, vc, t, lens)
    got = kc[1, 0, 3].float().cpu()
    assert got[:4].tolist() == [448.0, -448.0, 448.0, -448.0] and torch.isnan(got[4]) and got[5:].tolist() == [448.0, 448.0, 0.0]
    before = kc.clone()
    for bad, n in ((-1, 3), (2, 3), (1, 16)):
        t[0, 0] = bad
        with pytest.raises(ValueError, match="no block"):
            oc.append_paged(k, k, kc, vc, t, torch.tensor([n], dtype=torch.int32, device=DEV))
    oc.append_paged(k, k, kc, vc, t, torch.tensor([2 ** 31 - 1], dtype=torch.int32, device=DEV), sync=False)
    assert torch.equal(kc.view(torch.uint8), before.view(torch.uint8))


def test_append_refusals():
    import orthocache_gpu as oc
    k = _randn((2, 1, 64), torch.bfloat16, 1)
    kc, vc = (torch.zeros((4, 1, 16, 64), device=DEV, dtype=torch.bfloat16) for _ in range(2))
    t = torch.zeros((2, 2), dtype=torch.int32, device=DEV)
    lens = torch.zeros(2, dtype=torch.int32, device=DEV)
    with pytest.raises(ValueError, match="cu_seqlens"):
        oc.append_paged(k, k, kc, vc, t[:1], lens[:1])
    with pytest.raises(TypeError, match="int32"):
        oc.append_paged(k, k, kc, vc, t.long(), lens)
    with pytest.raises(TypeError, match="int32"):
        oc.append_paged(k, k, kc, vc, t, lens.long())
    with pytest.raises(ValueError, match="float8"):
        oc.append_paged(k, k, kc, vc, t, lens, k_scale=0.5)
    with pytest.raises(ValueError, match="power of 2"):
        oc.append_paged(k, k, kc[:, :, :12], vc[:, :, :12], t, lens)
    with pytest.raises(ValueError, match="share memory"):
        oc.append_paged(k, k, kc[:1].expand(4, 1, 16, 64), vc, t, lens)
    with pytest.raises(TypeError, match="dtype"):
        oc.append_paged(k, k.float(), kc, vc, t, lens)
    with pytest.raises(RuntimeError, match="GPU"):
        oc.append_paged(k.cpu(), k, kc, vc, t, lens)
    assert oc.append_paged(k[:0], k[:0], kc, vc, t[:0], lens[:0], q=k[:0]).shape == (0, 1, 64)
