"""Calls that the operators around the paged cache allow at their edges, and those they refuse: memory shared by
arguments, numbers outside their range, captured steps, two calls at once."""
import pytest
import torch

from tests import paged_oracle as O

pytestmark = pytest.mark.gpu
DEV = "cuda"


def _randn(shape, dt, seed):
    return torch.randn(shape, generator=torch.Generator().manual_seed(seed)).to(dt).to(DEV)


def _i32(x):
    return torch.tensor(x, dtype=torch.int32, device=DEV)


def test_append_rows_far_from_their_sequence():
    """Rows so far into their sequence that the number does not fit 32 bits have no block."""
    import orthocache_gpu as oc
    k, v = _randn((2, 2, 64), torch.bfloat16, 1), _randn((2, 2, 64), torch.bfloat16, 2)
    kc, vc = (torch.full((3, 2, 16, 64), 7.0, dtype=torch.bfloat16, device=DEV) for _ in range(2))
    for cu in ([-2 ** 31, 2], [-5, 2]):
        for lens in ([2 ** 31 - 1], [48]):
            with pytest.raises(ValueError, match="no block"):
                oc.append_paged(k, v, kc, vc, _i32([[0, 1, 2]]), _i32(lens), cu_seqlens=_i32(cu))
    assert bool((kc == 7.0).all()) and bool((vc == 7.0).all())
    oc.append_paged(k, v, kc, vc, _i32([[0, 1, 2]]), _i32([3]), cu_seqlens=_i32([-5, 2]))  # rows 5 and 6 of it
    assert torch.equal(kc[0, :, 8:10], k.transpose(0, 1)) and bool((kc[0, :, :8] == 7.0).all())


def test_shared_memory_is_refused():
    import orthocache_gpu as oc
    big = _randn((2, 3, 2, 16, 64), torch.bfloat16, 1)
    kc, vc = big[0], big[1]
    k = _randn((1, 2, 64), torch.bfloat16, 2)
    t, l, r = _i32([[0, 1]]), _i32([20]), _i32([1, 1, 0])
    for a, b in ((kc, kc), (kc, big.view(-1)[64:64 + kc.numel()].view_as(kc))):
        with pytest.raises(ValueError, match="different memory"):
            oc.append_paged(k, k, a, b, t, l)
        with pytest.raises(ValueError, match="different memory"):
            oc.fork_pages(a, b, t, l, r)
    oc.append_paged(k, k, kc, vc, t, l)  # halves of one tensor
    inter = _randn((3, 2, 2, 16, 64), torch.bfloat16, 3)
    oc.append_paged(k, k, inter[:, 0], inter[:, 1], t, l)  # and interleaved
    assert torch.equal(inter[1, 0, :, 4], k[0]) and torch.equal(inter[1, 1, :, 4], k[0])
    with pytest.raises(RuntimeError, match="no gradient"):
        oc.append_paged(k, k, kc.clone().requires_grad_(), vc, t, l)

    q = _randn((1, 4, 64), torch.bfloat16, 4)
    want = oc.attend_paged(q, kc, vc, t, l)
    row = torch.empty(5 * 64, dtype=torch.bfloat16, device=DEV)
    row[:256] = q.view(-1)
    with pytest.raises(ValueError, match="share no other memory"):
        oc.attend_paged(row[:256].view(1, 4, 64), kc, vc, t, l, out=row[64:].view(1, 4, 64))
    with pytest.raises(ValueError, match="share no other memory"):
        oc.attend_paged(q, kc, vc, t, l, out=kc.view(-1)[:256].view(1, 4, 64))
    assert torch.equal(oc.attend_paged(q, kc, vc, t, l, out=q), want) and torch.equal(q, want)  # into q itself

    x = _randn((1, 4, 8, 64), torch.float32, 5)
    table, pos = oc.rotary_table(64, device=DEV), torch.arange(8, device=DEV)
    flat = torch.zeros(x.numel() + 64, device=DEV)
    with pytest.raises(ValueError, match="different tensors"):
        oc.apply_rotary(flat[:x.numel()].view_as(x), flat[64:].view_as(x), pos, table, inplace=True)

    one = _i32([0, 0, 0])
    with pytest.raises(ValueError, match="out share"):
        oc.fork_pages(kc, vc, _i32([[0, 1]] * 3), _i32([0, 0, 0]), r, out=oc.PageTables(_i32([[0, 0]] * 3), one, one, _i32([0])))


@pytest.mark.parametrize("scale", [0.0, -0.3, 1e-20, 2.0])
@pytest.mark.parametrize("cap", [1e-12, 1e-3, 4.0, 1e6, 1e20])
@pytest.mark.parametrize("dt", [torch.float32, torch.float16, torch.bfloat16], ids=str)
def test_prompt_caps(dt, cap, scale):
    """Caps far below and far above the scores, scales of 0, below 0 and next to nothing."""
    import orthocache_gpu as oc
    n, d = 150, 64
    q, k, v = (_randn((1, 1, n, d), dt, s) for s in (1, 2, 3))
    out = oc.attend_prompt(q, k, v, scale=scale, softcap=cap, alibi_slopes=torch.tensor([0.1], device=DEV))
    step = {torch.float32: 0.0, torch.float16: 2.0 ** -11, torch.bfloat16: 2.0 ** -8}[dt]
    o, bound = O.attention(q[0, 0], k[0, 0], v[0, 0], torch.arange(n, device=DEV), scale=scale, softcap=cap, slopes=0.1,
                           p_step=step, p_tiny=2.0 ** -24 if dt == torch.float16 else 0.0)
    O.check_out(out[0, 0], o, bound, f"cap {cap} scale {scale}")


def test_captured_step():
    """A decode step (room, rotary and append, attention) captured once and replayed over changing tables and tokens."""
    import orthocache_gpu as oc
    n, hkv, g, bs, d, cols = 3, 2, 4, 16, 64, 8
    kc, vc = (torch.zeros((20, hkv, bs, d), dtype=torch.bfloat16, device=DEV) for _ in range(2))
    table = oc.rotary_table(d, device=DEV)
    refs = torch.zeros(20, dtype=torch.int32, device=DEV)
    tables, lens = torch.full((n, cols), -1, dtype=torch.int32, device=DEV), _i32([0, 0, 0])
    k, v, q = (torch.zeros((n, h, d), dtype=torch.bfloat16, device=DEV) for h in (hkv, hkv, hkv * g))
    slopes = torch.tensor([0.05] * (hkv * g), device=DEV)
    outs = oc.PageTables(tables.clone(), lens.clone(), refs.clone(), _i32([0]))

    def step(sync):
        p = oc.fork_pages(kc, vc, tables, lens, refs, new_tokens=1, sync=sync, out=outs)
        turned = oc.append_paged(k, v, kc, vc, p.block_tables, p.context_lens, q=q, table=table, sync=sync)
        return turned, oc.attend_paged(turned, kc, vc, p.block_tables, p.context_lens + 1, alibi_slopes=slopes, softcap=9.0, sync=sync)

    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        step(False)
    torch.cuda.current_stream().wait_stream(s)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got = step(False)
    for i in range(20):
        for x, seed in ((k, 1), (v, 2), (q, 3)):
            x.copy_(_randn(x.shape, torch.bfloat16, 10 * i + seed))
        graph.replay()
        mine = [x.clone() for x in got] + [kc.clone(), vc.clone()]
        want = step(True)
        for a, b in zip(mine, [*want, kc, vc]):
            assert torch.equal(a, b)
        tables.copy_(outs.block_tables), refs.copy_(outs.ref_counts), lens.add_(1)
    assert lens.tolist() == [20] * 3 and int(outs.status) == 0


def test_two_calls_at_once():
    """The same operators on two streams at once, on caches of their own."""
    import orthocache_gpu as oc
    streams = [torch.cuda.Stream(), torch.cuda.Stream()]

    def work(seed):
        big = _randn((2, 600, 2, 16, 128), torch.bfloat16, seed)
        t = torch.arange(600, dtype=torch.int32, device=DEV).view(4, 150)
        lens = _i32([2300, 2399, 1000, 37])
        return big[0], big[1], t, lens, torch.ones(600, dtype=torch.int32, device=DEV), _randn((4, 8, 128), torch.bfloat16, seed + 1)

    def run(kc, vc, t, lens, refs, q):
        mask = (torch.arange(37, device=DEV) % 3 == 0).expand(4, 37)
        p, _ = oc.evict_pages(t, lens, refs, mask, block_size=16, sync=False)
        p = oc.fork_pages(kc, vc, p.block_tables, p.context_lens, p.ref_counts, parents=_i32([0, 0, 1, 3]), new_tokens=1, sync=False)
        return [p.block_tables, p.context_lens, p.ref_counts, oc.attend_paged(q, kc, vc, p.block_tables, p.context_lens, sync=False),
                oc.attend_prompt(q.view(1, 8, 4, 128), kc.view(1, 2, 9600, 128)[:, :, :3000], vc.view(1, 2, 9600, 128)[:, :, :3000])]

    sets = [work(1), work(50)]
    want = [run(*[x.clone() for x in s]) for s in sets]
    torch.cuda.synchronize()
    got = [None, None]
    for _ in range(3):
        copies = [[x.clone() for x in s] for s in sets]
        torch.cuda.synchronize()
        for i, st in enumerate(streams):
            with torch.cuda.stream(st):
                got[i] = run(*copies[i])
        torch.cuda.synchronize()
        for g, w in zip(got, want):
            assert all(torch.equal(a, b) for a, b in zip(g, w))


@pytest.mark.parametrize("scale", [1.0, 0.02, 0.3, 7.0, 1e-25, 1e25, 1e38])
@pytest.mark.parametrize("dt", [torch.float32, torch.bfloat16], ids=str)
def test_append_fp8_quotients(dt, scale):
    """What an fp8 page holds is the rounded quotient, byte for byte: signed zeros, ties, the clamp, infinities, NaN."""
    import orthocache_gpu as oc
    g = torch.Generator().manual_seed(3)
    n, d = 64, 128
    x = torch.randn((n, 1, d), generator=g) * torch.exp2(torch.randint(-14, 12, (n, 1, d), generator=g).float()) * scale
    ties = torch.arange(-256, 256).float() / 16 * scale
    x.view(-1)[:512] = ties
    x.view(-1)[512:524] = torch.tensor([0.0, -0.0, float("inf"), -float("inf"), float("nan"), 448 * scale, -448 * scale, 449 * scale,
                                        464 * scale, 3e38, -3e38, 1e-38])
    x = x.to(dt).to(DEV)
    kc, vc = (torch.zeros((4, 1, 16, d), dtype=torch.float8_e4m3fn, device=DEV) for _ in range(2))
    oc.append_paged(x, x, kc, vc, _i32([[0, 1, 2, 3]]), _i32([0]), cu_seqlens=_i32([0, n]), k_scale=scale, v_scale=scale)
    want = (x.float() / torch.tensor(scale, dtype=torch.float32, device=DEV)).clamp(-448, 448).to(torch.float8_e4m3fn).view(torch.uint8)
    for c in (kc, vc):
        got = c.view(torch.uint8).view(n, 1, d)
        same = (got == want) | (((got & 127) == 127) & ((want & 127) == 127))  # (a NaN of either sign)
        assert bool(same.all()), (x[~same][:4], got[~same][:4], want[~same][:4])
