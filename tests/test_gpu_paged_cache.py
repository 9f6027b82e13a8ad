"""Forks, ends, room and evicted tiles of paged sequences, against plain Python."""

import random

import pytest
import torch

from tests import paged_oracle as O

pytestmark = pytest.mark.gpu
DEV = "cuda"


@pytest.fixture(scope="module", autouse=True)
def _gpu():
    if not torch.cuda.is_available():
        pytest.skip("no GPU")
    import orthocache_gpu._native as N
    N.lib()
    yield


def _i32(x):
    return torch.tensor(x, dtype=torch.int32, device=DEV)


def _state(rng, lens, bs, cols, spare, shared=0):
    """Tables of random distinct blocks; `shared` blocks are held twice (by sequence 0 and the last)."""
    need = [-(-n // bs) for n in lens]
    nb = sum(need) + spare
    order = rng.sample(range(nb), nb)
    tables, at = [], 0
    for n in need:
        tables.append(order[at:at + n] + [-1] * (cols - n))
        at += n
    for c in range(min(shared, need[0], need[-1])):
        tables[-1][c] = tables[0][c]
    refs = [0] * nb
    for row in tables:
        for b in row:
            if b >= 0:
                refs[b] += 1
    return tables, refs, nb


def _caches(nb, layers, h, bs, d, dt, seed):
    g = torch.Generator().manual_seed(seed)
    shape = (nb, h, bs, d) if layers == 0 else (layers, nb, h, bs, d)
    return [torch.randn(shape, generator=g).to(dt).to(DEV) for _ in range(2)]


def _raw(t):
    return t.contiguous().view(torch.uint8).cpu()


@pytest.mark.parametrize("bs", [1, 8, 16, 64, 256])
@pytest.mark.parametrize("dt,layers,d", [(torch.bfloat16, 0, 64), (torch.float8_e4m3fn, 3, 40), (torch.float32, 2, 10)], ids=str)
@pytest.mark.parametrize("seed", [1, 2])
def test_fork(bs, dt, layers, d, seed):
    import orthocache_gpu as oc
    rng = random.Random(seed * 100 + bs)
    lens = [0, 1, bs, bs + 1, 3 * bs - 1, 2 * bs, 77, 64, 5]
    parents = [3, 3, -1, 8, 3, 0, 4, 4, 1, 2, 6, 6, 5]
    fresh = [rng.choice((0, 1, bs, 2 * bs + 1)) for _ in parents]
    cols = max(-(-n // bs) for n in lens) + 4
    tables, refs, nb = _state(rng, lens, bs, cols, spare=60 + len(parents) * 3, shared=seed)
    want_t, want_l, want_r, copies = O.fork(tables, lens, refs, parents, fresh, bs, cols)
    kc, vc = _caches(nb, layers, 3, bs, d, dt, seed)
    want = []
    for c in (kc, vc):
        w = _raw(c).view(c.shape[:-1] + (-1,)) if layers else _raw(c).view((1,) + c.shape[:-1] + (-1,))
        for src, dst, n in copies:
            w[:, dst, :, :n] = w[:, src, :, :n]
        want.append(w)
    t, l, r = _i32(tables), _i32(lens), _i32(refs)
    res = oc.fork_pages(kc, vc, t, l, r, parents=_i32(parents), new_tokens=_i32(fresh))
    assert res.block_tables.tolist() == want_t
    assert res.context_lens.tolist() == want_l
    assert res.ref_counts.tolist() == want_r
    assert t.tolist() == tables and l.tolist() == lens and r.tolist() == refs  # the inputs stay
    for c, w in zip((kc, vc), want):
        assert torch.equal(_raw(c).view(w.shape), w)


def test_room_and_steps():
    """Every sequence goes on with room for more; what an earlier call made room with comes back."""
    import orthocache_gpu as oc
    rng = random.Random(3)
    lens, bs, cols = [5, 32, 0, 31], 16, 8
    tables, refs, nb = _state(rng, lens, bs, cols, spare=20)
    kc, vc = _caches(nb, 0, 2, bs, 64, torch.bfloat16, 1)
    a = oc.fork_pages(kc, vc, _i32(tables), _i32(lens), _i32(refs), new_tokens=40)
    w = O.fork(tables, lens, refs, [0, 1, 2, 3], [40] * 4, bs, cols)
    assert a.block_tables.tolist() == w[0] and a.ref_counts.tolist() == w[2]
    b = oc.fork_pages(kc, vc, a.block_tables, a.context_lens, a.ref_counts)
    w2 = O.fork(w[0], lens, w[2], [0, 1, 2, 3], [0] * 4, bs, cols)
    assert b.block_tables.tolist() == w2[0] == tables and b.ref_counts.tolist() == w2[2] == refs


def test_many_sequences():
    """Thousands of sequences and children (several rounds of the plan's sums), fewer children than sequences, and a
    wide pool."""
    import orthocache_gpu as oc
    rng = random.Random(9)
    bs, cols = 16, 4
    lens = [rng.randrange(0, 50) for _ in range(4000)]
    parents = [rng.choice((-1, rng.randrange(4000))) for _ in range(3001)]
    tables, refs, nb = _state(rng, lens, bs, cols, spare=15000)
    kc, vc = _caches(nb, 0, 1, bs, 8, torch.float16, 1)
    want_t, want_l, want_r, copies = O.fork(tables, lens, refs, parents, [1] * len(parents), bs, cols)
    k0 = kc.cpu()
    res = oc.fork_pages(kc, vc, _i32(tables), _i32(lens), _i32(refs), parents=_i32(parents), new_tokens=1)
    assert res.block_tables.tolist() == want_t and res.context_lens.tolist() == want_l
    assert res.ref_counts.tolist() == want_r
    for src, dst, n in copies:
        k0[dst, :, :n] = k0[src, :, :n]
    assert torch.equal(kc.cpu(), k0)


def test_fork_failures_leave_everything():
    import orthocache_gpu as oc
    from orthocache_gpu import _native as N
    rng = random.Random(4)
    lens, bs, cols = [20, 17], 16, 3
    tables, refs, nb = _state(rng, lens, bs, cols, spare=1)
    kc, vc = _caches(nb, 2, 2, bs, 64, torch.bfloat16, 1)
    k0 = kc.clone()
    args = (kc, vc, _i32(tables), _i32(lens), _i32(refs))
    with pytest.raises(oc.OutOfPages):
        oc.fork_pages(*args, parents=_i32([0, 0, 1, 1]))
    with pytest.raises(ValueError, match="parents"):
        oc.fork_pages(*args, parents=_i32([0, 2]))
    with pytest.raises(ValueError, match="parents"):
        oc.fork_pages(*args, parents=_i32([-2, 0]))
    with pytest.raises(ValueError, match="columns"):
        oc.fork_pages(*args, new_tokens=30)
    with pytest.raises(ValueError, match="columns"):
        oc.fork_pages(kc, vc, args[2][:, :1], args[3], args[4])
    r = oc.fork_pages(*args, parents=_i32([0, 0, 1, 1]), sync=False)
    assert r.status.tolist() == [N.OC_PAGES_NO_ROOM]
    assert r.block_tables.tolist() == [[-1] * cols] * 4 and r.context_lens.tolist() == [0] * 4
    assert r.ref_counts.tolist() == refs and torch.equal(kc, k0)
    bad = [list(x) for x in tables]
    bad[1][1] = nb  # the block that would be copied
    with pytest.raises(ValueError, match="outside"):
        oc.fork_pages(kc, vc, _i32(bad), args[3], args[4], parents=_i32([0, 1]))
    bad[1][1], bad[1][0] = tables[1][1], -7  # a block that is shared
    r = oc.fork_pages(kc, vc, _i32(bad), args[3], args[4], parents=_i32([0, 1]), sync=False)
    assert r.status.tolist() == [N.OC_PAGES_BAD_BLOCK] and r.block_tables.tolist()[1][0] == -1
    # one more block is enough
    ok = oc.fork_pages(*args, parents=_i32([0, 0, 1]))
    assert ok.status.tolist() == [0]


def test_fork_refusals():
    import orthocache_gpu as oc
    t, l, r = _i32([[0, 1]]), _i32([20]), _i32([1, 1, 0])
    kc, vc = _caches(3, 0, 1, 16, 64, torch.bfloat16, 1)
    with pytest.raises(TypeError, match="int32"):
        oc.fork_pages(kc, vc, t, l.long(), r)
    with pytest.raises(ValueError, match="ref_counts"):
        oc.fork_pages(kc, vc, t, l, r[:2])
    with pytest.raises(ValueError, match="new_tokens"):
        oc.fork_pages(kc, vc, t, l, r, new_tokens=-1)
    with pytest.raises(ValueError, match="overlaps"):
        oc.fork_pages(kc, vc, t, l, r, out=oc.PageTables(t, _i32([0]), _i32([0, 0, 0]), _i32([0])))
    with pytest.raises(NotImplementedError, match="4096"):
        oc.fork_pages(kc, vc, t, l, r, parents=torch.zeros(4097, dtype=torch.int32, device=DEV))
    with pytest.raises(ValueError, match="share memory"):
        oc.fork_pages(kc[:1].expand(3, 1, 16, 64), vc, t, l, r)
    e = oc.fork_pages(kc, vc, t[:0], l[:0], r, parents=_i32([]))
    assert e.block_tables.shape == (0, 2) and e.ref_counts.tolist() == [1, 1, 0]
    # children of nothing: empty sequences with room
    e = oc.fork_pages(kc, vc, t[:0], l[:0], _i32([0, 1, 0]), parents=_i32([-1, -1]), new_tokens=5)
    assert e.block_tables.tolist() == [[-1, -1], [-1, -1]] and e.context_lens.tolist() == [0, 0]


@pytest.mark.parametrize("bs", [1, 8, 16, 32, 64])
@pytest.mark.parametrize("heads", [0, 1, 5])
def test_evict(bs, heads):
    import orthocache_gpu as oc
    rng = random.Random(bs + heads)
    lens = [0, 1, 63, 64, 65, 640, 641, 17000, 16384, 130, -5, 100000]
    cols = 17024 // bs
    tables, refs, nb = _state(rng, [min(max(n, 0), cols * bs) for n in lens], bs, cols, spare=7, shared=0)
    tables[2][-1] = nb - 1  # room that an earlier call made
    refs[nb - 1] += 1
    tiles = 266 if bs != 16 else 200  # (a mask that is narrower than the longest sequence)
    shape = (len(lens), tiles) if heads == 0 else (len(lens), heads, tiles)
    mask = torch.rand(shape, generator=torch.Generator().manual_seed(bs)) < 0.6
    if heads:
        mask = mask | (torch.rand((len(lens), 1, tiles), generator=torch.Generator().manual_seed(bs + 1)) < 0.5)
    gone = (mask if heads == 0 else mask.all(1)).tolist()
    want = O.evict(tables, lens, refs, gone, bs, cols)
    res, tile_map = oc.evict_pages(_i32(tables), _i32(lens), _i32(refs), mask.to(DEV), block_size=bs)
    assert res.context_lens.tolist() == want[1]
    assert res.block_tables.tolist() == want[0]
    assert res.ref_counts.tolist() == want[2]
    assert tile_map.tolist() == want[3]


def test_evict_edges_and_refusals():
    import orthocache_gpu as oc
    t, l, r = _i32([[0, 1, 2, 3, 4], [5, -1, -1, -1, -1]]), _i32([70, 3]), _i32([1] * 6)
    all_gone = torch.ones((2, 3, 2), dtype=torch.uint8, device=DEV)
    res, m = oc.evict_pages(t, l, r, all_gone, block_size=16)
    assert res.block_tables.tolist() == [[4, -1, -1, -1, -1], [5, -1, -1, -1, -1]] and res.context_lens.tolist() == [6, 3]
    assert res.ref_counts.tolist() == [0, 0, 0, 0, 1, 1] and m.tolist() == [[1, -1], [0, -1]]
    res, _ = oc.evict_pages(t, l, r, all_gone[:, :, :0], block_size=16)
    assert res.block_tables.tolist() == t.tolist() and res.ref_counts.tolist() == r.tolist()
    with pytest.raises(ValueError, match="divide"):
        oc.evict_pages(t, l, r, all_gone, block_size=128)
    with pytest.raises(TypeError, match="bool or uint8"):
        oc.evict_pages(t, l, r, all_gone.float(), block_size=16)
    with pytest.raises(ValueError, match="evict_mask"):
        oc.evict_pages(t, l, r, all_gone[:1], block_size=16)
    t[0, 4] = 9
    with pytest.raises(ValueError, match="outside"):
        oc.evict_pages(t, l, r, all_gone, block_size=16)


def test_captured_with_out():
    """Both operators in a graph between two sets of tables, replayed with the eager work of other calls between."""
    import orthocache_gpu as oc
    rng = random.Random(6)
    lens, bs, cols = [100, 130, 64, 10], 16, 12
    tables, refs, nb = _state(rng, lens, bs, cols, spare=12)
    kc, vc = _caches(nb, 2, 2, bs, 64, torch.bfloat16, 1)
    t, l, r = _i32(tables), _i32(lens), _i32(refs)
    parents = _i32([0, 1, 2, 3])
    mask = torch.zeros((4, 2, 3), dtype=torch.bool, device=DEV)

    def out():
        return oc.PageTables(torch.empty_like(t), torch.empty_like(l), torch.empty_like(r), _i32([7]))
    o1, o2 = out(), out()
    stream = torch.cuda.Stream()
    stream.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(stream):
        oc.fork_pages(kc, vc, t, l, r, parents=parents, sync=False, out=o1)
    torch.cuda.current_stream().wait_stream(stream)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        oc.fork_pages(kc, vc, t, l, r, parents=parents, sync=False, out=o1)
        _, tile_map = oc.evict_pages(o1.block_tables, o1.context_lens, o1.ref_counts, mask, block_size=bs, sync=False, out=o2)
    for p, m in (([0, 0, 2, -1], 0.5), ([3, 2, 1, 0], 0.0), ([1, 1, 1, 1], 1.0)):
        parents.copy_(_i32(p))
        mask.copy_(torch.rand(mask.shape, device=DEV) < m)
        graph.replay()
        got = [x.clone() for x in (o2.block_tables, o2.context_lens, o2.ref_counts, tile_map)]
        a = oc.fork_pages(kc, vc, t, l, r, parents=parents)
        b, tm = oc.evict_pages(a.block_tables, a.context_lens, a.ref_counts, mask, block_size=bs)
        for x, y in zip(got, (b.block_tables, b.context_lens, b.ref_counts, tm)):
            assert torch.equal(x, y)
