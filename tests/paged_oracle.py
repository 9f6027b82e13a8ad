"""Plain float64 / Python restatements of the operators around a paged cache,
from their definitions, and the error bounds of their float32 kernels."""

import math

import torch

TILE = 64


def half_step(dt):
    """The largest relative error of one rounding to dt."""
    return torch.finfo(dt).eps / 2


# ------------------------------------------------------------ rotary

def turn(x, positions, inv_freq, scale=1.0, layout="half", backward=False):
    """x (..., tokens, d) float64 by positions (..., tokens)."""
    rot = 2 * inv_freq.shape[0]
    a = positions.double()[..., None] * inv_freq.double()
    if backward:
        a = -a
    c, s = a.cos() * scale, a.sin() * scale
    y = x.clone()
    if layout == "half":
        i0, i1 = slice(0, rot // 2), slice(rot // 2, rot)
    else:
        i0, i1 = slice(0, rot, 2), slice(1, rot, 2)
    y[..., i0] = x[..., i0] * c - x[..., i1] * s
    y[..., i1] = x[..., i1] * c + x[..., i0] * s
    return y


def turn_bound(x, y, dt, rot, layout, scale=1.0):
    """|error| of turning x to y: the rounding to dt, and 2^-20 of the pair's
    size for the float32 sine, cosine (2^-22 each, their arguments 2^-23 of half
    a turn: pi 2^-23) and products (2^-23)."""
    mag = x.abs()
    pair = mag.clone()
    if layout == "half":
        m = mag[..., :rot // 2] + mag[..., rot // 2:rot]
        pair[..., :rot // 2], pair[..., rot // 2:rot] = m, m
    else:
        m = mag[..., 0:rot:2] + mag[..., 1:rot:2]
        pair[..., 0:rot:2], pair[..., 1:rot:2] = m, m
    tiny = torch.finfo(dt).tiny * torch.finfo(dt).eps
    return half_step(dt) * y.abs() + 2.0 ** -20 * abs(scale) * pair + tiny


# ------------------------------------------------------------ attention

def attention(q, k, v, place, *, scale, softcap=0.0, slopes=None, window=0, prefix=0, seen_more=None, p_step=0.0,
              p_tiny=0.0):
    """One head in float64: q (n, d) at places `place` (n,), k, v (m, d).
    seen_more (n, m): further conditions.  Returns (out, bound): the bound of
    a float32 kernel's error before its output's rounding, per element.

    With dz_j the error of score j (its dot product's d + 4 roundings, the cap's
    exponential and reciprocal, the bias), a weight is off by the factor
    exp(2 max dz), rounded by p_step, and the output by sum p_j (2 dz_j + p_step +
    2^-18) (|v_j| + |out|), the last term for sums of up to 2^18 / 64 tiles."""
    q, k, v = q.double(), k.double(), v.double()
    n, m, d = q.shape[0], k.shape[0], q.shape[1]
    j = torch.arange(m, device=q.device)
    dist = place[:, None] - j[None, :]
    seen = (dist >= 0)
    if window > 0:
        seen = seen & (dist < window)
    seen = seen | (j[None, :] < prefix)
    if seen_more is not None:
        seen = seen & seen_more
    # what is not seen has no effect: nothing of it enters the oracle
    any_seen = seen.any(0)
    k = torch.where(any_seen[:, None], k, 0.0)
    v = torch.where(any_seen[:, None], v, 0.0)
    z = (q @ k.T) * scale
    dz = (d + 4) * 2.0 ** -24 * (q.abs() @ k.abs().T) * abs(scale)
    if softcap > 0:
        z = softcap * torch.tanh(z / softcap)
        dz = dz + softcap * 2.0 ** -21
    if slopes is not None:
        z = z - slopes * dist.abs()
        dz = dz + 2.0 ** -22 * abs(float(slopes)) * dist.abs()
    dz = dz + 2.0 ** -22 * z.abs()
    z = torch.where(seen, z, -math.inf)
    top = z.amax(1, keepdim=True) if m else torch.zeros((n, 1), dtype=torch.float64, device=q.device)
    none = ~seen.any(1, keepdim=True)
    p = torch.where(seen, torch.exp(z - torch.where(none, 0.0, top)), 0.0)
    dz = dz + 2.0 ** -22 * torch.where(none, 0.0, top).abs()
    l = p.sum(1, keepdim=True)
    w = torch.where(none, 0.0, p / torch.where(none, 1.0, l))
    out = torch.zeros((n, d), dtype=torch.float64, device=q.device)
    bound = torch.zeros_like(out)
    step = w * (2 * dz + p_step + 2.0 ** -18)
    for r in range(n):  # only the tokens that the row sees: the others' values may be NaN
        at = seen[r]
        out[r] = w[r, at] @ v[at]
        bound[r] = step[r, at] @ v[at].abs() + step[r, at].sum() * out[r].abs() + p_tiny * v[at].abs().sum(0)
    return out, bound


def check_out(got, want, bound, what=""):
    """got (any float type) within the bound plus its own rounding."""
    dt = got.dtype
    g = got.double()
    tol = bound + half_step(dt) * (want.abs() + bound) + torch.finfo(dt).tiny * torch.finfo(dt).eps
    assert torch.equal(torch.isnan(g), torch.isnan(want)), f"{what}: NaN in other places"
    inf = torch.isinf(want)
    assert torch.equal(g[inf], want[inf]), f"{what}: infinities differ"
    ok = ~(torch.isnan(want) | inf)
    over = ((g - want).abs() - tol)[ok]
    assert over.numel() == 0 or float(over.max()) <= 0.0, \
        f"{what}: {float((g - want).abs()[ok].max()):.3g} off, {float(over.max()):.3g} over the bound"


# ------------------------------------------------------------ pages

def fork(tables, lens, refs, parents, fresh, bs, cols):
    """(tables, lens, refs, copies, ok): lists; copies are (source, target, tokens)."""
    n = len(tables)
    new_t, new_l, copies = [], [], []
    free = [b for b, r in enumerate(refs) if r == 0]
    taken = 0
    first = {}
    for i, s in enumerate(parents):
        if s >= 0:
            first.setdefault(s, i)
    for i, s in enumerate(parents):
        if s < 0:
            new_t.append([-1] * cols)
            new_l.append(0)
            continue
        m = max(lens[s], 0)
        need = -(-(m + fresh[i]) // bs)
        row = list(tables[s][:m // bs])
        if m % bs:
            last = tables[s][m // bs]
            if first[s] == i and refs[last] <= 1:
                row.append(last)
            else:
                if taken >= len(free):
                    return None
                copies.append((last, free[taken], m % bs))
                row.append(free[taken])
                taken += 1
        while len(row) < need:
            if taken >= len(free):
                return None
            row.append(free[taken])
            taken += 1
        new_t.append(row + [-1] * (cols - len(row)))
        new_l.append(m)
    out = list(refs)
    for row in tables:
        for b in row:
            if b >= 0:
                out[b] -= 1
    for row in new_t:
        for b in row:
            if b >= 0:
                out[b] += 1
    return new_t, new_l, out, copies


def evict(tables, lens, refs, mask, bs, cols):
    """mask[b][t]: whether every head evicts tile t (True past its columns: False)."""
    per = TILE // bs
    tiles_cols = -(-cols * bs // TILE)
    new_t, new_l, maps = [], [], []
    for row, n, gone in zip(tables, lens, mask):
        n = min(max(n, 0), cols * bs)
        tiles = -(-n // TILE)
        kept = [t for t in range(tiles) if not (t < n // TILE and t < len(gone) and gone[t])]
        out = []
        for t in kept:
            out += [row[c] for c in range(t * per, min((t + 1) * per, -(-n // bs)))]
        new_t.append(out + [-1] * (cols - len(out)))
        new_l.append(n - TILE * (tiles - len(kept)))
        maps.append(kept + [-1] * (tiles_cols - len(kept)))
    count = list(refs)
    for row in tables:
        for b in row:
            if b >= 0:
                count[b] -= 1
    for row in new_t:
        for b in row:
            if b >= 0:
                count[b] += 1
    return new_t, new_l, count, maps
