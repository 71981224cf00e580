"""Sequences in which every page shows in the attention's result, however many
rows there are.

Each column of V but the last eight belongs to one stretch of consecutive rows:
values 1..2 there and zeros elsewhere.  The last eight columns belong to single
rows (the first, the last, and rows next to tile edges), with values as large as
the number of rows.  So a page, a tile or a CTA's share that is lost, taken twice
or weighted wrongly moves some column by far more than the bound below, which a
test on the CPU asserts for the very inputs that the GPU tests use."""
import math

import torch

EDGES = (0, -1, 15, 16, 63, 64, 127, 128)


def marked_values(n, hkv, d, dt, gen, cols=None, size=1.0, edges=True):
    v = torch.zeros(hkv, n, d, dtype=dt)
    seg = d - len(EDGES)
    cols = torch.arange(seg) if cols is None else cols
    r = torch.arange(n)
    v[:, r, cols[r * len(cols) // max(n, 1)]] = (size * (1 + torch.randint(0, 128, (hkv, n), generator=gen) / 128)).to(dt)
    for c, e in enumerate(EDGES if edges else ()):
        if n and -n <= e < n:
            v[:, e, seg + c] = float(n)
    return v


def mark(pool, prefix=False, seed=7):
    """Replaces the values of every sequence of the pool by marked ones.  prefix: the first sequence comes before each of
    the others; it has every other column, and their values are larger as their rows are fewer."""
    gen = torch.Generator().manual_seed(seed)
    seg = torch.arange(pool.d - len(EDGES))
    for b, n in enumerate(pool.lens):
        if not prefix:
            kw = {}
        elif b == 0:
            kw = dict(cols=seg[::2])
        else:
            kw = dict(cols=seg[1::2], size=2.0 ** round(math.log2((pool.lens[0] + n) / max(n, 1))), edges=False)
        pool.v[b] = marked_values(n, pool.hkv, pool.d, pool.dt, gen, **kw)
        rows = torch.arange(n)
        page = torch.tensor(pool.table_list[b], dtype=torch.long)[rows // pool.page] if n else rows
        pool.vp[page.to(pool.vp.device), :, (rows % pool.page).to(pool.vp.device)] = \
            pool.v[b].transpose(0, 1).to(pool.vp.device)
    return pool


def bound(dtype, ref, rows):
    """How far a result may be from the 64-bit one, entry by entry, where no value is negative: the weighted sum of the
    values' magnitudes is the result itself.

    bf16: each weight's rounding 2^-8 of it, so 2^-8 of the sum, and the output's rounding 2^-8 of it.  Both types: fp32
    sums of up to `rows` terms one after the other, 2^-24 each, and another 300 half steps for a score's 128 products
    and its exponential (scores here are below 8) and for joins."""
    return ref.abs() * ((2 * 2.0 ** -8 if dtype == "bf16" else 0.0) + (rows + 300) * 2.0 ** -24)


def least_shift(dtype, q, k, v, scale, rows, group):
    """q [d] over rows k, v [n, d] in float64, of which those in `rows` (a sorted index) are seen: the smallest ratio to
    the bound that losing, or counting twice, one group of `group` consecutive rows makes in the column that it moves
    most."""
    q, k, v = q.double(), k[rows].double(), v[rows].double()
    w = torch.softmax(k @ q * scale, 0)
    ref = w @ v
    limit = bound(dtype, ref, len(rows)) + 1e-30
    name = rows // group
    first = torch.unique(name, return_inverse=True)[1]
    n = int(first.max()) + 1
    den = torch.zeros(n, dtype=torch.float64).index_add_(0, first, w)
    num = torch.zeros(n, v.shape[1], dtype=torch.float64).index_add_(0, first, w[:, None] * v)
    lost = (ref - num) / (1 - den).clamp(min=1e-12)[:, None]
    twice = (ref + num) / (1 + den)[:, None]
    ratio = [((x - ref).abs() / limit).amax(1).min().item() for x in ([lost, twice] if n > 1 else [twice * 0])]
    return min(ratio)
