"""bf16 prefills long enough for the tensor-core kernel's two slots (each 128
query rows of its own over the same keys), and short ones whose slots share the
rows and take alternate key tiles.  Which of the two runs follows from the
units and the GPU's SMs; the tests assert it.  Marked values as in
tests/_paged_marks.py: a lost or doubled page shows."""
import pytest
import torch

from _paged import Pool, attend
from _paged_marks import bound, least_shift, mark

# new, past, hq, hkv, d, page, window, sinks
TWO_SLOTS = [([2400], [0], 16, 8, 128, 16, 0, 0),
             ([1500, 1100, 37], [0, 700, 2000], 32, 8, 128, 16, 0, 0),
             ([2000, 1300], [300, 0], 16, 8, 128, 128, 700, 200),         # first tokens across a tile's edge
             ([1290, 1153, 0, 65], [0, 129, 50, 1], 24, 8, 128, 64, 333, 5),   # three heads: 42 tokens a tile
             ([1100, 64, 1000], [70, 3000, 0], 16, 4, 128, 32, 0, 0),
             ([700, 800], [2, 0], 64, 4, 128, 16, 1, 0),                  # sixteen heads, each token sees itself
             ([1900, 5, 1200], [100, 0, 3], 12, 6, 64, 16, 0, 0),
             ([3000, 1], [0, 4000], 12, 6, 64, 128, 900, 140),
             ([2500], [0], 8, 8, 64, 16, 4000, 3)]
ONE_ROW_TILE = [([40], [9000], 4, 2, 128, 16, 0, 0), ([1, 3], [12000, 5], 16, 8, 128, 128, 0, 0),
                ([300], [5000], 8, 2, 64, 32, 3001, 130), ([17, 64], [3000, 6000], 8, 1, 128, 16, 0, 0)]
SPREAD = 0.25


def _two_slots(case, sms):
    """The launch's rule: units of one row tile that do not fit the GPU at once."""
    new, _, hq, hkv = case[:4]
    n, tokens = sum(new), 128 // (hq // hkv)
    return (n // tokens + min(len(new), n)) * hkv > sms


def _inputs(case, device):
    new, past, hq, hkv, d, page = case[:6]
    pool = mark(Pool([a + b for a, b in zip(past, new)], hkv, d, page, "bf16", seed=sum(new) + d, device=device))
    return pool, pool.q(sum(new), hq, SPREAD)


@pytest.mark.parametrize("case", TWO_SLOTS + ONE_ROW_TILE, ids=str)
def test_every_page_shows(case):
    new, past, hq, hkv, d, page, window, sinks = case
    pool, q = _inputs(case, "cpu")
    at = 0
    for b, n in enumerate(pool.lens):
        for t in {0, new[b] // 2, new[b] - 1}:
            p = n - new[b] + t
            if 0 <= t < new[b] and p > 32 and window != 1:
                r = torch.arange(p + 1)
                r = r[(r > p - window) | (r < sinks)] if window else r
                h = (b + t) % hq
                # where few rows share a column, one of its rows; where many do, a page
                assert least_shift("bf16", q[at + t, h], pool.k[b][h * hkv // hq], pool.v[b][h * hkv // hq], d ** -0.5, r,
                                   16) > 1, (b, t)
        at += new[b]


@pytest.mark.gpu
@pytest.mark.parametrize("case", TWO_SLOTS + ONE_ROW_TILE, ids=str)
def test_prefill_variants(case):
    import streaming_attention_b200 as sa
    new, past, hq, hkv, d, page, window, sinks = case
    with sa.Context(0) as ctx:
        assert _two_slots(case, ctx.num_sms) == (case in TWO_SLOTS)
        pool, q = _inputs(case, "cuda")
        if window:                                             # pages that no token of the chunk sees are given back
            for b, n in enumerate(pool.lens):
                first = n - new[b]
                pool.forget(b, lambda r: new[b] > 0 and (r < sinks or r > first - window))
        cu = torch.tensor([0] + new).cumsum(0)
        out = torch.full((q.shape[0] + 2, hq, d), 5.0, dtype=torch.bfloat16, device="cuda")
        qd = torch.cat([q, q[:2]]).cuda()
        sa.attn_paged_prefill(qd, pool.kp, pool.vp, pool.table, pool.kv_lens, cu.int().cuda(), d ** -0.5, window=window,
                              sinks=sinks, ctx=ctx, out=out)
        ctx.synchronize()
    out = out.cpu()
    assert (out[-2:] == 5.0).all() and torch.isfinite(out.float()).all()
    for b, n in enumerate(pool.lens):
        r = slice(int(cu[b]), int(cu[b + 1]))
        ref = attend(q[r], pool.k[b], pool.v[b], list(range(n - new[b], n)), d ** -0.5, window, sinks)
        off = (out[r].double() - ref).abs() - bound("bf16", ref, n)
        assert not off.numel() or off.max().item() <= 0, (b, off.max().item())


@pytest.mark.gpu
@pytest.mark.parametrize("hq,hkv,d", [(16, 8, 128), (12, 6, 64)])
def test_a_slot_before_the_first_row_beside_one_with_rows(hq, hkv, d):
    """A chunk longer than its sequence: the CTA that holds row 0 has a first slot of tokens that see nothing, whose
    queries are loaded all the same; they get zeros, and the second slot its results."""
    import streaming_attention_b200 as sa
    new, n = 2600, 985
    case = ([new], [0], hq, hkv, d, 16, 0, 0)
    per, first = 128 // (hq // hkv), new - n                     # tokens of a slot; the token at row 0
    assert first // per % 2 == 1 and first % per
    with sa.Context(0) as ctx:
        assert _two_slots(case, ctx.num_sms)
        pool = mark(Pool([n], hkv, d, 16, "bf16", seed=5))
        q = pool.q(new, hq, SPREAD)
        cu = torch.tensor([0, new], dtype=torch.int32, device="cuda")
        for _ in range(20):
            out = sa.attn_paged_prefill(q.cuda(), pool.kp, pool.vp, pool.table, pool.kv_lens, cu, d ** -0.5, ctx=ctx)
            ctx.synchronize()
            assert (out[:first] == 0).all()
    ref = attend(q[first:], pool.k[0], pool.v[0], list(range(n)), d ** -0.5)
    assert ((out[first:].double().cpu() - ref).abs() <= bound("bf16", ref, n)).all()
