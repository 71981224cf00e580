"""The operators over a paged KV cache on the GPU, against a plain 64-bit form
(tests/_paged.py).  Pages hold NaN wherever no row has been written, and freed
pages (no row of theirs visible) are NaN with -1 in the block table."""
import math

import pytest
import torch

from _paged import DT, Pool, attend, rotate, sees, tolerance

pytestmark = pytest.mark.gpu


def _sa():
    import streaming_attention_b200 as sa
    return sa


def _close(got, ref, dtype, v_max, what=""):
    got = got.double().cpu()
    assert torch.isfinite(got).all(), what
    off = (got - ref).abs() - tolerance(dtype, ref, v_max)
    assert off.max().item() <= 0 if off.numel() else True, (what, off.max().item(), (got - ref).abs().max().item())


def _v_max(pool):
    return max([x.double().abs().max().item() for x in pool.v if x.numel()] + [0.0])


# ---------------------------------------------------------------- append

def _fresh(pool):
    """The pool with every page empty (NaN) and the rows still to be appended at hand."""
    pool.kp.fill_(math.nan)
    pool.vp.fill_(math.nan)
    return pool


def _check_rows(pool, b, first, k, v, exact):
    """Rows first.. of sequence b hold k, v [n, hkv, d] (float64 references; `exact`: bit for bit after rounding)."""
    for i in range(k.shape[0]):
        r = first + i
        p = pool.table_list[b][r // pool.page]
        gk, gv = pool.kp[p, :, r % pool.page].cpu(), pool.vp[p, :, r % pool.page].cpu()
        assert torch.equal(gv, v[i].to(pool.dt)), (b, r)
        if exact:
            assert torch.equal(gk, k[i].to(pool.dt)), (b, r)
        else:   # two products and a sum in fp32: off by 3 half steps of 2^-24 of 2 max|x|; then one rounding
            half_step = 2.0 ** -8 if pool.dt == torch.bfloat16 else 2.0 ** -24
            bound = k[i].abs() * half_step + 3 * 2.0 ** -24 * 2 * k[i].abs().max()
            assert ((gk.double() - k[i]).abs() <= bound).all(), (b, r)


@pytest.mark.parametrize("x_dtype,dtype", [("bf16", "bf16"), ("f32", "f32"), ("f32", "bf16"), ("bf16", "f32")])
@pytest.mark.parametrize("hq,hkv,d,page,rot,inter", [(4, 2, 128, 16, 128, False), (3, 3, 64, 32, 32, True),
                                                     (2, 1, 256, 128, 128, False), (8, 1, 128, 64, 16, True),
                                                     (5, 5, 64, 16, 64, False)])
def test_append_ragged(x_dtype, dtype, hq, hkv, d, page, rot, inter):
    sa = _sa()
    past, new = [0, 5, 31, 100, 17], [1, 40, 1, 33, 0]
    pool = _fresh(Pool([p + n for p, n in zip(past, new)], hkv, d, page, dtype, seed=d + rot))
    n, tail, pos0 = sum(new), 3, 11
    cu = torch.tensor([0] + new).cumsum(0)
    g = torch.Generator().manual_seed(5)
    qkv = torch.randn(n + tail, (hq + 2 * hkv) * d, generator=g).to(DT[x_dtype])
    dev = qkv.cuda()
    q, k, v = (x.view(n + tail, -1, d) for x in dev.split([hq * d, hkv * d, hkv * d], 1))
    cos, sin = sa.rope_table(10000.0, rot, 200)
    q_out = torch.full((n + tail, hq, d), 7.0, dtype=pool.dt, device="cuda")
    before_k, before_v = pool.kp.clone(), pool.vp.clone()
    got = sa.paged_append(k, v, pool.kp, pool.vp, pool.table, pool.kv_lens, cu_q=cu.int().cuda(), q=q, rope=(cos, sin),
                          interleaved=inter, pos0=pos0, q_out=q_out)
    torch.cuda.synchronize()
    assert got is q_out
    assert (q_out[n:] == 7.0).all()                        # rows behind the last sequence
    x = qkv.view(n + tail, hq + 2 * hkv, d)
    touched = torch.zeros(pool.kp.shape[0], page, dtype=torch.bool)
    for b in range(len(new)):
        r0, r1 = int(cu[b]), int(cu[b + 1])
        pos = pos0 + past[b] + torch.arange(new[b])
        c, s = cos.cpu()[pos], sin.cpu()[pos]
        turned = rotate(x[r0:r1, :hq + hkv], c, s, rot, inter)
        _check_rows(pool, b, past[b], turned[:, hq:], x[r0:r1, hq + hkv:], exact=False)
        half_step = 2.0 ** -8 if pool.dt == torch.bfloat16 else 2.0 ** -24
        off = (q_out[r0:r1].double().cpu() - turned[:, :hq]).abs()
        assert (off <= turned[:, :hq].abs() * half_step + 3 * 2.0 ** -24 * 2 * (turned.abs().max() if new[b] else 0)).all()
        for r in range(past[b], past[b] + new[b]):
            touched[pool.table_list[b][r // page], r % page] = True
    same = ~touched.cuda()[:, None, :, None].expand_as(pool.kp)
    for now, old in ((pool.kp, before_k), (pool.vp, before_v)):   # every other row as it was (bit for bit: NaN)
        assert torch.equal(now[same].view(torch.int16 if dtype == "bf16" else torch.int32),
                           old[same].view(torch.int16 if dtype == "bf16" else torch.int32))


def test_append_copies_without_rotation_and_in_place_queries():
    sa = _sa()
    pool = _fresh(Pool([3, 0, 17], 2, 128, 16, "bf16", seed=3))
    k, v = pool.q(3, 2).cuda(), pool.q(3, 2).cuda()
    q = pool.q(3, 4).cuda()
    keep = q.clone()
    assert sa.paged_append(k, v, pool.kp, pool.vp, pool.table, pool.kv_lens) is None
    out = sa.paged_append(k, v, pool.kp, pool.vp, pool.table, pool.kv_lens, q=q, q_out=q)
    torch.cuda.synchronize()
    _check_rows(pool, 0, 2, k[:1].cpu(), v[:1].cpu(), exact=True)
    _check_rows(pool, 2, 16, k[2:].cpu(), v[2:].cpu(), exact=True)
    assert out is q and torch.equal(q, keep)
    assert torch.isnan(pool.kp).sum() == pool.kp.numel() - 2 * 2 * 128


def test_append_reports_rows_outside_the_cache():
    sa = _sa()
    with sa.Context(0) as ctx:
        pool = _fresh(Pool([16, 16], 1, 64, 16, "f32", seed=4, pad_cols=0))
        k = pool.q(2, 1).cuda()
        for table, lens, rope_n in ((pool.table, [17, 16], None), (torch.tensor([[99], [-5]], dtype=torch.int32), [16, 16], None),
                                    (pool.table, [16, 16], 15)):
            before = pool.kp.clone()
            rope = None if rope_n is None else sa.rope_table(1e4, 64, rope_n, ctx=ctx)
            sa.paged_append(k, k, pool.kp, pool.vp, table.cuda(), torch.tensor(lens, dtype=torch.int32).cuda(), rope=rope,
                            ctx=ctx)
            with pytest.raises(sa.SAError) as e:
                ctx.synchronize()
            assert e.value.code == -6
            ctx.synchronize()                               # reported once
            if lens == [16, 16]:
                assert torch.equal(torch.isnan(before), torch.isnan(pool.kp))


def test_rope_table_of_far_positions():
    sa = _sa()
    n, rot, theta = 1 << 20, 128, 1e6
    cos, sin = sa.rope_table(theta, rot, n)
    pos = torch.tensor([0, 1, 77, 4095, 65536, n - 1], dtype=torch.float64)
    inv = theta ** (-torch.arange(0, rot, 2, dtype=torch.float64) / rot)
    ang = pos[:, None] * inv
    at = pos.long().cuda()
    # 64-bit angles of up to 2^20 radians are off by 2^-32 at most; then one rounding to fp32
    for got, ref in ((cos, ang.cos()), (sin, ang.sin())):
        assert ((got[at].double().cpu() - ref).abs() <= 2.0 ** -24 + 2.0 ** -30).all()


# ---------------------------------------------------------------- decode

LENS = [1, 0, 700, 15, 16, 17, 129, 64, 65, 333]


def _decode(pool, hq, window=0, sinks=0, scale=None, spread=1.0, q_pad=0, **kw):
    sa = _sa()
    n, d = len(pool.lens), pool.d
    scale = scale or 1.0 / math.sqrt(d)
    q = pool.q(n, hq, spread)
    qd = torch.empty(n, hq + q_pad, d, dtype=pool.dt, device="cuda")
    qd[:, :hq] = q.cuda()
    out = sa.attn_paged_decode(qd[:, :hq], pool.kp, pool.vp, pool.table, pool.kv_lens, scale, window=window, sinks=sinks, **kw)
    ref = torch.cat([attend(q[b:b + 1], pool.k[b], pool.v[b], [m - 1], scale, window, sinks) for b, m in enumerate(pool.lens)])
    return out, ref


@pytest.mark.parametrize("dtype", ["bf16", "f32"])
@pytest.mark.parametrize("d,page", [(64, 16), (64, 128), (128, 16), (128, 64), (128, 128), (256, 16), (256, 32)])
@pytest.mark.parametrize("hq,hkv", [(1, 1), (4, 2), (6, 2), (8, 1)])
def test_decode_ragged(dtype, d, page, hq, hkv):
    pool = Pool(LENS, hkv, d, page, dtype, seed=d + page + hq)
    out, ref = _decode(pool, hq)
    _close(out, ref, dtype, _v_max(pool))
    assert (out[1] == 0).all()                             # an empty sequence


@pytest.mark.parametrize("dtype", ["bf16", "f32"])
@pytest.mark.parametrize("hq,hkv", [(9, 1), (16, 1), (24, 2)])
@pytest.mark.parametrize("d", [64, 128])
def test_decode_wide_groups(dtype, hq, hkv, d):
    pool = Pool([200, 3, 0, 65], hkv, d, 16, dtype, seed=hq)
    out, ref = _decode(pool, hq)
    _close(out, ref, dtype, _v_max(pool))


@pytest.mark.parametrize("dtype,d,page", [("bf16", 128, 16), ("bf16", 64, 64), ("f32", 128, 32), ("f32", 64, 16)])
@pytest.mark.parametrize("window,sinks", [(1, 0), (1, 1), (16, 4), (100, 0), (100, 70), (64, 130), (128, 16), (5000, 4)])
def test_decode_window(dtype, d, page, window, sinks):
    pool = Pool(LENS + [1000], 2, d, page, dtype, seed=window + sinks)
    for b, n in enumerate(pool.lens):                      # pages that the query does not see have been given back
        pool.forget(b, lambda r, n=n: sees(n - 1, r, window, sinks))
    with _sa().Context(0) as ctx:
        out, ref = _decode(pool, 4, window, sinks, ctx=ctx)
        ctx.synchronize()                                  # and no freed page counts as a bad index
    _close(out, ref, dtype, _v_max(pool), (window, sinks))


@pytest.mark.parametrize("dtype", ["bf16", "f32"])
def test_decode_scores_of_all_sizes(dtype):
    """Logits with a spread of hundreds: the running maximum moves many times."""
    pool = Pool([300, 1000, 40], 2, 128, 16, dtype, seed=9)
    out, ref = _decode(pool, 4, scale=1.0 if dtype == "bf16" else 0.5, spread=2.0)
    if dtype == "f32":   # scores up to ~1500: fp32 sums of 128 products off by 2^-24 * 1500 * 8, so weights by 7e-4
        assert (out.double().cpu() - ref).abs().max() <= 1.5e-3 * _v_max(pool)
    else:                # bf16 products are exact in fp32: sums off by 2^-24 * 3000 * 8, weights by 1.5e-3
        assert ((out.double().cpu() - ref).abs() <= tolerance(dtype, ref, _v_max(pool)) + 1.5e-3 * _v_max(pool)).all()


def test_decode_many_sequences_and_few_long_ones():
    for lens, hkv, hq in (([(7 * i) % 50 for i in range(1500)], 1, 2), ([60000], 1, 1), ([3, 30000, 2], 8, 16)):
        pool = Pool(lens, hkv, 64, 16, "bf16", seed=len(lens))
        out, ref = _decode(pool, hq)
        _close(out, ref, "bf16", _v_max(pool), lens[:3])


@pytest.mark.parametrize("dtype", ["bf16", "f32"])
def test_decode_strides(dtype):
    """K and V interleaved in one pool, q and out rows wider than their heads, a wider block table."""
    pool = Pool([100, 33, 250], 2, 128, 32, dtype, seed=2, interleaved_kv=True, pad_cols=5)
    wide = torch.full((3, 6, 128), 3.0, dtype=pool.dt, device="cuda")
    out, ref = _decode(pool, 4, window=60, sinks=3, q_pad=2, out=wide[:, :4])
    _close(out, ref, dtype, _v_max(pool))
    assert (wide[:, 4:] == 3.0).all()


def test_decode_same_result_twice_and_on_another_stream():
    pool = Pool([5000, 77, 0, 1234], 4, 128, 16, "bf16", seed=6)
    sa = _sa()
    q = pool.q(4, 16).cuda()
    a = sa.attn_paged_decode(q, pool.kp, pool.vp, pool.table, pool.kv_lens, 0.1)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        b = sa.attn_paged_decode(q, pool.kp, pool.vp, pool.table, pool.kv_lens, 0.1)
        c = sa.attn_paged_decode(q, pool.kp, pool.vp, pool.table, pool.kv_lens, 0.1)
    torch.cuda.synchronize()
    assert torch.equal(a, b) and torch.equal(a, c)


def test_decode_reports_bad_pages_and_lengths():
    sa = _sa()
    with sa.Context(0) as ctx:
        pool = Pool([40, 20], 1, 64, 16, "bf16", seed=8, pad_cols=0)
        q = pool.q(2, 1).cuda()
        bad = pool.table.clone()
        bad[0, 1] = pool.kp.shape[0]
        for table, lens in ((bad, pool.kv_lens), (pool.table, pool.kv_lens + 9)):
            sa.attn_paged_decode(q, pool.kp, pool.vp, table, lens, 1.0, ctx=ctx)
            with pytest.raises(sa.SAError) as e:
                ctx.synchronize()
            assert e.value.code == -6
        good = sa.attn_paged_decode(q, pool.kp, pool.vp, pool.table, pool.kv_lens, 1.0, ctx=ctx)
        ctx.synchronize()
        assert torch.isfinite(good).all()


# ---------------------------------------------------------------- prefill

def _prefill(pool, new, hq, window=0, sinks=0, tail=0, ctx=None, scale=None, q_pad=0, spread=1.0):
    sa = _sa()
    d, n = pool.d, sum(new)
    scale = scale or 1.0 / math.sqrt(d)
    cu = torch.tensor([0] + list(new)).cumsum(0)
    q = pool.q(n + tail, hq, spread)
    qd = torch.empty(n + tail, hq + q_pad, d, dtype=pool.dt, device="cuda")
    qd[:, :hq] = q.cuda()
    out = torch.full((n + tail, hq + q_pad, d), 5.0, dtype=pool.dt, device="cuda")
    got = sa.attn_paged_prefill(qd[:, :hq], pool.kp, pool.vp, pool.table, pool.kv_lens, cu.int().cuda(), scale, window=window,
                                sinks=sinks, ctx=ctx, out=out[:, :hq])
    ref = torch.cat([attend(q[cu[b]:cu[b + 1]], pool.k[b], pool.v[b], list(range(m - new[b], m)), scale, window, sinks)
                     for b, m in enumerate(pool.lens)])
    torch.cuda.synchronize()
    assert (out[n:] == 5.0).all() and (out[:, hq:] == 5.0).all()
    return got[:n], ref


@pytest.mark.parametrize("dtype", ["bf16", "f32"])
@pytest.mark.parametrize("d,page", [(64, 16), (128, 16), (128, 32), (64, 64), (128, 128)])
@pytest.mark.parametrize("hq,hkv", [(1, 1), (4, 2), (3, 1), (8, 1), (16, 1)])
def test_prefill_ragged(dtype, d, page, hq, hkv):
    new = [1, 0, 130, 64, 5, 300]
    past = [0, 17, 0, 64, 250, 129]
    pool = Pool([a + b for a, b in zip(past, new)], hkv, d, page, dtype, seed=d + page + hq)
    out, ref = _prefill(pool, new, hq, tail=3)
    _close(out, ref, dtype, _v_max(pool))


@pytest.mark.parametrize("dtype,d,page,hq,hkv", [("bf16", 128, 16, 4, 2), ("bf16", 64, 32, 8, 1), ("bf16", 128, 128, 2, 2),
                                                 ("f32", 128, 16, 4, 2), ("f32", 64, 64, 5, 1)])
@pytest.mark.parametrize("window,sinks", [(1, 0), (1, 1), (16, 4), (100, 0), (129, 70), (64, 130), (128, 16), (300, 140),
                                          (5000, 4)])
def test_prefill_window(dtype, d, page, hq, hkv, window, sinks):
    new, past = [200, 3, 77, 1], [500, 0, 13, 300]
    pool = Pool([a + b for a, b in zip(past, new)], hkv, d, page, dtype, seed=window + sinks)
    for b, n in enumerate(pool.lens):                      # pages that none of the queries sees have been given back
        pool.forget(b, lambda r, n=n, m=new[b]: any(sees(p, r, window, sinks) for p in range(n - m, n)))
    with _sa().Context(0) as ctx:
        out, ref = _prefill(pool, new, hq, window, sinks, ctx=ctx)
        ctx.synchronize()
    _close(out, ref, dtype, _v_max(pool), (window, sinks))


@pytest.mark.parametrize("dtype", ["bf16", "f32"])
def test_prefill_lengths_around_tiles(dtype):
    """Lengths and chunk sizes around 64, 128 and the slots' sizes, many sequences in one call."""
    new, past = [], []
    for n in (1, 2, 31, 32, 33, 63, 64, 65, 127, 128, 129, 255, 256, 257):
        for p in (0, 1, 127, 128):
            new.append(n)
            past.append(p)
    pool = Pool([a + b for a, b in zip(past, new)], 1, 64, 16, dtype, seed=1)
    out, ref = _prefill(pool, new, 4, window=90, sinks=2)
    _close(out, ref, dtype, _v_max(pool))


@pytest.mark.parametrize("dtype", ["bf16", "f32"])
def test_prefill_scores_of_all_sizes(dtype):
    pool = Pool([700, 64], 1, 128, 16, dtype, seed=12)
    out, ref = _prefill(pool, [300, 64], 2, scale=1.0 if dtype == "bf16" else 0.5, spread=2.0, q_pad=1)
    # as test_decode_scores_of_all_sizes
    off = (out.double().cpu() - ref).abs()
    assert (off <= (tolerance(dtype, ref, _v_max(pool)) if dtype == "bf16" else 0) + 1.5e-3 * _v_max(pool)).all()


def test_prefill_more_sequences_than_threads():
    new = [(5 * i) % 4 for i in range(900)]
    pool = Pool([n + i % 3 for i, n in enumerate(new)], 1, 64, 16, "bf16", seed=13)
    out, ref = _prefill(pool, new, 2)
    _close(out, ref, "bf16", _v_max(pool))
    pool = Pool([n + i % 3 for i, n in enumerate(new)], 1, 64, 16, "f32", seed=13)
    out, ref = _prefill(pool, new, 2)
    _close(out, ref, "f32", _v_max(pool))


@pytest.mark.parametrize("dtype", ["bf16", "f32"])
def test_prefill_queries_before_the_first_row_get_zeros(dtype):
    """A length shorter than the chunk: the chunk's first queries lie before row 0 and see nothing."""
    sa = _sa()
    pool = Pool([40], 1, 64, 16, dtype, seed=14)
    q = pool.q(100, 2)
    out = sa.attn_paged_prefill(q.cuda(), pool.kp, pool.vp, pool.table, pool.kv_lens,
                                torch.tensor([0, 100], dtype=torch.int32).cuda(), 0.125)
    torch.cuda.synchronize()
    assert (out[:60] == 0).all()
    _close(out[60:], attend(q[60:], pool.k[0], pool.v[0], range(40), 0.125), dtype, _v_max(pool))


@pytest.mark.parametrize("dtype", ["bf16", "f32"])
def test_prefill_reports_bad_pages_and_token_ranges(dtype):
    sa = _sa()
    with sa.Context(0) as ctx:
        pool = Pool([40, 20], 1, 64, 16, dtype, seed=8, pad_cols=0)
        q = pool.q(10, 1).cuda()
        bad = pool.table.clone()
        bad[0, 1] = -7
        good_cu = torch.tensor([0, 5, 10], dtype=torch.int32).cuda()
        for table, lens, cu in ((bad, pool.kv_lens, good_cu), (pool.table, pool.kv_lens + 9, good_cu),
                                (pool.table, pool.kv_lens, good_cu + 1), (pool.table, pool.kv_lens, -good_cu)):
            sa.attn_paged_prefill(q, pool.kp, pool.vp, table, lens, cu, 1.0, ctx=ctx)
            with pytest.raises(sa.SAError) as e:
                ctx.synchronize()
            assert e.value.code == -6
        sa.attn_paged_prefill(q, pool.kp, pool.vp, pool.table, pool.kv_lens, good_cu, 1.0, ctx=ctx)
        ctx.synchronize()


# ---------------------------------------------------------------- shared prefix

def _prefix(lens, prefix, hq, hkv, d, page, dtype, seed=0, scale=None, spread=1.0, interleaved_kv=False, ctx=None):
    """The pool's first sequence is the prefix, the others the batch."""
    sa = _sa()
    pool = Pool([prefix] + list(lens), hkv, d, page, dtype, seed=seed, interleaved_kv=interleaved_kv)
    scale = scale or 1.0 / math.sqrt(d)
    n = len(lens)
    q = pool.q(n, hq, spread)
    out = sa.attn_paged_decode_prefix(q.cuda(), pool.kp, pool.vp, pool.table[0], prefix, pool.table[1:], pool.kv_lens[1:],
                                      scale, ctx=ctx)
    ref = torch.cat([attend(q[b:b + 1], torch.cat([pool.k[0], pool.k[b + 1]], 1), torch.cat([pool.v[0], pool.v[b + 1]], 1),
                            [prefix + m - 1], scale) for b, m in enumerate(lens)])
    return out, ref, _v_max(pool)


@pytest.mark.parametrize("dtype", ["bf16", "f32"])
@pytest.mark.parametrize("d,page", [(64, 16), (128, 16), (128, 128), (64, 32)])
@pytest.mark.parametrize("hq,hkv,n", [(1, 1, 1), (4, 2, 4), (16, 2, 17), (3, 1, 90), (2, 1, 65), (16, 1, 25)])
def test_prefix(dtype, d, page, hq, hkv, n):
    lens = [(37 * i) % 90 for i in range(n)]               # 0 among them
    out, ref, v_max = _prefix(lens, 333, hq, hkv, d, page, dtype, seed=n)
    _close(out, ref, dtype, v_max)


@pytest.mark.parametrize("dtype", ["bf16", "f32"])
@pytest.mark.parametrize("prefix", [0, 1, 15, 16, 64, 127, 128, 129, 256, 5000])
def test_prefix_lengths(dtype, prefix):
    out, ref, v_max = _prefix([0, 5, 200, 1, 64], prefix, 4, 2, 128, 16, dtype, seed=prefix)
    _close(out, ref, dtype, v_max)
    if prefix == 0:
        assert (out[0] == 0).all()                         # nothing to see at all


@pytest.mark.parametrize("dtype", ["bf16", "f32"])
def test_prefix_long_own_rows_and_large_batches(dtype):
    out, ref, v_max = _prefix([9000, 0, 3], 700, 8, 2, 128, 16, dtype, seed=1, interleaved_kv=True)
    _close(out, ref, dtype, v_max)
    out, ref, v_max = _prefix([i % 5 for i in range(700)], 257, 2, 1, 64, 16, dtype, seed=2)
    _close(out, ref, dtype, v_max)


@pytest.mark.parametrize("dtype", ["bf16", "f32"])
def test_prefix_reports_bad_pages(dtype):
    sa = _sa()
    with sa.Context(0) as ctx:
        pool = Pool([40, 20], 1, 64, 16, dtype, seed=8)
        q = pool.q(1, 1).cuda()
        bad = pool.table[0].clone()
        bad[2] = 1 << 20
        sa.attn_paged_decode_prefix(q, pool.kp, pool.vp, bad, 40, pool.table[1:], pool.kv_lens[1:], 1.0, ctx=ctx)
        with pytest.raises(sa.SAError) as e:
            ctx.synchronize()
        assert e.value.code == -6
        sa.attn_paged_decode_prefix(q, pool.kp, pool.vp, pool.table[0], 40, pool.table[1:], pool.kv_lens[1:], 1.0, ctx=ctx)
        ctx.synchronize()
