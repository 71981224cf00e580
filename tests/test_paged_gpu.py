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


@pytest.mark.parametrize("hq,hkv,d,page", [(5, 1, 64, 16), (16, 2, 128, 32), (14, 2, 256, 16), (16, 1, 64, 64), (22, 2, 128, 16)])
@pytest.mark.parametrize("window,sinks", [(1, 0), (40, 3), (0, 0), (200, 70)])
def test_decode_f32_many_heads(hq, hkv, d, page, window, sinks):
    """More than four heads per KV head: masked rows inside a block of eight, freed pages, NaN behind the end."""
    pool = Pool(LENS + [1000], hkv, d, page, "f32", seed=hq + sinks)
    for b, n in enumerate(pool.lens):
        pool.forget(b, lambda r, n=n: sees(n - 1, r, window, sinks))
    out, ref = _decode(pool, hq, window, sinks, q_pad=1)
    _close(out, ref, "f32", _v_max(pool), (window, sinks))


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


@pytest.mark.parametrize("hq,hkv,new,past", [(28, 14, [1100, 1001], [0, 70]), (32, 4, [700, 613, 500], [64, 0, 33]),
                                             (24, 8, [900], [10]), (128, 8, [290, 0, 260], [100, 7, 0])])
@pytest.mark.parametrize("window,sinks", [(0, 0), (150, 5)])
def test_prefill_f32_long_chunks(hq, hkv, new, past, window, sinks):
    """Chunks long enough for the widest row tile of fp32."""
    pool = Pool([a + b for a, b in zip(past, new)], hkv, 128, 16, "f32", seed=hq)
    out, ref = _prefill(pool, new, hq, window, sinks, tail=2)
    _close(out, ref, "f32", _v_max(pool))


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


@pytest.mark.parametrize("hq,hkv,n", [(4, 2, 60), (3, 1, 80), (16, 1, 7), (1, 1, 500)])
def test_prefix_f32_many_rows(hq, hkv, n):
    """Rows that fill the widest row tile of fp32."""
    for prefix in (1, 700):
        out, ref, v_max = _prefix([(37 * i) % 90 for i in range(n)], prefix, hq, hkv, 128, 16, "f32", seed=n)
        _close(out, ref, "f32", v_max)


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


def test_a_bad_page_fails_no_later_call():
    """Bad pages are reported once; other operators on the context go on."""
    sa = _sa()
    with sa.Context(0) as ctx:
        pool = Pool([40], 1, 64, 16, "f32", seed=8, pad_cols=0)
        q = pool.q(1, 1).cuda()
        sa.attn_paged_decode(q, pool.kp, pool.vp, pool.table + 1000, pool.kv_lens, 1.0, ctx=ctx)
        k = torch.randn(1, 50, 64, device="cuda")
        out = sa.attn_decode(q[0], k, k, 1.0, ctx=ctx)
        good = sa.attn_paged_decode(q, pool.kp, pool.vp, pool.table, pool.kv_lens, 1.0, ctx=ctx)
        with pytest.raises(sa.SAError):
            ctx.synchronize()
        assert torch.isfinite(out).all() and torch.isfinite(good).all()


@pytest.mark.parametrize("power", [-70, 100])
def test_f32_magnitudes(power):
    """Values of 2^-70 and 2^100 through the fp32 products keep their precision: the exact scaled result."""
    sa = _sa()
    pool = Pool([300, 40, 130, 77], 1, 128, 16, "f32", seed=21)
    pool.vp.mul_(2.0 ** power)
    new = [100, 40, 0, 3]
    cu = torch.tensor([0] + new).cumsum(0)
    scale = 1.0 / math.sqrt(128)
    q = pool.q(sum(new), 8)
    out = sa.attn_paged_prefill(q.cuda(), pool.kp, pool.vp, pool.table, pool.kv_lens, cu.int().cuda(), scale)
    ref = torch.cat([attend(q[cu[b]:cu[b + 1]], pool.k[b], pool.v[b], list(range(m - new[b], m)), scale)
                     for b, m in enumerate(pool.lens)])
    _close(out.double() * 2.0 ** -power, ref, "f32", _v_max(pool))
    out = sa.attn_paged_decode(q[:4].cuda(), pool.kp, pool.vp, pool.table, pool.kv_lens, scale)
    ref = torch.cat([attend(q[b:b + 1], pool.k[b], pool.v[b], [m - 1], scale) for b, m in enumerate(pool.lens)])
    _close(out.double() * 2.0 ** -power, ref, "f32", _v_max(pool))


# ---------------------------------------------------------------- together

def _rope_ref(cos, sin, rot, x, pos, dt):
    return rotate(x, cos.cpu()[pos], sin.cpu()[pos], rot, False).to(dt)


@pytest.mark.parametrize("dtype", ["bf16", "f32"])
@pytest.mark.parametrize("window,sinks", [(0, 0), (70, 4)])
def test_serving_a_batch(dtype, window, sinks):
    """Three prompts in ragged chunks, then decode steps, through append and the two attentions: every output
    against a plain cache of the same tokens."""
    sa = _sa()
    hq, hkv, d, page, dt = 4, 2, 64, 16, DT[dtype]
    prompts, steps = [90, 33, 150], 5
    max_pages = 12
    g = torch.Generator().manual_seed(3)
    kp = torch.full((40, hkv, page, d), math.nan, dtype=dt, device="cuda")
    vp = kp.clone()
    table = torch.randperm(40, generator=g)[:36].reshape(3, max_pages).int().cuda()
    cos, sin = sa.rope_table(1e4, d, 400)
    plain_k, plain_v = [torch.zeros(hkv, 0, d, dtype=dt) for _ in prompts], [torch.zeros(hkv, 0, d, dtype=dt) for _ in prompts]
    lens, left = [0, 0, 0], list(prompts)
    v_max = 5.0
    while any(left):
        new = [min(x, n) for x, n in zip(left, (64, 17, 100))]
        lens = [a + b for a, b in zip(lens, new)]
        left = [a - b for a, b in zip(left, new)]
        n = sum(new)
        qkv = torch.randn(n, hq + 2 * hkv, d, generator=g).to(dt)
        dev = qkv.cuda()
        cu = torch.tensor([0] + new).cumsum(0)
        kv = torch.tensor(lens, dtype=torch.int32).cuda()
        q = sa.paged_append(dev[:, hq:hq + hkv], dev[:, hq + hkv:], kp, vp, table, kv, cu_q=cu.int().cuda(), q=dev[:, :hq],
                            rope=(cos, sin))
        out = sa.attn_paged_prefill(q, kp, vp, table, kv, cu.int().cuda(), d ** -0.5, window=window, sinks=sinks)
        torch.cuda.synchronize()
        for b in range(3):
            r, pos = slice(int(cu[b]), int(cu[b + 1])), torch.arange(lens[b] - new[b], lens[b])
            plain_k[b] = torch.cat([plain_k[b], _rope_ref(cos, sin, d, qkv[r, hq:hq + hkv], pos, dt).transpose(0, 1)], 1)
            plain_v[b] = torch.cat([plain_v[b], qkv[r, hq + hkv:].transpose(0, 1)], 1)
            ref = attend(q[r].cpu(), plain_k[b], plain_v[b], pos, d ** -0.5, window, sinks)
            _close(out[r], ref, dtype, v_max)
    for _ in range(steps):
        lens = [x + 1 for x in lens]
        kv = torch.tensor(lens, dtype=torch.int32).cuda()
        qkv = torch.randn(3, hq + 2 * hkv, d, generator=g).to(dt)
        dev = qkv.cuda()
        q = sa.paged_append(dev[:, hq:hq + hkv], dev[:, hq + hkv:], kp, vp, table, kv, q=dev[:, :hq], rope=(cos, sin))
        out = sa.attn_paged_decode(q, kp, vp, table, kv, d ** -0.5, window=window, sinks=sinks)
        torch.cuda.synchronize()
        for b in range(3):
            pos = torch.tensor([lens[b] - 1])
            plain_k[b] = torch.cat([plain_k[b], _rope_ref(cos, sin, d, qkv[b:b + 1, hq:hq + hkv], pos, dt).transpose(0, 1)], 1)
            plain_v[b] = torch.cat([plain_v[b], qkv[b:b + 1, hq + hkv:].transpose(0, 1)], 1)
            _close(out[b:b + 1], attend(q[b:b + 1].cpu(), plain_k[b], plain_v[b], [lens[b] - 1], d ** -0.5, window, sinks),
                   dtype, v_max)


@pytest.mark.parametrize("dtype", ["bf16", "f32"])
def test_beams_behind_a_prompt(dtype):
    """Four continuations of one prompt: the prompt prefilled once, their own tokens appended behind it."""
    sa = _sa()
    hq, hkv, d, page, dt, n = 8, 2, 128, 32, DT[dtype], 4
    P = 205
    pool = Pool([P], hkv, d, page, dtype, seed=21, extra_pages=12)
    cos, sin = sa.rope_table(1e4, d, 400)
    own = torch.tensor(pool.free[:8], dtype=torch.int32).reshape(n, 2).cuda()
    plain_k, plain_v = torch.zeros(n, hkv, 0, d, dtype=dt), torch.zeros(n, hkv, 0, d, dtype=dt)
    for step in range(1, 36):
        qkv = torch.randn(n, hq + 2 * hkv, d, generator=pool.gen).to(dt)
        dev = qkv.cuda()
        kv = torch.full((n,), step, dtype=torch.int32, device="cuda")
        q = sa.paged_append(dev[:, hq:hq + hkv], dev[:, hq + hkv:], pool.kp, pool.vp, own, kv, q=dev[:, :hq], rope=(cos, sin),
                            pos0=P)
        plain_k = torch.cat([plain_k, _rope_ref(cos, sin, d, qkv[:, hq:hq + hkv], torch.full((n,), P + step - 1), dt)[:, :, None]], 2)
        plain_v = torch.cat([plain_v, qkv[:, hq + hkv:][:, :, None]], 2)
        if step in (1, 2, 32, 33, 35):
            out = sa.attn_paged_decode_prefix(q, pool.kp, pool.vp, pool.table[0], P, own, kv, d ** -0.5)
            torch.cuda.synchronize()
            for b in range(n):
                ref = attend(q[b:b + 1].cpu(), torch.cat([pool.k[0], plain_k[b]], 1), torch.cat([pool.v[0], plain_v[b]], 1),
                             [P + step - 1], d ** -0.5)
                _close(out[b:b + 1], ref, dtype, max(_v_max(pool), 6.0), (step, b))


@pytest.mark.parametrize("dtype", ["bf16", "f32"])
def test_captured_calls_follow_lengths_and_tables(dtype):
    """A captured step replayed after the lengths, the tables and the rows changed; two graphs with their own
    workspaces replayed on two streams at once."""
    sa = _sa()
    pool = Pool([500, 40, 900], 2, 64, 16, dtype, seed=30, extra_pages=70, pad_cols=10)
    q = pool.q(3, 4)
    qd = q.cuda()
    kv, table = pool.kv_lens.clone(), pool.table.clone()
    tok = pool.q(7, 4)
    tokd, cu = tok.cuda(), torch.tensor([0, 3, 4, 7], dtype=torch.int32).cuda()

    def step():
        return (sa.attn_paged_decode(qd, pool.kp, pool.vp, table, kv, 0.125, window=300, sinks=2),
                sa.attn_paged_prefill(tokd, pool.kp, pool.vp, table, kv, cu, 0.125),
                sa.attn_paged_decode_prefix(qd, pool.kp, pool.vp, pool.table[0], 500, table, kv, 0.125))

    side = torch.cuda.Stream()
    graphs, outs = [], []
    with torch.cuda.stream(side):
        step()
        torch.cuda.synchronize()
        for _ in range(2):
            g = torch.cuda.CUDAGraph()
            with torch.cuda.graph(g, stream=side):
                outs.append(step())
            graphs.append(g)
    other = torch.cuda.Stream()
    for lens in ([500, 40, 900], [17, 0, 640], [499, 39, 1]):
        kv.copy_(torch.tensor(lens, dtype=torch.int32))
        table.copy_(pool.table)
        torch.cuda.synchronize()
        for _ in range(3):
            with torch.cuda.stream(side):
                graphs[0].replay()
            with torch.cuda.stream(other):
                graphs[1].replay()
        torch.cuda.synchronize()
        dec = torch.cat([attend(q[b:b + 1], pool.k[b][:, :n], pool.v[b][:, :n], [n - 1], 0.125, 300, 2) for b, n in enumerate(lens)])
        new = [3, 1, 3]
        at = [0, 3, 4, 7]
        pre = torch.cat([attend(tok[at[b]:at[b + 1]], pool.k[b][:, :n], pool.v[b][:, :n], list(range(n - new[b], n)), 0.125)
                         for b, n in enumerate(lens)])
        fix = torch.cat([attend(q[b:b + 1], torch.cat([pool.k[0], pool.k[b][:, :n]], 1), torch.cat([pool.v[0], pool.v[b][:, :n]], 1),
                                [500 + n - 1], 0.125) for b, n in enumerate(lens)])
        for o in outs:
            for got, ref in zip(o, (dec, pre, fix)):
                _close(got, ref, dtype, _v_max(pool), lens)
    del graphs


def test_out_may_be_the_queries():
    sa = _sa()
    for dtype in ("bf16", "f32"):
        pool = Pool([700, 33], 2, 128, 16, dtype, seed=31)
        q, t = pool.q(2, 8).cuda(), pool.q(300, 8).cuda()
        cu = torch.tensor([0, 280, 300], dtype=torch.int32).cuda()
        args = (pool.kp, pool.vp, pool.table, pool.kv_lens)
        for f in (lambda x, o: sa.attn_paged_decode(x, *args, 0.1, out=o),
                  lambda x, o: sa.attn_paged_decode_prefix(x, pool.kp, pool.vp, pool.table[0], 650, pool.table, pool.kv_lens, 0.1, out=o)):
            want, got = f(q, None), q.clone()
            assert f(got, got) is got
            torch.cuda.synchronize()
            assert torch.equal(got, want)
        want, got = sa.attn_paged_prefill(t, *args, cu, 0.1), t.clone()
        sa.attn_paged_prefill(got, *args, cu, 0.1, out=got)
        torch.cuda.synchronize()
        assert torch.equal(got, want)


def test_pools_past_32_bit_offsets():
    """Pages 2^31 elements apart: offsets of 2^32 elements and 2^33 bytes in every operator."""
    sa = _sa()
    page, d, hkv, far = 16, 64, 2, 1 << 31
    lens = [40, 20]
    for dtype in ("bf16", "f32"):
        small = Pool(lens, hkv, d, page, dtype, seed=33, extra_pages=0)
        n_pages = 3
        raw = torch.empty((n_pages - 1) * far + 2 * hkv * page * d, dtype=DT[dtype], device="cuda")
        k = raw.as_strided((n_pages, hkv, page, d), (far, page * d, d, 1))
        v = raw.as_strided((n_pages, hkv, page, d), (far, page * d, d, 1), hkv * page * d)
        # sequence 0 in pages 2, 0, 1
        table = torch.tensor([[2, 0, 1]], dtype=torch.int32).cuda()
        kv = torch.tensor([40], dtype=torch.int32).cuda()
        rows = torch.cat([small.k[0], small.v[0]]).transpose(0, 1).contiguous().cuda()      # [40, 2 hkv, d]
        cu = torch.tensor([0, 40], dtype=torch.int32).cuda()
        sa.paged_append(rows[:, :hkv], rows[:, hkv:], k, v, table, kv, cu_q=cu)
        assert torch.equal(k[2, :, :].cpu(), small.k[0][:, :16]) and torch.equal(v[1, :, :8].cpu(), small.v[0][:, 32:])
        q = small.q(40, 4)
        out = sa.attn_paged_prefill(q.cuda(), k, v, table, kv, cu, 0.125)
        _close(out, attend(q, small.k[0], small.v[0], range(40), 0.125), dtype, _v_max(small))
        out = sa.attn_paged_decode(q[:1].cuda(), k, v, table, kv, 0.125)
        _close(out, attend(q[:1], small.k[0], small.v[0], [39], 0.125), dtype, _v_max(small))
        out = sa.attn_paged_decode_prefix(q[:1].cuda(), k, v, table[0], 39, table, kv, 0.125)
        both = [torch.cat([x[:, :39], x], 1) for x in (small.k[0], small.v[0])]
        _close(out, attend(q[:1], *both, [78], 0.125), dtype, _v_max(small))
        del raw, k, v


def test_python_wrappers_check_gpu_tensors():
    sa = _sa()
    pool = Pool([5, 5], 2, 64, 16, "bf16", seed=1)
    args = (pool.kp, pool.vp, pool.table, pool.kv_lens)
    q = pool.q(2, 4).cuda()
    for bad, exc in ((q.float(), TypeError), (q[:1], ValueError), (q[:, :, :32], ValueError),
                     (q.transpose(1, 2).contiguous().transpose(1, 2), ValueError), (q.cpu(), ValueError), (q[:, :3], sa.SAError)):
        with pytest.raises(exc):
            sa.attn_paged_decode(bad, *args, 0.1)
    for over in (dict(block_table=pool.table.long()), dict(block_table=pool.table[:1]), dict(kv_lens=pool.kv_lens.float()),
                 dict(kv_lens=pool.kv_lens[:1]), dict(v_pages=pool.vp.float()), dict(k_pages=pool.kp.transpose(1, 2))):
        kw = dict(zip(("k_pages", "v_pages", "block_table", "kv_lens"), args)) | over
        with pytest.raises((ValueError, TypeError)):
            sa.attn_paged_decode(q, scale=0.1, **kw)
    with pytest.raises(ValueError):
        sa.attn_paged_prefill(q, *args, torch.tensor([0, 1], dtype=torch.int32).cuda(), 0.1)
    with pytest.raises(ValueError):
        sa.attn_paged_decode_prefix(q, pool.kp, pool.vp, pool.table[0], 10000, pool.table, pool.kv_lens, 0.1)
    with pytest.raises(ValueError):
        sa.paged_append(q[:1, :2], q[:1, 2:], *args)                       # two sequences, one token, no cu_q
    with pytest.raises(ValueError):
        sa.attn_paged_decode(q, *args, 0.1, out=q[:, :2])
    torch.cuda.synchronize()
