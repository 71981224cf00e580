"""Long sequences in the paged decodes: marked values (tests/_paged_marks.py), so
that a lost, doubled or mis-weighted page of thousands shows."""
import math

import pytest
import torch

from _paged import Pool, attend, sees
from _paged_marks import bound, least_shift, mark

# lens, hq, hkv, d, page, window, sinks
DECODE = [([60000], 1, 1, 128, 16, 0, 0), ([3, 30000, 2], 16, 8, 64, 16, 0, 0), ([40000, 9000, 1, 0, 700], 8, 2, 128, 16, 0, 0),
          ([20011], 16, 1, 128, 128, 0, 0), ([9000, 5], 4, 2, 256, 32, 0, 0), ([50000, 1200], 8, 2, 128, 16, 20000, 600),
          ([30000], 3, 1, 64, 64, 9001, 130), ([333] * 90 + [7000] * 3, 4, 2, 128, 16, 0, 0)]
# own lens, prefix, hq, hkv, d, page: few and many rows, joined in the decode and by a kernel
PREFIX = [([0, 5, 200, 1, 64], 5000, 4, 2, 128, 16), ([700, 0, 33, 2000], 20000, 8, 2, 128, 32), ([90] * 40, 9000, 8, 2, 64, 16),
          ([3000], 30000, 16, 8, 128, 16), ([12] * 150, 1500, 4, 1, 128, 128), ([40, 0, 7], 1900, 6, 2, 128, 16)]
SPREAD = 0.25                                   # of the scores: no page carries hardly any weight


def _queries(pool, n, hq):
    return pool.q(n, hq, SPREAD)


def _seen(n, window, sinks):
    r = torch.arange(n)
    return r[(r >= (max(0, n - window) if window else 0)) | (r < sinks)]


def _decode_inputs(case, dtype, device):
    lens, hq, hkv, d, page, window, sinks = case
    pool = mark(Pool(lens, hkv, d, page, dtype, seed=lens[0] + d, device=device))
    return pool, _queries(pool, len(lens), hq)


def _prefix_inputs(case, dtype, device):
    lens, prefix, hq, hkv, d, page = case
    pool = mark(Pool([prefix] + lens, hkv, d, page, dtype, seed=prefix + d, device=device), prefix=True)
    return pool, _queries(pool, len(lens), hq)


@pytest.mark.parametrize("dtype", ["bf16", "f32"])
@pytest.mark.parametrize("case", range(len(DECODE)))
def test_every_page_of_a_decode_shows(case, dtype):
    pool, q = _decode_inputs(DECODE[case], dtype, "cpu")
    _, hq, hkv, d, page, window, sinks = DECODE[case]
    for b, n in enumerate(pool.lens[:5]):
        if n > 1:
            h = b % hq
            assert least_shift(dtype, q[b, h], pool.k[b][h * hkv // hq], pool.v[b][h * hkv // hq], d ** -0.5,
                               _seen(n, window, sinks), 16) > 1, (b, n)


@pytest.mark.parametrize("dtype", ["bf16", "f32"])
@pytest.mark.parametrize("case", range(len(PREFIX)))
def test_every_page_of_a_prefix_shows(case, dtype):
    pool, q = _prefix_inputs(PREFIX[case], dtype, "cpu")
    lens, prefix, hq, hkv, d, page = PREFIX[case]
    for b, n in enumerate(lens[:4]):
        k, v = (torch.cat([x[0][0], x[b + 1][0]]) for x in (pool.k, pool.v))
        assert least_shift(dtype, q[b, 0], k, v, d ** -0.5, torch.arange(prefix + n), 16) > 1, b


def _check(out, ref, dtype, rows):
    out = out.double().cpu()
    assert torch.isfinite(out).all()
    off = (out - ref).abs() - bound(dtype, ref, rows)
    assert off.max().item() <= 0, (off.max().item(), ((out - ref).abs() / ref.clamp(min=1e-9)).max().item())


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", ["bf16", "f32"])
@pytest.mark.parametrize("case", range(len(DECODE)))
def test_long_decodes(case, dtype):
    import streaming_attention_b200 as sa
    pool, q = _decode_inputs(DECODE[case], dtype, "cuda")
    _, hq, _, d, _, window, sinks = DECODE[case]
    if window:
        for b, n in enumerate(pool.lens):
            pool.forget(b, lambda r, n=n: sees(n - 1, r, window, sinks))
    out = sa.attn_paged_decode(q.cuda(), pool.kp, pool.vp, pool.table, pool.kv_lens, d ** -0.5, window=window, sinks=sinks)
    for b, n in enumerate(pool.lens):
        _check(out[b:b + 1], attend(q[b:b + 1], pool.k[b], pool.v[b], [n - 1], d ** -0.5, window, sinks), dtype, n)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", ["bf16", "f32"])
@pytest.mark.parametrize("case", range(len(PREFIX)))
def test_long_prefixes(case, dtype):
    import streaming_attention_b200 as sa
    pool, q = _prefix_inputs(PREFIX[case], dtype, "cuda")
    lens, prefix, _, _, d, _ = PREFIX[case]
    out = sa.attn_paged_decode_prefix(q.cuda(), pool.kp, pool.vp, pool.table[0], prefix, pool.table[1:], pool.kv_lens[1:],
                                      d ** -0.5)
    for b, n in enumerate(lens):
        ref = attend(q[b:b + 1], torch.cat([pool.k[0], pool.k[b + 1]], 1), torch.cat([pool.v[0], pool.v[b + 1]], 1),
                     [prefix + n - 1], d ** -0.5)
        _check(out[b:b + 1], ref, dtype, prefix + n)


def test_the_bound_rejects_zeros_and_holds_for_rounded_weights():
    """The bound against the arithmetic that it stands for, in float64 with weights and outputs rounded to bf16."""
    pool, q = _decode_inputs(DECODE[0], "bf16", "cpu")
    s = pool.k[0][0].double() @ q[0, 0].double() / math.sqrt(128)
    p = torch.exp(s - s.max())
    ref = p @ pool.v[0][0].double() / p.sum()
    got = (p.bfloat16().double() @ pool.v[0][0].double() / p.sum()).bfloat16().double()
    limit = bound("bf16", ref, 60000)
    assert ((got - ref).abs() <= limit).all() and (ref > limit).all()
