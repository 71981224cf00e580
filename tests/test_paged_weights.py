"""The bf16 decode's softmax weights keep more bits than bf16 has: the output's
rounding is the only one that shows, also where one row decides a column."""
import pytest
import torch

from _paged import Pool, attend
from _paged_marks import EDGES, mark

# lens, hq, hkv, d, page, window
CASES = [([700, 64, 1, 0, 129], 8, 2, 128, 16, 0), ([5000, 333], 16, 1, 64, 32, 0), ([900, 2000], 12, 3, 256, 16, 0),
         ([1500, 1400], 6, 6, 128, 64, 800)]


def _inputs(case, device):
    lens, hq, hkv, d, page, _ = case
    pool = mark(Pool(lens, hkv, d, page, "bf16", seed=lens[0], device=device))
    return pool, pool.q(len(lens), hq, 0.5)


def _bound(ref, rows):
    """The output's rounding, 2^-8 of it; each weight off by 2^-16 of itself (values are not negative, so the weighted
    sum of their magnitudes is the output); fp32 sums and scores as in _paged_marks.bound."""
    return ref.abs() * (2.0 ** -8 + 2.0 ** -16 + (rows + 300) * 2.0 ** -24)


def _weighted(p, v):
    """sum p v / sum p of weights as one bf16 number and as two, rounded to bf16 at the end; and unrounded."""
    one = p.bfloat16().double()
    two = one + (p - one).bfloat16().double()
    return [((x @ v) / p.sum()).bfloat16().double() for x in (one, two)] + [(p @ v) / p.sum()]


def test_one_bf16_weight_exceeds_the_bound_and_two_keep_it():
    over = 0
    for case in CASES[:2]:
        pool, q = _inputs(case, "cpu")
        hq, hkv, d = case[1:4]
        for b, n in enumerate(pool.lens):
            for h in range(hq if n > 1 else 0):
                s = pool.k[b][h * hkv // hq].double() @ q[b, h].double() * d ** -0.5
                one, two, ref = _weighted(torch.exp(s - s.max()), pool.v[b][h * hkv // hq].double())
                assert ((two - ref).abs() <= _bound(ref, n)).all()
                over += int(((one - ref).abs() > _bound(ref, n))[-len(EDGES):].any())
    assert over > 10


@pytest.mark.gpu
@pytest.mark.parametrize("case", range(len(CASES)))
def test_decode_keeps_the_weights(case):
    import streaming_attention_b200 as sa
    pool, q = _inputs(CASES[case], "cuda")
    d, window = CASES[case][3], CASES[case][5]
    out = sa.attn_paged_decode(q.cuda(), pool.kp, pool.vp, pool.table, pool.kv_lens, d ** -0.5, window=window).double().cpu()
    for b, n in enumerate(pool.lens):
        ref = attend(q[b:b + 1], pool.k[b], pool.v[b], [n - 1], d ** -0.5, window)
        assert ((out[b:b + 1] - ref).abs() <= _bound(ref, n)).all(), b
