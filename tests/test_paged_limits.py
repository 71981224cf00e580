"""The limits that include/sa_cuda.h gives for the paged operators' numbers, on
both sides: what is refused on the CPU, and results just inside on the GPU."""
import pytest
import torch

from _paged import DT, Pool
from test_paged_args import P, _decode, _kv, _prefill, _prefix, _refused

# largest fp32 whose product with fp32 log2(e) = 0x1.715476p+0 is finite, and the next one
SCALE_MAX, SCALE_OVER = float.fromhex("0x1.62e42ep+127"), float.fromhex("0x1.62e430p+127")


@pytest.mark.parametrize("call", [_decode, _prefill, _prefix])
def test_scales_that_log2e_takes_past_fp32_are_refused(call):
    log2e = torch.tensor(1.4426950408889634)
    assert torch.isfinite(torch.tensor(SCALE_MAX) * log2e) and torch.isinf(torch.tensor(SCALE_OVER) * log2e)
    for scale in (SCALE_OVER, 3.0e38, float("inf")):
        _refused(call(_kv(), scale=scale), "scale")
    _refused(call(_kv(), scale=SCALE_MAX), "ctx is NULL")          # taken: the next check's error


def _all_forms(pool, q, scale):
    """The rows of ``pool``'s first sequence through every attention: decode, a prefill whose last token is the query,
    and a decode behind a prefix that is all of the sequence or its first 1024 rows.  q [1, hq, d] on the GPU."""
    import streaming_attention_b200 as sa
    n, pages = pool.lens[0], (pool.kp, pool.vp)
    none, empty = pool.table[:1], torch.zeros(1, dtype=torch.int32, device="cuda")
    cu = torch.tensor([0, 1], dtype=torch.int32, device="cuda")
    first = 1024 // pool.page
    rest = torch.tensor([n - 1024], dtype=torch.int32, device="cuda")
    yield "decode", sa.attn_paged_decode(q, *pages, pool.table[:1], pool.kv_lens[:1], scale)
    yield "prefill", sa.attn_paged_prefill(q, *pages, pool.table[:1], pool.kv_lens[:1], cu, scale)
    yield "prefix", sa.attn_paged_decode_prefix(q, *pages, pool.table[0], n, none, empty, scale)
    yield "prefix and own", sa.attn_paged_decode_prefix(q, *pages, pool.table[0], 1024, pool.table[:1, first:].contiguous(),
                                                        rest, scale)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype,power", [("f32", 127), ("bf16", 118)])
@pytest.mark.parametrize("hq", [2, 16])
@pytest.mark.parametrize("n", [4096, 4001])
def test_values_up_to_the_bound_over_the_rows(dtype, power, hq, n):
    """Evenly weighted rows of one value 2^power / 4096: q = 0, so every weight is 1, and sums of up to 4096 equal
    powers of two are exact; 1 / n and the product with it are off by 2^-24 each, less than half a step of bf16."""
    pool = Pool([n], 2, 128, 16, dtype, seed=1)
    value = 2.0 ** (power - 12)
    pool.vp.fill_(value)
    for name, out in _all_forms(pool, torch.zeros(1, hq, 128, dtype=DT[dtype], device="cuda"), 0.1):
        off = (out.double() / value - 1).abs().max().item()
        assert off <= (2.0 ** -22 if dtype == "f32" else 0.0), (name, off)


@pytest.mark.gpu
def test_bf16_weights_above_one_keep_the_bound():
    """Scores that rise by less than 2^8 after the first tile: the running maximum stays, weights are 2^7.5.  All values
    are equal, so the result is the value but for the weights' rounding to bf16 (2^-8) and the output's (2^-8)."""
    pool = Pool([4096], 2, 128, 16, "bf16", seed=2)
    value = 2.0 ** 106
    pool.vp.fill_(value)
    pool.kp.zero_()
    for j, p in enumerate(pool.table_list[0][:256]):
        if j >= 8:
            pool.kp[p, :, :, 0] = 5.1875                        # times log2(e): 7.48
    q = torch.zeros(1, 16, 128, dtype=torch.bfloat16, device="cuda")
    q[:, :, 0] = 1.0
    for name, out in _all_forms(pool, q, 1.0):
        assert ((out.double() / value - 1).abs() <= 2.0 ** -7).all(), name


@pytest.mark.gpu
@pytest.mark.parametrize("dtype,power", [("bf16", 24), ("f32", 24), ("f32", 120)])
@pytest.mark.parametrize("sign", [1.0, -1.0])
def test_scores_up_to_the_bound(dtype, power, sign):
    """Scores of +-2^power (1 - i / 128), i < 100, one product each: a row's two largest ones lie further apart than any
    weight reaches, so the rows with the largest score share the output evenly.  bf16: the two weights are rounded
    (2^-8 of w |v|), and so is the output."""
    pool = Pool([2000], 1, 128, 16, dtype, seed=3)
    half = power // 2
    g = torch.Generator().manual_seed(4)
    step = torch.randint(3, 100, (2000,), generator=g)
    step[[700, 1999]] = 0 if sign > 0 else 101                  # the two largest scores
    pool.kp.zero_()
    for r in range(2000):
        pool.kp[pool.table_list[0][r // 16], :, r % 16, 5] = 2.0 ** half * (1 - float(step[r]) / 128)
    q = torch.zeros(1, 8, 128, dtype=DT[dtype], device="cuda")
    q[:, :, 5] = sign * 2.0 ** (power - half)
    ref = (pool.v[0][0, 700].double() + pool.v[0][0, 1999].double()) / 2
    weighted = (pool.v[0][0, 700].double().abs() + pool.v[0][0, 1999].double().abs()) / 2
    bound = (ref.abs() + weighted) * (2.0 ** -8 if dtype == "bf16" else 0.0) + 2.0 ** -21 * weighted
    for name, out in _all_forms(pool, q, 1.0):
        assert ((out[0].double().cpu() - ref).abs() <= bound).all(), name
