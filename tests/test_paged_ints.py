"""Numbers that do not fit the C int they become: refused by the Python wrappers,
not cut (2^32 + 5 rows of window would be five)."""
import pytest
import torch

import streaming_attention_b200 as sa

KP = torch.zeros(4, 2, 16, 64)
TABLE = torch.zeros(1, 2, dtype=torch.int32)
LENS = torch.ones(1, dtype=torch.int32)
Q = torch.zeros(1, 2, 64)
BIG = [2 ** 32 + 5, 2 ** 31, 2 ** 63, -2 ** 32 + 1]


@pytest.mark.parametrize("x", BIG)
def test_numbers_past_an_int_are_refused(x):
    for name in ("window", "sinks"):
        with pytest.raises(ValueError, match=f"{name}: .*fit"):
            sa.attn_paged_decode(Q, KP, KP, TABLE, LENS, 1.0, **{name: x})
        with pytest.raises(ValueError, match=f"{name}: .*fit"):
            sa.attn_paged_prefill(Q, KP, KP, TABLE, LENS, torch.zeros(2, dtype=torch.int32), 1.0, **{name: x})
    with pytest.raises(ValueError, match="prefix_len: .*fit"):
        sa.attn_paged_decode_prefix(Q, KP, KP, TABLE[0], x, TABLE, LENS, 1.0)
    with pytest.raises(ValueError, match="pos0: .*fit"):
        sa.paged_append(Q, Q, KP, KP, TABLE, LENS, pos0=x)
    with pytest.raises(ValueError, match="n_pos: .*fit"):
        sa.rope_table(1e4, 64, x)
    with pytest.raises(ValueError, match="rotary_dim: .*fit"):
        sa.rope_table(1e4, x, 4)


def test_the_largest_ints_are_taken_to_the_next_check():
    with pytest.raises(ValueError, match="CUDA"):
        sa.attn_paged_decode(Q, KP, KP, TABLE, LENS, 1.0, window=2 ** 31 - 1, sinks=2 ** 31 - 1)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", ["bf16", "f32"])
def test_the_largest_window_and_first_tokens_are_no_window(dtype):
    from _paged import Pool
    pool = Pool([300, 17], 2, 64, 16, dtype, seed=1)
    args, cu = (pool.kp, pool.vp, pool.table, pool.kv_lens), torch.tensor([0, 40, 57], dtype=torch.int32, device="cuda")
    q = pool.q(57, 4).cuda()
    top = 2 ** 31 - 1
    for kw in (dict(window=top), dict(window=top, sinks=top), dict(window=1, sinks=top)):
        assert torch.equal(sa.attn_paged_decode(q[:2], *args, 0.1, **kw), sa.attn_paged_decode(q[:2], *args, 0.1))
        assert torch.equal(sa.attn_paged_prefill(q, *args, cu, 0.1, **kw), sa.attn_paged_prefill(q, *args, cu, 0.1))
