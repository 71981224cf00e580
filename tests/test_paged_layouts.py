"""Layouts of a cache that are contiguous by what they hold, whatever the strides
of dimensions of size one say."""
import pytest
import torch

from _paged import Pool, attend, tolerance


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", ["bf16", "f32"])
def test_one_head_pages_laid_out_by_token(dtype):
    """[n_pages, page_size, 1, d] transposed: with one KV head the same bytes as [n_pages, 1, page_size, d]."""
    import streaming_attention_b200 as sa
    pool = Pool([70, 5], 1, 64, 16, dtype, seed=3)
    kp, vp = (x.reshape(-1, 16, 1, 64).transpose(1, 2) for x in (pool.kp, pool.vp))
    assert kp.stride() != pool.kp.stride() and kp.shape == pool.kp.shape
    q = pool.q(2, 4)
    out = sa.attn_paged_decode(q.cuda(), kp, vp, pool.table, pool.kv_lens, 0.125)
    for b, n in enumerate(pool.lens):
        ref = attend(q[b:b + 1], pool.k[b], pool.v[b], [n - 1], 0.125)
        assert ((out[b:b + 1].double().cpu() - ref).abs() <= tolerance(dtype, ref, pool.v[b].abs().max().item())).all()
    both = sa.attn_paged_decode(q.cuda(), kp, pool.vp, pool.table, pool.kv_lens, 0.125)
    assert torch.equal(both, out)


@pytest.mark.gpu
def test_two_heads_laid_out_by_token_are_refused():
    import streaming_attention_b200 as sa
    pool = Pool([70, 5], 2, 64, 16, "bf16", seed=3)
    kp = pool.kp.reshape(-1, 16, 2, 64).transpose(1, 2)
    with pytest.raises(ValueError, match="contiguous"):
        sa.attn_paged_decode(pool.q(2, 4).cuda(), kp, kp, pool.table, pool.kv_lens, 0.125)
