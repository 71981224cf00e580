"""What the operators over a paged KV cache refuse, on the CPU: the C entry
points check their arguments before they look at the context, and the Python
wrappers check shapes, types and places."""
import ctypes as C

import pytest
import torch

from streaming_attention_b200 import lib
from streaming_attention_b200._capi import SA_BF16, SA_F32, SA_PAGED_MAX_SEQS, PagedKV

P = 0x10000          # an address that no check reads through


def _kv(**over):
    f = dict(k_pages=P, v_pages=P, dtype=SA_BF16, n_pages=10, page_size=16, hkv=2, d=128, page_stride=2 * 16 * 128,
             block_table=P, table_stride=4, max_pages=4, kv_lens=P, n_seqs=3)
    f.update(over)
    return PagedKV(**f)


def _decode(kv, q=P, qs=4 * 128, hq=4, window=0, sinks=0, scale=1.0, out=P, os=4 * 128, ws=P, n=1 << 30):
    return lib().sa_attn_paged_decode(None, C.byref(kv) if kv is not None else None, q, qs, hq, window, sinks, scale,
                                      out, os, ws, n)


def _append(kv, xd=SA_BF16, q=P, qs=4 * 128, k=P, ks=256, v=P, vs=256, n=5, hq=4, cu=P, pos0=0, cos=P, sin=P, n_pos=100,
            rot=128, inter=0, qo=P, qos=512):
    return lib().sa_paged_append(None, C.byref(kv) if kv is not None else None, xd, q, qs, k, ks, v, vs, n, hq, cu, pos0,
                                 cos, sin, n_pos, rot, inter, qo, qos)


def _prefill(kv, q=P, qs=512, n=5, hq=4, cu=P, window=0, sinks=0, scale=1.0, out=P, os=512):
    return lib().sa_attn_paged_prefill(None, C.byref(kv) if kv is not None else None, q, qs, n, hq, cu, window, sinks,
                                       scale, out, os)


def _prefix(kv, table=P, n=100, q=P, qs=512, hq=4, scale=1.0, out=P, os=512, ws=P, nb=1 << 30):
    return lib().sa_attn_paged_decode_prefix(None, C.byref(kv) if kv is not None else None, table, n, q, qs, hq, scale,
                                             out, os, ws, nb)


def _refused(rc, text):
    msg = lib().sa_last_error().decode()
    assert rc == -1 and text in msg, (rc, msg)


BAD_CACHE = [(dict(dtype=7), "dtype 7"), (dict(k_pages=None), "null k_pages"), (dict(v_pages=None), "null k_pages"),
             (dict(d=96), "d = 96"), (dict(page_size=8), "page_size = 8"), (dict(page_size=48), "page_size = 48"),
             (dict(hkv=0), "hkv = 0"), (dict(n_pages=0), "n_pages = 0"), (dict(n_seqs=-1), "n_seqs = -1"),
             (dict(n_seqs=SA_PAGED_MAX_SEQS + 1), "n_seqs ="), (dict(max_pages=5), "max_pages 5"),
             (dict(max_pages=-1), "max_pages -1"), (dict(block_table=None), "null block_table"),
             (dict(kv_lens=None), "null block_table"), (dict(page_stride=2 * 16 * 128 - 8), "page_stride"),
             (dict(page_stride=2 * 16 * 128 + 4), "page_stride"), (dict(k_pages=P + 8), "16-byte"),
             (dict(max_pages=1 << 28, table_stride=1 << 28), "2^31")]


@pytest.mark.parametrize("over,text", BAD_CACHE)
def test_bad_caches(over, text):
    _refused(_decode(_kv(**over)), text)
    _refused(_append(_kv(**over)), text)
    _refused(_prefill(_kv(**over)), text)
    _refused(_prefix(_kv(**over)), text)


@pytest.mark.parametrize("over,text", [
    (dict(hq=3), "hq = 3"), (dict(hq=40, qs=5120, os=5120), "hq = 40"), (dict(window=-5), "window -5"),
    (dict(sinks=-5), "sinks -5"), (dict(scale=-0.5), "scale"), (dict(n=-1), "n_tokens -1"), (dict(cu=None), "cu_q is NULL"),
    (dict(q=P + 2), "q is NULL or not"), (dict(qs=504), "q token stride"), (dict(out=None), "out is NULL"),
    (dict(os=511), "out token stride")])
def test_bad_prefill_arguments(over, text):
    _refused(_prefill(_kv(), **over), text)


@pytest.mark.parametrize("over,text", [
    (dict(hq=3), "hq = 3"), (dict(n=-1), "prefix_len -1"), (dict(n=2 ** 31 - 1), "prefix_len"),
    (dict(table=None), "prefix_table is NULL"), (dict(scale=0.0), "scale"), (dict(q=None), "q is NULL"),
    (dict(out=P + 8), "out is NULL or not"), (dict(os=300), "out token stride")])
def test_bad_prefix_arguments(over, text):
    _refused(_prefix(_kv(), **over), text)


def test_tiled_attention_takes_heads_of_64_and_128():
    wide = _kv(d=256, page_stride=2 * 16 * 256)
    _refused(_prefill(wide, qs=1024, os=1024), "d = 256")
    _refused(_prefix(wide, qs=1024, os=1024), "d = 256")


def test_null_description_and_context():
    _refused(_decode(None), "kv is NULL")
    _refused(_append(None), "kv is NULL")
    _refused(_prefill(None), "kv is NULL")
    _refused(_prefix(None), "kv is NULL")
    _refused(_decode(_kv()), "ctx is NULL")
    _refused(_prefill(_kv()), "ctx is NULL")
    _refused(_prefix(_kv()), "ctx is NULL")
    _refused(_prefix(_kv(), table=None, n=0), "ctx is NULL")
    _refused(_append(_kv()), "ctx is NULL")


@pytest.mark.parametrize("over,text", [
    (dict(hq=3), "hq = 3"), (dict(hq=0), "hq = 0"), (dict(hq=34, qs=34 * 128, os=34 * 128), "hq = 34"),
    (dict(window=-1), "window -1"), (dict(sinks=-1), "sinks -1"), (dict(scale=0.0), "scale"),
    (dict(scale=-1.0), "scale"), (dict(scale=float("nan")), "scale"), (dict(scale=float("inf")), "scale"),
    (dict(q=None), "q is NULL"), (dict(q=P + 4), "q is NULL or not"), (dict(qs=511), "q token stride"),
    (dict(qs=516), "q token stride"), (dict(out=None), "out is NULL"), (dict(os=504), "out token stride")])
def test_bad_decode_arguments(over, text):
    _refused(_decode(_kv(), **over), text)


def test_wide_heads_take_fewer_queries_per_key():
    kv = _kv(d=256, page_stride=2 * 16 * 256)
    _refused(_decode(kv, hq=18, qs=18 * 256, os=18 * 256), "d = 256")
    _refused(_decode(kv, hq=16, qs=16 * 256, os=16 * 256), "ctx is NULL")


@pytest.mark.parametrize("over,text", [
    (dict(xd=3), "x_dtype 3"), (dict(n=-1), "n_tokens -1"), (dict(pos0=-1), "pos0 -1"),
    (dict(cos=None), "one of cos and sin"), (dict(sin=None), "one of cos and sin"), (dict(qo=None), "q without q_out"),
    (dict(rot=8), "rotary_dim = 8"), (dict(rot=24), "rotary_dim = 24"), (dict(rot=144), "rotary_dim = 144"),
    (dict(n_pos=0), "n_pos = 0"), (dict(cos=P + 4), "cos/sin not"), (dict(k=None), "k is NULL"),
    (dict(v=None), "v is NULL"), (dict(ks=248), "k token stride"), (dict(vs=260), "v token stride"),
    (dict(hq=0), "hq = 0"), (dict(qos=500), "q_out token stride")])
def test_bad_append_arguments(over, text):
    _refused(_append(_kv(), **over), text)


def test_nothing_to_do_is_no_error():
    assert _append(_kv(), n=0, k=None, v=None) == 0
    assert _append(_kv(n_seqs=0, block_table=None, kv_lens=None, max_pages=0)) == 0
    assert _prefill(_kv(), n=0, q=None, out=None, cu=None) == 0
    assert _prefix(_kv(n_seqs=0, block_table=None, kv_lens=None, max_pages=0), q=None, out=None) == 0
    assert _decode(_kv(n_seqs=0, block_table=None, kv_lens=None, max_pages=0), q=None, out=None) == 0


@pytest.mark.parametrize("n_pos,rot,theta,cos,text", [
    (0, 128, 1e4, P, "n_pos 0"), (5, 3, 1e4, P, "rotary_dim 3"), (5, 128, 1.0, P, "theta"), (5, 128, 1e4, None, "null table"),
    (5, 128, float("nan"), P, "theta"), (5, 128, 1e4, P, "ctx is NULL")])
def test_bad_rope_tables(n_pos, rot, theta, cos, text):
    _refused(lib().sa_rope_table(None, n_pos, rot, theta, cos, P), text)


def test_python_wrappers_refuse_host_tensors_and_wrong_shapes():
    import streaming_attention_b200 as sa
    kp = torch.zeros(4, 2, 16, 64)
    table = torch.zeros(1, 2, dtype=torch.int32)
    lens = torch.ones(1, dtype=torch.int32)
    with pytest.raises(ValueError, match="CUDA"):
        sa.attn_paged_decode(torch.zeros(1, 2, 64), kp, kp, table, lens, 1.0)
    with pytest.raises(ValueError, match="pages"):
        sa.attn_paged_decode(torch.zeros(1, 2, 64), kp, kp[:2], table, lens, 1.0)
    meta = torch.zeros(4, 2, 16, 64, device="meta")
    with pytest.raises(ValueError, match="CUDA"):
        sa.paged_append(torch.zeros(1, 2, 64), torch.zeros(1, 2, 64), meta, meta, table, lens)


def test_packed_description_is_the_struct():
    from streaming_attention_b200.paged import _pack
    kv = _kv(k_pages=1 << 40, v_pages=3 << 40, page_stride=1 << 35, table_stride=7, n_seqs=9)
    vals = [getattr(kv, f) for f, _ in PagedKV._fields_]
    assert bytes(kv)[:len(_pack(*vals))] == _pack(*vals) and C.sizeof(kv) - len(_pack(*vals)) < 8
