"""Operators over a paged KV cache: batches of sequences whose keys and values
lie in pages (include/sa_cuda.h, "Attention over a paged KV cache").

All arrays are CUDA torch tensors; the calls run on torch's current stream of
the pages' device, asynchronously.

  k_pages, v_pages  [n_pages, hkv, page_size, d], fp32 or bf16 (any stride
                    between pages, the rest contiguous)
  block_table       [n_seqs, max_pages] int32: row r of sequence b lies in page
                    block_table[b, r // page_size]
  kv_lens           [n_seqs] int32: rows of each sequence, the tokens of the
                    call included
  cu_q              [n_seqs + 1] int32: sequence b's tokens are rows
                    cu_q[b] .. cu_q[b + 1] - 1 of the token tensors

Each call takes its workspace from torch's allocator, so calls on different
streams and calls captured into different graphs do not share one.
"""
from __future__ import annotations

import ctypes as C

from ._capi import SA_BF16, SA_F32, Context, PagedKV, check, default_context, lib


def _code(x, what: str) -> int:
    import torch
    if x.dtype == torch.bfloat16:
        return SA_BF16
    if x.dtype == torch.float32:
        return SA_F32
    raise TypeError(f"{what}: dtype {x.dtype} (want float32 or bfloat16)")


def _index(x, what: str, shape, device):
    import torch
    if x.dtype != torch.int32 or x.device != device or tuple(x.shape) != tuple(shape):
        raise ValueError(f"{what}: want int32 {tuple(shape)} on {device}, got {x.dtype} {tuple(x.shape)} on {x.device}")
    return x


def _rows(x, what: str, heads, d: int, device, dtype=None):
    """A [rows, heads, d] tensor whose heads are contiguous; returns its row stride."""
    if x.dim() != 3 or x.shape[2] != d or (heads is not None and x.shape[1] != heads):
        raise ValueError(f"{what}: shape {tuple(x.shape)}, want [rows, {heads if heads is not None else 'hq'}, {d}]")
    if x.device != device:
        raise ValueError(f"{what}: on {x.device}, the pages on {device}")
    if dtype is not None and x.dtype != dtype:
        raise TypeError(f"{what}: dtype {x.dtype}, the pages' is {dtype}")
    if x.numel() and (x.stride(2) != 1 or (x.shape[1] > 1 and x.stride(1) != d)):
        raise ValueError(f"{what}: the heads of a row must be contiguous (strides {x.stride()})")
    return x.stride(0) if x.shape[0] > 1 else x.shape[1] * d


def _cache(k_pages, v_pages, block_table, kv_lens) -> PagedKV:
    if k_pages.dim() != 4 or k_pages.shape != v_pages.shape or k_pages.dtype != v_pages.dtype \
            or k_pages.device != v_pages.device:
        raise ValueError(f"pages: k {tuple(k_pages.shape)} {k_pages.dtype} on {k_pages.device}, "
                         f"v {tuple(v_pages.shape)} {v_pages.dtype} on {v_pages.device}")
    dev = k_pages.device
    if dev.type != "cuda":
        raise ValueError(f"pages: on {dev}, want CUDA tensors")
    n_pages, hkv, page, d = k_pages.shape
    whole = hkv * page * d
    stride = k_pages.stride(0) if n_pages > 1 else whole
    for x in (k_pages, v_pages):
        if tuple(x.stride()[1:]) != (page * d, d, 1) and x.numel():
            raise ValueError(f"pages: [hkv, page_size, d] of a page must be contiguous (strides {x.stride()})")
        if n_pages > 1 and x.stride(0) != stride:
            raise ValueError("pages: k and v have different page strides")
    if block_table.dim() != 2:
        raise ValueError(f"block_table: shape {tuple(block_table.shape)}, want [n_seqs, max_pages]")
    n_seqs, max_pages = block_table.shape
    _index(block_table, "block_table", (n_seqs, max_pages), dev)
    _index(kv_lens, "kv_lens", (n_seqs,), dev)
    if max_pages > 1 and block_table.stride(1) != 1:
        raise ValueError("block_table: a sequence's entries must be contiguous")
    if not kv_lens.is_contiguous():
        raise ValueError("kv_lens: must be contiguous")
    return PagedKV(k_pages=k_pages.data_ptr(), v_pages=v_pages.data_ptr(), dtype=_code(k_pages, "pages"), n_pages=n_pages,
                   page_size=page, hkv=hkv, d=d, page_stride=stride, block_table=block_table.data_ptr(),
                   table_stride=block_table.stride(0) if n_seqs > 1 else max_pages, max_pages=max_pages,
                   kv_lens=kv_lens.data_ptr(), n_seqs=n_seqs)


def _bind(ctx: Context | None, device) -> Context:
    import torch
    if ctx is None:
        ctx = default_context(device.index or 0)
    elif ctx.device != (device.index or 0):
        raise ValueError(f"the context is on GPU {ctx.device}, the pages on {device}")
    ctx.set_stream(torch.cuda.current_stream(device).cuda_stream)
    return ctx


def _workspace(size_fn, device, *args):
    import torch
    n = C.c_size_t()
    check(size_fn(*args, C.byref(n)))
    return torch.empty(n.value, dtype=torch.uint8, device=device), n.value


def rope_table(theta: float, rotary_dim: int, n_pos: int, device="cuda", ctx: Context | None = None):
    """(cos, sin), each [n_pos, rotary_dim // 2] fp32, of the angles p * theta^(-2i / rotary_dim) (sa_rope_table)."""
    import torch
    device = torch.device(device)
    if device.index is None:
        device = torch.device("cuda", torch.cuda.current_device())
    cos = torch.empty(n_pos, rotary_dim // 2, dtype=torch.float32, device=device)
    sin = torch.empty_like(cos)
    ctx = _bind(ctx, device)
    check(lib().sa_rope_table(ctx.h, n_pos, rotary_dim, theta, cos.data_ptr(), sin.data_ptr()))
    return cos, sin


def paged_append(k, v, k_pages, v_pages, block_table, kv_lens, cu_q=None, q=None, rope=None, interleaved: bool = False,
                 pos0: int = 0, q_out=None, ctx: Context | None = None):
    """Write new tokens' k, v [n_tokens, hkv, d] into their sequences' pages (sa_paged_append).

    ``rope`` = (cos, sin), each [n_pos, rotary_dim // 2] fp32, rotates the keys
    (and q [n_tokens, hq, d], if given) by position ``pos0`` + row:
    ``interleaved`` pairs neighbouring elements, else element i turns with
    i + rotary_dim // 2.  Without ``cu_q`` every sequence gets one token.
    k, v and q share a dtype (fp32 or bf16), any row stride.  Returns the
    rotated queries in the pages' dtype (None without q).
    """
    import torch
    kv = _cache(k_pages, v_pages, block_table, kv_lens)
    dev, dt = k_pages.device, k_pages.dtype
    n = k.shape[0]
    ks = _rows(k, "k", kv.hkv, kv.d, dev)
    vs = _rows(v, "v", kv.hkv, kv.d, dev, k.dtype)
    if v.shape[0] != n:
        raise ValueError(f"k has {n} tokens, v {v.shape[0]}")
    qs = os = hq = 0
    if q is not None:
        qs = _rows(q, "q", None, kv.d, dev, k.dtype)
        hq = q.shape[1]
        if q.shape[0] != n:
            raise ValueError(f"k has {n} tokens, q {q.shape[0]}")
        if q_out is None:
            q_out = torch.empty(n, hq, kv.d, dtype=dt, device=dev)
        os = _rows(q_out, "q_out", hq, kv.d, dev, dt)
        if q_out.shape[0] != n:
            raise ValueError(f"q has {n} tokens, q_out {q_out.shape[0]}")
    if cu_q is None:
        if n != kv.n_seqs:
            raise ValueError(f"without cu_q every sequence has one token: {n} tokens, {kv.n_seqs} sequences")
    elif not _index(cu_q, "cu_q", (kv.n_seqs + 1,), dev).is_contiguous():
        raise ValueError("cu_q: must be contiguous")
    cos = sin = None
    n_pos = rot = 0
    if rope is not None:
        cos, sin = rope
        n_pos, rot = cos.shape[0], 2 * cos.shape[1]
        for x in (cos, sin):
            if x.dtype != torch.float32 or x.shape != cos.shape or x.device != dev or not x.is_contiguous():
                raise ValueError(f"rope: want contiguous float32 {tuple(cos.shape)} on {dev}")
    ctx = _bind(ctx, dev)
    check(lib().sa_paged_append(
        ctx.h, C.byref(kv), _code(k, "k"), q.data_ptr() if q is not None else None, qs, k.data_ptr(), ks, v.data_ptr(),
        vs, n, hq, cu_q.data_ptr() if cu_q is not None else None, pos0, cos.data_ptr() if rope is not None else None,
        sin.data_ptr() if rope is not None else None, n_pos, rot, 1 if interleaved else 0,
        q_out.data_ptr() if q is not None else None, os))
    return q_out


def _out(out, q, device):
    import torch
    if out is None:
        return torch.empty(q.shape, dtype=q.dtype, device=device)
    if out.shape != q.shape:
        raise ValueError(f"out: shape {tuple(out.shape)}, q {tuple(q.shape)}")
    return out


def attn_paged_decode(q, k_pages, v_pages, block_table, kv_lens, scale: float, window: int = 0, sinks: int = 0,
                      ctx: Context | None = None, out=None):
    """One query token per sequence over its pages (sa_attn_paged_decode).

    q [n_seqs, hq, d] in the pages' dtype, each at its sequence's last row.
    ``window`` > 0: a query sees the last ``window`` rows, its own included,
    and the first ``sinks`` rows.  Returns [n_seqs, hq, d] in q's dtype; a
    sequence of length 0 gets zeros.
    """
    kv = _cache(k_pages, v_pages, block_table, kv_lens)
    dev = k_pages.device
    qs = _rows(q, "q", None, kv.d, dev, k_pages.dtype)
    if q.shape[0] != kv.n_seqs:
        raise ValueError(f"q has {q.shape[0]} tokens, the block table {kv.n_seqs} sequences")
    out = _out(out, q, dev)
    os = _rows(out, "out", q.shape[1], kv.d, dev, q.dtype)
    ctx = _bind(ctx, dev)
    L = lib()
    ws, n = _workspace(L.sa_attn_paged_decode_workspace, dev, ctx.h, C.byref(kv), q.shape[1])
    check(L.sa_attn_paged_decode(ctx.h, C.byref(kv), q.data_ptr(), qs, q.shape[1], window, sinks, scale, out.data_ptr(),
                                 os, ws.data_ptr(), n))
    return out


def attn_paged_prefill(q, k_pages, v_pages, block_table, kv_lens, cu_q, scale: float, window: int = 0, sinks: int = 0,
                       ctx: Context | None = None, out=None):
    """A ragged batch of prompt chunks over the sequences' pages (sa_attn_paged_prefill).

    q [n_tokens, hq, d] in the pages' dtype, d 64 or 128: tokens
    cu_q[b] .. cu_q[b + 1] - 1 are the last ones of sequence b, whose keys and
    values have been appended.  Causal, with ``window`` and ``sinks`` as in
    attn_paged_decode.  Returns [n_tokens, hq, d]; rows behind the last
    sequence are left as they were.
    """
    kv = _cache(k_pages, v_pages, block_table, kv_lens)
    dev = k_pages.device
    qs = _rows(q, "q", None, kv.d, dev, k_pages.dtype)
    if not _index(cu_q, "cu_q", (kv.n_seqs + 1,), dev).is_contiguous():
        raise ValueError("cu_q: must be contiguous")
    out = _out(out, q, dev)
    os = _rows(out, "out", q.shape[1], kv.d, dev, q.dtype)
    ctx = _bind(ctx, dev)
    check(lib().sa_attn_paged_prefill(ctx.h, C.byref(kv), q.data_ptr(), qs, q.shape[0], q.shape[1], cu_q.data_ptr(),
                                      window, sinks, scale, out.data_ptr(), os))
    return out


def attn_paged_decode_prefix(q, k_pages, v_pages, prefix_table, prefix_len: int, block_table, kv_lens, scale: float,
                             ctx: Context | None = None, out=None):
    """One query token per sequence behind a prefix that all share (sa_attn_paged_decode_prefix).

    prefix_table [>= ceil(prefix_len / page_size)] int32 lists the prefix's
    pages; block_table and kv_lens are those of each sequence's own rows (a
    length may be 0).  q [n_seqs, hq, d] sees all of both.  d 64 or 128.
    Returns [n_seqs, hq, d].
    """
    kv = _cache(k_pages, v_pages, block_table, kv_lens)
    dev = k_pages.device
    qs = _rows(q, "q", None, kv.d, dev, k_pages.dtype)
    if q.shape[0] != kv.n_seqs:
        raise ValueError(f"q has {q.shape[0]} tokens, the block table {kv.n_seqs} sequences")
    if prefix_table.dim() != 1 or prefix_table.shape[0] * kv.page_size < prefix_len:
        raise ValueError(f"prefix_table: shape {tuple(prefix_table.shape)} for {prefix_len} rows")
    if not _index(prefix_table, "prefix_table", prefix_table.shape, dev).is_contiguous():
        raise ValueError("prefix_table: must be contiguous")
    out = _out(out, q, dev)
    os = _rows(out, "out", q.shape[1], kv.d, dev, q.dtype)
    ctx = _bind(ctx, dev)
    L = lib()
    ws, n = _workspace(L.sa_attn_paged_decode_prefix_workspace, dev, ctx.h, C.byref(kv), q.shape[1], prefix_len)
    check(L.sa_attn_paged_decode_prefix(ctx.h, C.byref(kv), prefix_table.data_ptr(), prefix_len, q.data_ptr(), qs,
                                        q.shape[1], scale, out.data_ptr(), os, ws.data_ptr(), n))
    return out
