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

A context, the default one of a GPU included, serves one thread at a time;
threads that call at once pass one each as ``ctx``.

Workspaces come from torch's allocator: calls with different contexts, calls on
different streams and calls captured into different graphs do not share one.

A call costs the host 11 to 17 us, as much as or more than a small batch's step
takes the GPU, so the wrappers do little: one look at each tensor's layout, the
cache description packed in one go, workspace sizes kept by shape.  A captured
step leaves the host's part out.
"""
from __future__ import annotations

import ctypes as C
import struct

from ._capi import SA_BF16, SA_F32, SA_PAGED_ZERO_BYTES, Context, check, default_context, lib

_torch = None
_lib = None
_sizes: dict = {}
# the members of sa_paged_kv in order, natively aligned
_pack = struct.Struct("@PPiiiiiqPqiPi").pack


def _load():
    """torch and the library, at the first call (the package imports without torch)."""
    global _torch, _lib
    if _lib is None:
        import torch
        _torch, _lib = torch, lib()
    return _torch


def _code(x, what: str) -> int:
    if x.dtype is _torch.bfloat16:
        return SA_BF16
    if x.dtype is _torch.float32:
        return SA_F32
    raise TypeError(f"{what}: dtype {x.dtype} (want float32 or bfloat16)")


_INT_MAX = 0x7fffffff


def _ints(**numbers: int) -> None:
    """Refuses numbers that do not fit a C int (ctypes cuts them); negative ones that do are the library's to refuse."""
    for what, x in numbers.items():
        if not -0x80000000 <= x <= _INT_MAX:
            raise ValueError(f"{what}: {x} does not fit an int")


def _index(x, what: str, n: int, dev: int) -> int:
    """The address of a contiguous int32 vector of n entries."""
    if x.dtype is not _torch.int32 or x.get_device() != dev or x.dim() != 1 or x.shape[0] != n or not x.is_contiguous():
        raise ValueError(f"{what}: want a contiguous int32 vector of {n} on GPU {dev}, "
                         f"got {x.dtype} {tuple(x.shape)} strides {x.stride()} on {x.device}")
    return x.data_ptr()


def _rows(x, what: str, n: int, heads, d: int, dev: int, dtype) -> int:
    """The row stride of an [n, heads, d] tensor whose heads are contiguous."""
    shape, stride = x.shape, x.stride()
    if len(shape) != 3 or shape[2] != d or shape[0] != n or (heads is not None and shape[1] != heads):
        raise ValueError(f"{what}: shape {tuple(shape)}, want [{n}, {heads if heads is not None else 'hq'}, {d}]")
    if x.dtype is not dtype:
        raise TypeError(f"{what}: dtype {x.dtype}, want {dtype}")
    if x.get_device() != dev:
        raise ValueError(f"{what}: on {x.device}, the pages on GPU {dev}")
    if stride[2] != 1 or (stride[1] != d and shape[1] > 1):
        raise ValueError(f"{what}: the heads of a row must be contiguous (strides {stride})")
    return stride[0] if n > 1 else shape[1] * d


def _cache(k_pages, v_pages, block_table, kv_lens):
    """Checks a cache; returns (packed sa_paged_kv, GPU, dtype, code, hkv, d, page_size, n_seqs)."""
    if _lib is None:
        _load()
    shape, stride = k_pages.shape, k_pages.stride()
    dt, dev = k_pages.dtype, k_pages.get_device()
    if len(shape) != 4 or v_pages.shape != shape or v_pages.dtype is not dt or v_pages.get_device() != dev:
        raise ValueError(f"pages: k {tuple(shape)} {dt} on {k_pages.device}, "
                         f"v {tuple(v_pages.shape)} {v_pages.dtype} on {v_pages.device}")
    if not k_pages.is_cuda:
        raise ValueError(f"pages: on {k_pages.device}, want CUDA tensors")
    code = _code(k_pages, "pages")
    n_pages, hkv, page, d = shape
    for s in (stride, v_pages.stride()):
        if s[3] != 1 or s[2] != d or (hkv > 1 and s[1] != page * d) or (n_pages > 1 and s[0] != stride[0]):
            raise ValueError(f"pages: [hkv, page_size, d] of a page must be contiguous, k and v alike (strides {s})")
    if block_table.dim() != 2 or block_table.dtype is not _torch.int32 or block_table.get_device() != dev:
        raise ValueError(f"block_table: want int32 [n_seqs, max_pages] on GPU {dev}, "
                         f"got {block_table.dtype} {tuple(block_table.shape)} on {block_table.device}")
    n_seqs, max_pages = block_table.shape
    table_stride, inner = block_table.stride()
    if max_pages > 1 and inner != 1:
        raise ValueError("block_table: a sequence's entries must be contiguous")
    kv = _pack(k_pages.data_ptr(), v_pages.data_ptr(), code, n_pages, page, hkv, d,
               stride[0] if n_pages > 1 else hkv * page * d, block_table.data_ptr(),
               table_stride if n_seqs > 1 else max_pages, max_pages, _index(kv_lens, "kv_lens", n_seqs, dev), n_seqs)
    return kv, dev, dt, code, hkv, d, page, n_seqs


def _bind(ctx: Context | None, dev: int) -> Context:
    """The context, bound to torch's current stream of its GPU."""
    if ctx is None:
        ctx = default_context(dev)
    elif ctx.device != dev:
        raise ValueError(f"the context is on GPU {ctx.device}, the pages on GPU {dev}")
    check(_lib.sa_ctx_set_stream(ctx.h, _torch._C._cuda_getCurrentRawStream(dev)))
    return ctx


def _size(key, size_fn, *args) -> int:
    n = _sizes.get(key)
    if n is None:
        out = C.c_size_t()
        check(size_fn(*args, C.byref(out)))
        if len(_sizes) > 4096:
            _sizes.clear()
        n = _sizes[key] = out.value
    return n


def _capturing(dev: int) -> bool:
    """Whether torch's current stream of that GPU, which need not be the current one, is being captured."""
    if _torch._C._cuda_getDevice() == dev:
        return _torch._C._cuda_isCurrentStreamCapturing()
    with _torch.cuda.device(dev):
        return _torch._C._cuda_isCurrentStreamCapturing()


def _workspace(ctx: Context, dev: int, n: int):
    """A decode's workspace, its head zero; a captured call has its own.

    Kept from call to call of one context on one stream: those follow one another.
    Calls of threads that share a stream (torch's default one, unless they set
    another) do not: they have a context each, and a call may be several launches,
    which pass states through the workspace while another call's lie between them.
    """
    if _capturing(dev):
        ws = _torch.empty(n, dtype=_torch.uint8, device=dev)
        ws[:SA_PAGED_ZERO_BYTES].zero_()
        return ws
    stream = _torch._C._cuda_getCurrentRawStream(dev)
    ws = ctx.workspaces.get(stream)
    if ws is None or ws.numel() < n:
        ws = ctx.workspaces[stream] = _torch.zeros(n, dtype=_torch.uint8, device=dev)
    return ws


def rope_table(theta: float, rotary_dim: int, n_pos: int, device="cuda", ctx: Context | None = None):
    """(cos, sin), each [n_pos, rotary_dim // 2] fp32, of the angles p * theta^(-2i / rotary_dim) (sa_rope_table)."""
    torch = _load()
    _ints(n_pos=n_pos, rotary_dim=rotary_dim)
    device = torch.device(device)
    dev = device.index if device.index is not None else torch.cuda.current_device()
    cos = torch.empty(n_pos, rotary_dim // 2, dtype=torch.float32, device=torch.device("cuda", dev))
    sin = torch.empty_like(cos)
    check(_lib.sa_rope_table(_bind(ctx, dev).h, n_pos, rotary_dim, theta, cos.data_ptr(), sin.data_ptr()))
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
    if not 0 <= pos0 <= _INT_MAX:
        _ints(pos0=pos0)
    kv, dev, dt, _, hkv, d, _, n_seqs = _cache(k_pages, v_pages, block_table, kv_lens)
    n, xdt = k.shape[0], k.dtype
    ks, vs = _rows(k, "k", n, hkv, d, dev, xdt), _rows(v, "v", n, hkv, d, dev, xdt)
    qp = qop = cp = cosp = sinp = None
    qs = os = hq = n_pos = rot = 0
    if q is not None:
        qs = _rows(q, "q", n, None, d, dev, xdt)
        hq = q.shape[1]
        if q_out is None:
            q_out = q.new_empty((n, hq, d), dtype=dt)
            os = hq * d
        else:
            os = _rows(q_out, "q_out", n, hq, d, dev, dt)
        qp, qop = q.data_ptr(), q_out.data_ptr()
    if cu_q is not None:
        cp = _index(cu_q, "cu_q", n_seqs + 1, dev)
    elif n != n_seqs:
        raise ValueError(f"without cu_q every sequence has one token: {n} tokens, {n_seqs} sequences")
    if rope is not None:
        cos, sin = rope
        n_pos, half = cos.shape
        if n_pos > _INT_MAX:
            _ints(rope_positions=n_pos)
        rot = 2 * half
        for x in rope:
            if x.dtype is not _torch.float32 or x.shape != cos.shape or x.get_device() != dev or not x.is_contiguous():
                raise ValueError(f"rope: want contiguous float32 {tuple(cos.shape)} on GPU {dev}")
        cosp, sinp = cos.data_ptr(), sin.data_ptr()
    check(_lib.sa_paged_append(_bind(ctx, dev).h, kv, _code(k, "k"), qp, qs, k.data_ptr(), ks, v.data_ptr(), vs, n, hq, cp,
                               pos0, cosp, sinp, n_pos, rot, 1 if interleaved else 0, qop, os))
    return q_out


def attn_paged_decode(q, k_pages, v_pages, block_table, kv_lens, scale: float, window: int = 0, sinks: int = 0,
                      ctx: Context | None = None, out=None):
    """One query token per sequence over its pages (sa_attn_paged_decode).

    q [n_seqs, hq, d] in the pages' dtype, each at its sequence's last row.
    ``window`` > 0: a query sees the last ``window`` rows, its own included,
    and the first ``sinks`` rows.  Returns [n_seqs, hq, d] in q's dtype; a
    sequence of length 0 gets zeros.
    """
    if not (0 <= window <= _INT_MAX and 0 <= sinks <= _INT_MAX):
        _ints(window=window, sinks=sinks)
    kv, dev, dt, code, hkv, d, _, n_seqs = _cache(k_pages, v_pages, block_table, kv_lens)
    qs = _rows(q, "q", n_seqs, None, d, dev, dt)
    hq = q.shape[1]
    if out is None:
        out, os = _torch.empty_like(q, memory_format=_torch.contiguous_format), hq * d
    else:
        os = _rows(out, "out", n_seqs, hq, d, dev, dt)
    ctx = _bind(ctx, dev)
    n = _size((dev, code, hkv, hq, d), _lib.sa_attn_paged_decode_workspace, ctx.h, kv, hq)
    ws = _workspace(ctx, dev, n)
    check(_lib.sa_attn_paged_decode(ctx.h, kv, q.data_ptr(), qs, hq, window, sinks, scale, out.data_ptr(), os, ws.data_ptr(), n))
    return out


def attn_paged_prefill(q, k_pages, v_pages, block_table, kv_lens, cu_q, scale: float, window: int = 0, sinks: int = 0,
                       ctx: Context | None = None, out=None):
    """A ragged batch of prompt chunks over the sequences' pages (sa_attn_paged_prefill).

    q [n_tokens, hq, d] in the pages' dtype, d 64 or 128: tokens
    cu_q[b] .. cu_q[b + 1] - 1 are the last ones of sequence b, whose keys and
    values have been appended.  Causal, with ``window`` and ``sinks`` as in
    attn_paged_decode.  Returns [n_tokens, hq, d]; rows behind the last
    sequence are not written.
    """
    if not (0 <= window <= _INT_MAX and 0 <= sinks <= _INT_MAX):
        _ints(window=window, sinks=sinks)
    kv, dev, dt, _, _, d, _, n_seqs = _cache(k_pages, v_pages, block_table, kv_lens)
    n = q.shape[0]
    qs = _rows(q, "q", n, None, d, dev, dt)
    hq = q.shape[1]
    cp = _index(cu_q, "cu_q", n_seqs + 1, dev)
    if out is None:
        out, os = _torch.empty_like(q, memory_format=_torch.contiguous_format), hq * d
    else:
        os = _rows(out, "out", n, hq, d, dev, dt)
    check(_lib.sa_attn_paged_prefill(_bind(ctx, dev).h, kv, q.data_ptr(), qs, n, hq, cp, window, sinks, scale,
                                     out.data_ptr(), os))
    return out


def attn_paged_decode_prefix(q, k_pages, v_pages, prefix_table, prefix_len: int, block_table, kv_lens, scale: float,
                             ctx: Context | None = None, out=None):
    """One query token per sequence behind a prefix that all share (sa_attn_paged_decode_prefix).

    prefix_table [>= ceil(prefix_len / page_size)] int32 lists the prefix's
    pages; block_table and kv_lens are those of each sequence's own rows (a
    length may be 0).  q [n_seqs, hq, d] sees all of both.  d 64 or 128.
    Returns [n_seqs, hq, d].
    """
    if not 0 <= prefix_len <= _INT_MAX:
        _ints(prefix_len=prefix_len)
    kv, dev, dt, code, hkv, d, page, n_seqs = _cache(k_pages, v_pages, block_table, kv_lens)
    qs = _rows(q, "q", n_seqs, None, d, dev, dt)
    hq = q.shape[1]
    pp = _index(prefix_table, "prefix_table", prefix_table.shape[0], dev)
    if prefix_table.shape[0] * page < prefix_len:
        raise ValueError(f"prefix_table: {prefix_table.shape[0]} pages of {page} for {prefix_len} rows")
    if out is None:
        out, os = _torch.empty_like(q, memory_format=_torch.contiguous_format), hq * d
    else:
        os = _rows(out, "out", n_seqs, hq, d, dev, dt)
    ctx = _bind(ctx, dev)
    n = _size((dev, code, hkv, hq, d, n_seqs, prefix_len), _lib.sa_attn_paged_decode_prefix_workspace, ctx.h, kv, hq, prefix_len)
    ws = _workspace(ctx, dev, n)
    check(_lib.sa_attn_paged_decode_prefix(ctx.h, kv, pp, prefix_len, q.data_ptr(), qs, hq, scale, out.data_ptr(), os,
                                           ws.data_ptr(), n))
    return out
