"""Caches of pages and a plain 64-bit form of the operators over them, for the
paged-cache tests.  torch on any device; nothing here uses the library."""
import math

import torch

DT = {"f32": torch.float32, "bf16": torch.bfloat16}


class Pool:
    """Pages filled with NaN, and sequences' rows laid into randomly chosen ones.

    k[b], v[b] [hkv, len_b, d] are the rows as the cache's type holds them;
    table rows are -1 behind a sequence's last page.  `stride_pad` pages lie
    between neighbouring ones (any page stride is allowed)."""

    def __init__(self, lens, hkv, d, page, dtype, seed=0, extra_pages=2, pad_cols=1, interleaved_kv=False, device="cuda"):
        g = torch.Generator().manual_seed(seed)
        self.lens, self.hkv, self.d, self.page, self.dt = list(lens), hkv, d, page, DT[dtype]
        need = [-(-n // page) for n in lens]
        n_pages = sum(need) + extra_pages
        perm = torch.randperm(n_pages, generator=g).tolist()
        width = max(need + [0]) + pad_cols
        self.table_list, at = [], 0
        for n in need:
            self.table_list.append(perm[at:at + n] + [-1] * (width - n))
            at += n
        self.free = perm[at:]
        self.k = [torch.randn(hkv, n, d, generator=g).to(self.dt) for n in lens]
        self.v = [torch.randn(hkv, n, d, generator=g).to(self.dt) for n in lens]
        if interleaved_kv:
            both = torch.full((n_pages, 2, hkv, page, d), math.nan, dtype=self.dt)
            kp, vp = both[:, 0], both[:, 1]
        else:
            kp = torch.full((n_pages, hkv, page, d), math.nan, dtype=self.dt)
            vp = kp.clone()
        for b, n in enumerate(lens):
            for j in range(need[b]):
                r = slice(j * page, min(n, (j + 1) * page))
                m = r.stop - r.start
                kp[self.table_list[b][j], :, :m] = self.k[b][:, r]
                vp[self.table_list[b][j], :, :m] = self.v[b][:, r]
        if interleaved_kv:
            both = both.to(device)
            self.kp, self.vp = both[:, 0], both[:, 1]
        else:
            self.kp, self.vp = kp.to(device), vp.to(device)
        self.table = torch.tensor(self.table_list, dtype=torch.int32).reshape(len(lens), width).to(device)
        self.kv_lens = torch.tensor(lens, dtype=torch.int32).to(device)
        self.gen = g

    def q(self, n, hq, spread=1.0):
        return (spread * torch.randn(n, hq, self.d, generator=self.gen)).to(self.dt)

    def forget(self, b, keep):
        """Pages of sequence b without a row that keep(row) names: freed (-1 in the table, NaN in the pool)."""
        for j, p in enumerate(self.table_list[b]):
            if p >= 0 and not any(keep(r) for r in range(j * self.page, min(self.lens[b], (j + 1) * self.page))):
                self.kp[p], self.vp[p] = math.nan, math.nan
                self.table_list[b][j] = -1
                self.table[b, j] = -1


def sees(p, j, window, sinks):
    return j <= p and (window == 0 or j > p - window or j < sinks)


def attend(q, k, v, positions, scale, window=0, sinks=0):
    """q [n, hq, d] at `positions` over k, v [hkv, len, d], in float64."""
    n, hq, d = q.shape
    hkv, length, _ = k.shape
    g = hq // hkv
    out = torch.zeros(n, hq, d, dtype=torch.float64)
    if length == 0:
        return out
    p = torch.as_tensor(positions)[:, None]
    j = torch.arange(length)[None, :]
    vis = j <= p
    if window:
        vis &= (j > p - window) | (j < sinks)
    for h in range(hq):
        s = (q[:, h].double() @ k[h // g].double().T * scale).masked_fill(~vis, -math.inf)
        m = s.amax(1, keepdim=True)
        w = torch.exp(s - torch.where(m == -math.inf, torch.zeros_like(m), m))
        l = w.sum(1, keepdim=True)
        out[:, h] = (w @ v[h // g].double()) / torch.where(l == 0, torch.ones_like(l), l)
    return out


def tolerance(dtype, ref, v_max, p_rounded=True):
    """How far an output may be from the 64-bit one, entry by entry.

    bf16: the output's rounding is off by at most 2^-9 of |out| relative to a
    value (half a step, 2^-8 relative to the power of two below it: 2^-8 |out|);
    each softmax weight's rounding to bf16 by at most 2^-8 of the weight, so the
    weighted sum by 2^-8 max|v|.  fp32 arithmetic adds at most a few hundred
    half steps of 2^-24 to scores of a few tens: below 1e-4 of max|v|.
    fp32: scores up to ~64 in the exponent, their rounding 2^-24 * 64 * a few,
    sums of up to 2^14 terms kept in partial sums: below 4e-5 of max|v|."""
    if dtype == "bf16":
        return ref.abs() * 2.0 ** -8 + v_max * ((2.0 ** -8 if p_rounded else 0.0) + 1e-4)
    return torch.full_like(ref, 4e-5 * v_max)


def rotate(x, cos, sin, rot, interleaved):
    """x [n, heads, d] rotated by cos, sin [n, rot/2], in float64."""
    y = x.double().clone()
    half = rot // 2
    i = torch.arange(half) * (2 if interleaved else 1)
    j = i + (1 if interleaved else half)
    c, s = cos.double()[:, None, :], sin.double()[:, None, :]
    a, b = y[..., i].clone(), y[..., j].clone()
    y[..., i] = a * c - b * s
    y[..., j] = b * c + a * s
    return y
