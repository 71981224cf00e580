"""The operators over a paged KV cache, as cases that can be timed and compared.

A cache is a pool of pages [n_pages, hkv, page_size, d] for keys and one for
values, a block table that lists each sequence's pages, and the sequences'
lengths.  ``run`` makes one pass through one operator: in its plain form
(elementary torch operations in 32 bits, rounded once at the end), or, where
``own`` is true, by the calls a user makes of this package.

Operators (``case["op"]``):
  append   rotate the new tokens' keys (and queries) by their positions and
           write keys and values into the sequences' pages
  decode   one query token per sequence over its pages, with a sliding window
           and first tokens that stay visible
  prefill  a ragged batch of prompt chunks over the pages, causal, with the
           same window and first tokens
  prefix   one query token per sequence over a prefix that all sequences
           share and each sequence's own pages
"""
import math
import random

import torch

own = False

_DT = {"f32": torch.float32, "bf16": torch.bfloat16}


# ---------------------------------------------------------------- the cases

def listed():
    return [
        # one decode step of eight running sequences: the call that latency decides
        _case("append", "append step", "bf16", 16, 8, 128, 16, seqs=8, new=1, past=900, rot=128),
        # the prompts of a batch, sixteen ragged ones of up to 1024 tokens, written in one call
        _case("append", "append prompts", "bf16", 16, 8, 128, 16, seqs=16, new=1024, past=2000, rot=128),
        # a float32 cache with narrow heads, half of each head rotated, adjacent pairs
        _case("append", "append f32 pairs", "f32", 12, 4, 64, 32, seqs=5, new=333, past=77, rot=32, pairs=True),
        # one short conversation: latency again
        _case("decode", "decode one short", "bf16", 16, 8, 128, 16, seqs=1, kv=700, window=256, sinks=4),
        # a full serving batch of long conversations under a window
        _case("decode", "decode batch window", "bf16", 32, 8, 128, 16, seqs=64, kv=16384, window=4096, sinks=4),
        # a float32 cache without a window, ragged, an odd number of sequences
        _case("decode", "decode f32 ragged", "f32", 16, 8, 128, 32, seqs=13, kv=8191, window=0, sinks=0),
        # a chunk of one prompt on top of what is cached, narrow window
        _case("prefill", "prefill chunk", "bf16", 16, 8, 128, 16, seqs=1, new=512, past=3584, window=1000, sinks=4),
        # a whole long prompt, window of half its length
        _case("prefill", "prefill long", "bf16", 16, 8, 128, 16, seqs=1, new=8192, past=0, window=4096, sinks=4),
        # ragged float32 chunks, narrow heads
        _case("prefill", "prefill f32 ragged", "f32", 8, 4, 64, 32, seqs=3, new=300, past=257, window=129, sinks=1),
        # four beams of one request
        _case("prefix", "prefix beams", "bf16", 16, 8, 128, 16, seqs=4, prefix=1000, kv=60),
        # a batch behind one long system prompt
        _case("prefix", "prefix batch", "bf16", 32, 8, 128, 16, seqs=64, prefix=32768, kv=512),
        # the same from a float32 cache
        _case("prefix", "prefix f32", "f32", 16, 8, 128, 32, seqs=16, prefix=4001, kv=130),
    ]


def _case(op, name, dtype, hq, hkv, d, page, *, seqs, lens=1, new=0, past=0, kv=0, prefix=0, window=0, sinks=0,
          rot=0, pairs=False):
    c = {"op": op, "name": name, "dtype": dtype, "hq": hq, "hkv": hkv, "d": d, "page": page, "seqs": seqs,
         "lens": lens, "new": new, "past": past, "kv": kv, "prefix": prefix, "window": window, "sinks": sinks,
         "rot": rot, "pairs": pairs}
    if name is None:
        del c["name"]
    return c


def _spread(rng, lo, hi):
    """A whole number in [lo, hi], even over its logarithm."""
    return min(hi, max(lo, round(math.exp(rng.uniform(math.log(lo), math.log(hi + 0.49))))))


def draw(rng):
    op = rng.choice(["append", "decode", "decode", "prefill", "prefill", "prefix", "prefix"])
    dtype = rng.choice(["bf16", "bf16", "f32"])
    hkv = rng.choice([1, 2, 4, 8, 8])
    hq = hkv * rng.choice([1, 2, 2, 3, 4, 4, 6, 7, 8])
    d = rng.choice([64, 128, 128])
    page = rng.choice([16, 16, 32, 64, 128])
    lens = rng.randrange(1 << 20)
    window, sinks = 0, 0
    if op in ("decode", "prefill") and rng.random() < 0.75:
        window, sinks = _spread(rng, 1, 4096), rng.choice([0, 1, 4, 4, 17, 130])
    if op == "append":
        d = rng.choice([64, 128, 128, 256])
        seqs = _spread(rng, 1, 64)
        return _case(op, None, dtype, hq, hkv, d, page, seqs=seqs, lens=lens, past=_spread(rng, 1, 4096) - 1,
                     new=_spread(rng, 1, max(1, 8192 // seqs)), rot=rng.choice([d, d, d // 2]),
                     pairs=rng.random() < 0.3)
    if op == "decode":
        d = rng.choice([64, 128, 128, 256])
        seqs = _spread(rng, 1, 64)
        kv = _spread(rng, 1, min(16384, (1 << 29) // (seqs * hkv * d * (4 if dtype == "f32" else 2))))
        return _case(op, None, dtype, hq, hkv, d, page, seqs=seqs, lens=lens, kv=kv, window=window, sinks=sinks)
    if op == "prefill":
        seqs = rng.choice([1, 1, 2, 3, 5, 8])
        new = _spread(rng, 1, 4096 // seqs)
        past = min(_spread(rng, 1, 4096) - 1, (1 << 30) // (seqs * hq * new) - new)
        return _case(op, None, dtype, hq, hkv, d, page, seqs=seqs, lens=lens, new=new, past=past, window=window,
                     sinks=sinks)
    seqs = _spread(rng, 1, 128)
    return _case(op, None, dtype, hq, hkv, d, page, seqs=seqs, lens=lens, prefix=_spread(rng, 16, 32768),
                 kv=_spread(rng, 1, 512))


def _lengths(case):
    """Per sequence: rows cached before the call, new tokens, and rows after it.  The first sequence has the
    largest of each; the others are ragged.  They go by the case alone."""
    r = random.Random(case["lens"])
    rows = []
    for b in range(case["seqs"]):
        if case["op"] in ("append", "prefill"):
            past = case["past"] if b == 0 else r.randint(0, case["past"])
            new = case["new"] if b == 0 else r.randint(1, case["new"])
            rows.append((past, new, past + new))
        else:
            kv = case["kv"] if b == 0 else r.randint(case["kv"] // 2, case["kv"])
            if case["op"] == "prefix" and b % 7 == 5:
                kv = 0                                  # a sequence with nothing of its own yet
            rows.append((kv, 1, kv))
    return rows


def _visible(case, pos):
    """How many rows a query at `pos` sees."""
    if not case["window"]:
        return pos + 1
    lo = max(0, pos - case["window"] + 1)
    return pos + 1 - lo + min(case["sinks"], lo)


def work(case):
    e = 4 if case["dtype"] == "f32" else 2
    hq, hkv, d = case["hq"], case["hkv"], case["d"]
    rows = _lengths(case)
    if case["op"] == "append":
        n = sum(new for _, new, _ in rows)
        pos = len({p + t for p, new, _ in rows for t in range(new)})
        return {"bytes": 2 * n * (hq + 2 * hkv) * d * e + pos * case["rot"] * 4, "flops": 3 * n * (hq + hkv) * case["rot"]}
    if case["op"] == "prefill":
        n = sum(new for _, new, _ in rows)
        seen, flops = 0, 0
        for past, new, kv in rows:
            lo = max(0, past - case["window"] + 1) if case["window"] else 0
            seen += kv - lo + min(case["sinks"], lo)
            flops += 4 * hq * d * sum(_visible(case, past + t) for t in range(new))
        return {"bytes": (2 * n * hq + 2 * seen * hkv) * d * e, "flops": flops}
    seen = sum(_visible(case, kv - 1) if kv else 0 for _, _, kv in rows)
    b = case["seqs"]
    return {"bytes": (2 * (seen + case["prefix"]) * hkv + 2 * b * hq) * d * e,
            "flops": 4 * hq * d * (seen + b * case["prefix"])}


# ---------------------------------------------------------------- the inputs

def prepare(case, seed):
    dev = "cuda"
    g = torch.Generator(device=dev).manual_seed(seed)
    dt = _DT[case["dtype"]]
    hq, hkv, d, page = case["hq"], case["hkv"], case["d"], case["page"]
    rows = _lengths(case)
    b = len(rows)
    kv = torch.tensor([r[2] for r in rows], dtype=torch.int32, device=dev)
    new = torch.tensor([r[1] for r in rows], dtype=torch.int32, device=dev)
    need = [-(-r[2] // page) for r in rows]
    max_pages = max(1, max(need))
    n_prefix = -(-case["prefix"] // page)
    n_pages = sum(need) + n_prefix + 3

    def normal(*shape):
        return torch.randn(*shape, device=dev, generator=g, dtype=torch.float32 if dt == torch.float32 else dt)

    # a pool that has been in use: every sequence's pages lie anywhere in it
    perm = torch.randperm(n_pages, device=dev, generator=g).to(torch.int32)
    width = torch.tensor(need, device=dev)
    col = torch.arange(max_pages, device=dev)[None, :]
    at = (width.cumsum(0) - width)[:, None] + col
    table = torch.where(col < width[:, None], perm[at.clamp(max=n_pages - 1)], torch.full_like(at, -1, dtype=torch.int32))
    s = {"case": dict(case), "k_pages": normal(n_pages, hkv, page, d), "v_pages": normal(n_pages, hkv, page, d),
         "table": table.to(torch.int32).contiguous(), "kv_lens": kv, "scale": 1.0 / math.sqrt(d)}
    # the first key of a sequence draws attention, as first tokens do
    first = table[:, 0].clamp(min=0).long()
    s["k_pages"][first, :, 0] = 2.0 * s["k_pages"][first, :, 0]
    n = int(sum(r[1] for r in rows))
    if case["op"] in ("append", "prefill"):
        s["cu_q"] = torch.cat([torch.zeros(1, dtype=torch.int32, device=dev), new.cumsum(0).to(torch.int32)])
        s["max_new"] = max(r[1] for r in rows)
    if case["op"] == "append":
        # the projection's output: queries, keys and values of a token side by side
        s["qkv"] = normal(n, (hq + 2 * hkv) * d)
        half = case["rot"] // 2
        inv = 10000.0 ** (-torch.arange(half, device=dev, dtype=torch.float64) / half)
        ang = torch.arange(max(r[2] for r in rows) + 1, device=dev, dtype=torch.float64)[:, None] * inv
        s["cos"], s["sin"] = ang.cos().float(), ang.sin().float()
    else:
        s["q"] = normal(n, hq, d)
    if case["op"] == "prefix":
        s["prefix_table"] = perm[sum(need):sum(need) + n_prefix].contiguous()
    return s


# ---------------------------------------------------------------- plain forms

def _rows_of(pages, table):
    """The rows that a table of pages [..., P] lists, as [..., hkv, P * page, d] in 32 bits."""
    x = pages[table.clamp(min=0).long()].float()
    x = x.movedim(-4, -3)
    return x.reshape(*x.shape[:-3], x.shape[-3] * x.shape[-2], x.shape[-1])


def _softmax_over(s, vis):
    """exp(s - max) over the visible entries of the last axis, and its sum; zeros where nothing is visible."""
    s = s.masked_fill(~vis, -math.inf)
    m = s.amax(-1, keepdim=True)
    p = (s - m.masked_fill(m == -math.inf, 0.0)).exp()
    return p, p.sum(-1, keepdim=True)


def _sees(case, pos, key):
    vis = key <= pos
    if case["window"]:
        vis = vis & ((key > pos - case["window"]) | (key < case["sinks"]))
    return vis


def _token_places(s):
    """Of each new token: its sequence, its index there, its row in the cache."""
    cu = s["cu_q"].long()
    n = (s["qkv"] if "qkv" in s else s["q"]).shape[0]
    tok = torch.arange(n, device=cu.device)
    seq = torch.searchsorted(cu, tok, right=True) - 1
    t = tok - cu[seq]
    return seq, t, s["kv_lens"].long()[seq] - (cu[seq + 1] - cu[seq]) + t


def _turned(x, cos, sin, case):
    r, half = case["rot"], case["rot"] // 2
    x = x.float()
    cos, sin = cos[:, None, :], sin[:, None, :]
    if case["pairs"]:
        a, b = x[..., 0:r:2], x[..., 1:r:2]
        y = torch.stack([a * cos - b * sin, b * cos + a * sin], -1).flatten(-2)
    else:
        a, b = x[..., :half], x[..., half:r]
        y = torch.cat([a * cos - b * sin, b * cos + a * sin], -1)
    return torch.cat([y, x[..., r:]], -1)


def _plain_append(s):
    case = s["case"]
    hq, hkv, d, page = case["hq"], case["hkv"], case["d"], case["page"]
    seq, _, pos = _token_places(s)
    q, k, v = (x.view(x.shape[0], -1, d) for x in s["qkv"].split([hq * d, hkv * d, hkv * d], 1))
    cos, sin = s["cos"][pos], s["sin"][pos]
    at = s["table"][seq, pos // page].long()
    dt = s["k_pages"].dtype
    s["k_pages"][at, :, pos % page] = _turned(k, cos, sin, case).to(dt)
    s["v_pages"][at, :, pos % page] = v
    return s["k_pages"], s["v_pages"], _turned(q, cos, sin, case).to(dt)


def _plain_decode(s):
    case, q = s["case"], s["q"]
    b, hq, d = q.shape
    hkv = case["hkv"]
    k, v = _rows_of(s["k_pages"], s["table"]), _rows_of(s["v_pages"], s["table"])
    key = torch.arange(k.shape[2], device=q.device)
    vis = _sees(case, s["kv_lens"].long()[:, None] - 1, key)[:, None, None, :]
    p, l = _softmax_over((q.float() * s["scale"]).view(b, hkv, hq // hkv, d) @ k.transpose(-1, -2), vis)
    return ((p @ v) / l.masked_fill(l == 0, 1.0)).reshape(b, hq, d).to(q.dtype)


def _plain_prefill(s):
    case, q = s["case"], s["q"]
    n, hq, d = q.shape
    hkv, t = case["hkv"], s["max_new"]
    seq, at, _ = _token_places(s)
    cu, kv = s["cu_q"].long(), s["kv_lens"].long()
    b = kv.shape[0]
    k, v = _rows_of(s["k_pages"], s["table"]), _rows_of(s["v_pages"], s["table"])
    step = torch.arange(t, device=q.device)
    rows = (q.float() * s["scale"])[(cu[:-1, None] + step).clamp(max=n - 1)]           # [b, t, hq, d]
    rows = rows.view(b, t, hkv, hq // hkv, d).permute(0, 2, 3, 1, 4)
    pos = (kv - (cu[1:] - cu[:-1]))[:, None] + step
    vis = _sees(case, pos[:, :, None], torch.arange(k.shape[2], device=q.device))[:, None, None]
    p, l = _softmax_over(rows @ k[:, :, None].transpose(-1, -2), vis)
    out = (p @ v[:, :, None]) / l.masked_fill(l == 0, 1.0)                               # [b, hkv, g, t, d]
    return out.permute(0, 3, 1, 2, 4).reshape(b, t, hq, d)[seq, at].to(q.dtype)


def _plain_prefix(s):
    case, q = s["case"], s["q"]
    b, hq, d = q.shape
    hkv, n = case["hkv"], case["prefix"]
    g = hq // hkv
    rows = (q.float() * s["scale"]).view(b, hkv, g, d)
    pk, pv = _rows_of(s["k_pages"], s["prefix_table"])[:, :n], _rows_of(s["v_pages"], s["prefix_table"])[:, :n]
    k, v = _rows_of(s["k_pages"], s["table"]), _rows_of(s["v_pages"], s["table"])
    shared = rows.transpose(0, 1).reshape(hkv, b * g, d) @ pk.transpose(-1, -2)          # once for all sequences
    shared = shared.view(hkv, b, g, n).transpose(0, 1)
    mine = rows @ k.transpose(-1, -2)
    key = torch.arange(k.shape[2], device=q.device)
    vis = (key < s["kv_lens"][:, None])[:, None, None, :].expand_as(mine)
    p, l = _softmax_over(torch.cat([shared, mine], -1), torch.cat([torch.ones_like(shared, dtype=torch.bool), vis], -1))
    ps = p[..., :n].transpose(0, 1).reshape(hkv, b * g, n) @ pv
    out = ps.view(hkv, b, g, d).transpose(0, 1) + p[..., n:] @ v
    return (out / l).reshape(b, hq, d).to(q.dtype)


# ---------------------------------------------------------------- one pass

def run(s):
    case = s["case"]
    op = case["op"]
    if not own:
        return {"append": _plain_append, "decode": _plain_decode, "prefill": _plain_prefill,
                "prefix": _plain_prefix}[op](s)
    import streaming_attention_b200 as sa
    kp, vp, table, kv = s["k_pages"], s["v_pages"], s["table"], s["kv_lens"]
    if op == "append":
        hq, hkv, d = case["hq"], case["hkv"], case["d"]
        q, k, v = (x.view(x.shape[0], -1, d) for x in s["qkv"].split([hq * d, hkv * d, hkv * d], 1))
        q_out = sa.paged_append(k, v, kp, vp, table, kv, cu_q=s["cu_q"], q=q, rope=(s["cos"], s["sin"]),
                                interleaved=case["pairs"])
        return kp, vp, q_out
    if op == "decode":
        return sa.attn_paged_decode(s["q"], kp, vp, table, kv, s["scale"], window=case["window"], sinks=case["sinks"])
    if op == "prefill":
        return sa.attn_paged_prefill(s["q"], kp, vp, table, kv, s["cu_q"], s["scale"], window=case["window"],
                                     sinks=case["sinks"])
    return sa.attn_paged_decode_prefix(s["q"], kp, vp, s["prefix_table"], case["prefix"], table, kv, s["scale"])


# ---------------------------------------------------------------- the definition, in 64 bits

def exact(case, seed):
    s = prepare(case, seed)
    hq, hkv, d, page = case["hq"], case["hkv"], case["d"], case["page"]
    g = hq // hkv
    table, rows = s["table"].tolist(), _lengths(case)
    if case["op"] == "append":
        kp, vp = s["k_pages"].double(), s["v_pages"].double()
        x = s["qkv"].double().view(-1, hq + 2 * hkv, d)
        half = case["rot"] // 2
        lo = torch.arange(half, device=x.device) * (2 if case["pairs"] else 1)
        hi = lo + (1 if case["pairs"] else half)
        at = 0
        for b, (past, new, kv) in enumerate(rows):
            y = x[at:at + new].clone()
            c, sn = (s[t][past:kv].double()[:, None, :] for t in ("cos", "sin"))
            turn = y[:, :hq + hkv]
            u, w = turn[..., lo].clone(), turn[..., hi].clone()
            turn[..., lo] = c * u - sn * w
            turn[..., hi] = c * w + sn * u
            x[at:at + new] = y
            for j in range(past // page, -(-kv // page)):
                r0, r1 = max(past, j * page), min(kv, (j + 1) * page)
                part = y[r0 - past:r1 - past].transpose(0, 1)
                kp[table[b][j], :, r0 - j * page:r1 - j * page] = part[hq:hq + hkv]
                vp[table[b][j], :, r0 - j * page:r1 - j * page] = part[hq + hkv:]
            at += new
        return kp, vp, x[:, :hq].contiguous()
    out = torch.zeros(s["q"].shape, dtype=torch.float64, device="cuda")

    def cached(pages, ids, count):
        return pages[torch.tensor(ids, device="cuda", dtype=torch.long)].double().transpose(0, 1).reshape(hkv, -1, d)[:, :count]

    before = None
    if case["op"] == "prefix":
        before = [cached(s[n], s["prefix_table"].tolist(), case["prefix"]) for n in ("k_pages", "v_pages")]
    at = 0
    for b, (past, new, kv) in enumerate(rows):
        if case["op"] != "prefill":
            past = kv - 1
        ids = table[b][:-(-kv // page)]
        k, v = cached(s["k_pages"], ids, kv), cached(s["v_pages"], ids, kv)
        if before is not None:
            k, v = torch.cat([before[0], k], 1), torch.cat([before[1], v], 1)
            past = k.shape[1] - 1
        if k.shape[1]:
            i = past + torch.arange(new, device="cuda")[:, None]
            j = torch.arange(k.shape[1], device="cuda")[None, :]
            hidden = j > i
            if case["window"]:
                hidden = hidden | ((i - j >= case["window"]) & (j >= case["sinks"]))
            for h in range(hkv):
                q = s["q"][at:at + new, h * g:(h + 1) * g].double().transpose(0, 1)      # [g, new, d]
                w = torch.softmax((q @ k[h].T * s["scale"]).masked_fill(hidden, -math.inf), -1)
                out[at:at + new, h * g:(h + 1) * g] = (w @ v[h]).transpose(0, 1)
        at += new
    return out
