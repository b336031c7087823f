"""Performance cases of the paged key/value cache: what a program that serves many sequences has it do.

The cache holds each sequence's keys and values in pages of a shared pool, as f16 or as 4-bit codes (blocks of 32
dims, value = (code - 8) * scale); a table names the pages of each sequence.  A batch is `seqs` sequences with 1 to
`q` new tokens each: tokens q_start[i] .. q_start[i + 1] - 1 belong to sequence i and are the last ones of its
kv_len[i] positions.

Kinds (hd head dim, kvh KV heads, g query heads for each of them):
  append   head norms + rotation of raw q|k|v rows, K and V into their pages, q out   PagedKV.append_dev
           (4 bits: then the new rows are read back as f16, PagedKV.gather_dev)
  attn     attention of prepped queries over the cache: causal, over all keys or      PagedKV.attn_dev
           over a sliding window and the first `sinks` positions
  step     both, as each layer of a serving step runs them
"""
import math
import os
import random
import sys

import numpy as np
import torch

own = False

EPS = 1e-6
_PKG = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "e4b-webgpu_amd")


def _case(kind, type, hd, kvh, g, page, seqs, q, kv, x="f32", qt="f32", window=0, sinks=0, ragged=False, scale=1.0,
          name=None):
    """x: type of the raw rows, qt: of the prepped queries, kv: positions of the longest sequence."""
    c = dict(kind=kind, type=type, hd=hd, kvh=kvh, g=g, page=page, seqs=seqs, q=q, kv=kv, x=x, qt=qt, window=window,
             sinks=sinks, ragged=ragged, scale=scale)
    return dict(c, name=name) if name else c


def listed():
    return [
        # one decoded token of one conversation: nothing but latency
        _case("append", "f16", 256, 2, 4, 64, 1, 1, 700, name="append_1"),
        # a decode step of a full batch
        _case("append", "f16", 256, 2, 4, 64, 64, 1, 2048, ragged=True, name="append_64"),
        # a few prompts of unlike lengths at once, queries kept in 16 bits for the matrix cores
        _case("append", "f16", 256, 8, 2, 128, 5, 1000, 1000, qt="f16", ragged=True, name="append_prompts"),
        # the same batch of decoded tokens into 4 bits
        _case("append", "q4", 256, 2, 4, 64, 64, 1, 2048, ragged=True, name="append_q4_64"),
        # a long prompt's chunk into 4 bits, heads of 512 dims
        _case("append", "q4", 512, 2, 8, 32, 3, 701, 9000, x="f16", qt="f16", ragged=True, name="append_q4_chunk"),
        # one decoded token early in a conversation
        _case("attn", "f16", 256, 2, 4, 64, 1, 1, 300, name="attn_1"),
        # a full batch late in long conversations: the cache's bytes are the time
        _case("attn", "f16", 256, 2, 4, 64, 64, 1, 8192, qt="f16", name="attn_64x8192"),
        # a sliding layer with sinks, sequences of unlike lengths, small pages
        _case("attn", "f16", 256, 2, 4, 16, 32, 1, 16000, window=512, sinks=4, ragged=True, name="attn_window_sinks"),
        # the last quarter of four prompts of 4096 tokens: the matrix cores' work
        _case("attn", "f16", 256, 2, 4, 64, 4, 1024, 4096, qt="f16", name="attn_prompts"),
        # one decoded token at the end of the longest context, 4-bit cache
        _case("attn", "q4", 256, 2, 4, 128, 1, 1, 32767, name="attn_q4_32767"),
        # a decode batch over a 4-bit cache, heads of 512 dims
        _case("attn", "q4", 512, 2, 8, 64, 48, 1, 4096, qt="f16", ragged=True, scale=512 ** -0.5, name="attn_q4_48"),
        # a layer of a mixed batch: short chunks appended to a 4-bit cache and attended over window and sinks
        _case("step", "q4", 256, 2, 4, 32, 6, 300, 3000, qt="f16", window=1024, sinks=4, ragged=True, name="step_q4"),
    ]


def _log(rng, lo, hi):
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    kind, type = rng.choice(["append", "attn", "attn", "step"]), rng.choice(["f16", "q4"])
    hd, kvh, g = rng.choice([128, 256, 256, 512]), rng.choice([1, 2, 2, 4, 8]), rng.choice([1, 2, 3, 4, 4, 6, 8])
    page, seqs = rng.choice([16, 32, 64, 128]), _log(rng, 1, 64)
    q = 1 if rng.random() < 0.5 else _log(rng, 2, 1024)
    kv = max(q, _log(rng, 1, 32767))
    # no more than the largest listed cases: appended elements, cache bytes, products
    while seqs * q * (g + 2) * kvh * hd > 4e6 * (5 if kind == "append" else 1) and q > 1:
        q = max(1, q * 2 // 3)
    while seqs * kv * kvh * hd > 64 * 8192 * 2 * 256 and kv > q:
        kv = max(q, kv * 2 // 3)
    while seqs * q * kvh * g * kv * hd > 4 * 1024 * 8 * 4096 * 256 and seqs > 1:
        seqs = max(1, seqs * 2 // 3)
    while q * kvh * g * kv * hd > 4 * 1024 * 8 * 4096 * 256 and kv > q:
        kv = max(q, kv * 2 // 3)
    window = rng.choice([0, 0, 512, _log(rng, 1, 4096)])
    return _case(kind, type, hd, kvh, g, page, seqs, q, kv, x=rng.choice(["f32", "f16"]), qt=rng.choice(["f32", "f16"]),
                 window=window, sinks=rng.choice([0, 4, rng.randrange(1, 70)]) if window else 0,
                 ragged=rng.random() < 0.7, scale=rng.choice([1.0, hd ** -0.5]))


def _lengths(c):
    """q_len and kv_len of each sequence; they follow from the case alone."""
    if not c["ragged"]:
        return [c["q"]] * c["seqs"], [c["kv"]] * c["seqs"]
    r = random.Random("%(seqs)d %(q)d %(kv)d %(page)d" % c)
    q = [c["q"]] + [r.randint(1, c["q"]) for _ in range(c["seqs"] - 1)]
    kv = [c["kv"]] + [r.randint(max(n, c["kv"] // 8), c["kv"]) for n in q[1:]]
    return q, kv


# ---- inputs --------------------------------------------------------------------------------------------------------

def _dtype(name):
    return torch.float16 if name == "f16" else torch.float32


def _inv_freq(c):
    angles = c["hd"] // 8 if c["hd"] == 512 else c["hd"] // 2  # heads of 512 dims rotate a quarter of their pairs
    theta = 1e4 if c["window"] else 1e6
    return (theta ** (-2.0 * np.arange(angles) / c["hd"])).astype(np.float32)


def _quantise(x):
    """Blocks of 32 along the last dim -> (codes 0..15, scales as f16)."""
    b = x.reshape(*x.shape[:-1], x.shape[-1] // 32, 32)
    m = b.abs()
    at = torch.where(m == m.amax(-1, keepdim=True), torch.arange(32, device=x.device), 32).amin(-1, keepdim=True)
    # the scale: the block's largest element is -8 steps, rounded to 8 significant bits, so that 3-bit steps of it
    # are exact in f16
    u = (torch.gather(b, -1, at).double() / -8).view(torch.int64)
    u = (u + ((u >> 45) & 1) + (1 << 44) - 1) >> 45 << 45
    d = u.view(torch.float64).clamp(-8160, 8160).half()
    by = torch.where(d == 0, torch.ones_like(d), d).to(x.dtype)
    code = ((b / by).round() + 8).clamp(0, 15)
    return torch.where(d == 0, torch.full_like(code, 8), code).to(torch.int32).reshape(x.shape), d[..., 0]


def _pack(codes):
    """Codes [..., hd] -> bytes [..., hd / 2]: eight dims in four bytes, dims 0 2 1 3 in the low and 4 6 5 7 in the
    high halves."""
    e = codes.reshape(*codes.shape[:-1], codes.shape[-1] // 8, 8)
    b = e[..., [0, 2, 1, 3]] + 16 * e[..., [4, 6, 5, 7]]
    return b.to(torch.uint8).reshape(*codes.shape[:-1], codes.shape[-1] // 2)


def _pool(c, n_pages, rows):
    """Rows [n_pages, kvh, page, hd] as a pool of the case's type."""
    if c["type"] == "f16":
        return rows.half()
    codes, d = _quantise(rows)
    n = (n_pages, c["kvh"], -1)
    return torch.cat([_pack(codes).reshape(n), d.contiguous().view(torch.uint8).reshape(n)], -1)


def prepare(case, seed):
    c, gen = case, torch.Generator(device="cuda").manual_seed(seed)
    normal = lambda *s: torch.randn(*s, generator=gen, device="cuda")  # noqa: E731
    hd, kvh, qh, page = c["hd"], c["kvh"], c["kvh"] * c["g"], c["page"]
    q_len, kv_len = _lengths(c)
    blocks = [-(-n // page) for n in kv_len]
    n_pages, stride = sum(blocks) + 3, max(blocks) + 1
    order = np.random.default_rng(seed).permutation(n_pages).astype(np.int32)
    table, at = np.full((c["seqs"], stride), -1, np.int32), 0
    for i, n in enumerate(blocks):
        table[i, :n] = order[at:at + n]
        at += n
    half = lambda std: torch.empty(n_pages, kvh, page, hd, dtype=torch.float16, device="cuda").normal_(0, std, generator=gen)  # noqa: E731
    n_tok = sum(q_len)
    s = {"c": c, "n_tok": n_tok, "n_pages": n_pages, "max_q": max(q_len), "max_kv": max(kv_len),
         # keys as after their head norm and its weight, values of unit size
         "k": _pool(c, n_pages, half(0.25)), "v": _pool(c, n_pages, half(1.0)),
         "table": torch.from_numpy(table).cuda(),
         "q_start": torch.tensor(np.concatenate([[0], np.cumsum(q_len)]), dtype=torch.int32).cuda(),
         "kv_len": torch.tensor(kv_len, dtype=torch.int32).cuda(),
         "out": torch.empty(n_tok, qh * hd, dtype=torch.float16, device="cuda")}
    if c["kind"] == "attn":
        s["q"] = normal(n_tok, qh * hd).to(_dtype(c["qt"]))
    else:
        s.update(x=normal(n_tok, (qh + 2 * kvh) * hd).to(_dtype(c["x"])), inv=torch.from_numpy(_inv_freq(c)).cuda(),
                 qw=1 + 0.1 * normal(hd), kw=0.25 * (1 + 0.1 * normal(hd)),
                 q=torch.empty(n_tok, qh * hd, dtype=_dtype(c["qt"]), device="cuda"),
                 k_rows=torch.empty(n_tok, kvh, hd, dtype=torch.float16, device="cuda"),
                 v_rows=torch.empty(n_tok, kvh, hd, dtype=torch.float16, device="cuda"))
    return s


# ---- one pass ------------------------------------------------------------------------------------------------------

def _tokens(s):
    """Sequence and position of every token."""
    t = torch.arange(s["n_tok"], device="cuda", dtype=torch.int32)
    seq = torch.searchsorted(s["q_start"][1:], t, right=True)
    return seq, (s["kv_len"][seq] - s["q_start"][seq + 1] + t).long()


def _rms(x):
    return x * torch.rsqrt((x * x).mean(-1, keepdim=True) + EPS)


def _rotate(x, pos, inv):
    """Pairs (d, d + hd / 2), d < angles.  Angles in 64 bits: far positions are thousands of turns."""
    n, h = inv.numel(), x.shape[-1] // 2
    ang = pos.double()[:, None, None] * inv.double()
    cos, sin = ang.cos().to(x.dtype), ang.sin().to(x.dtype)
    a, b = x[..., :n], x[..., h:h + n]
    return torch.cat([a * cos - b * sin, x[..., n:h], b * cos + a * sin, x[..., h + n:]], -1)


def _append(s):
    c = s["c"]
    hd, kvh, qh, page = c["hd"], c["kvh"], c["kvh"] * c["g"], c["page"]
    seq, pos = _tokens(s)
    x = s["x"].to(torch.float64 if c["type"] == "q4" else torch.float32)  # 64 bits beside the borders of the codes
    x = x.reshape(s["n_tok"], qh + 2 * kvh, hd)
    q = _rotate(_rms(x[:, :qh]) * s["qw"].to(x.dtype), pos, s["inv"])
    k = _rotate(_rms(x[:, qh:qh + kvh]) * s["kw"].to(x.dtype), pos, s["inv"])
    v = _rms(x[:, qh + kvh:])
    q = q.reshape(s["n_tok"], qh * hd).to(_dtype(c["qt"]))
    pg, row = s["table"][seq, pos // page].long(), pos % page
    if c["type"] == "f16":
        s["k"][pg, :, row], s["v"][pg, :, row] = k.half(), v.half()
        return {"q": q, "k": s["k"], "v": s["v"]}
    got = {"q": q}
    for name, y in (("k", k), ("v", v)):
        codes, d = _quantise(y)
        cut = page * hd // 2
        s[name][..., :cut].unflatten(-1, (page, hd // 2))[pg, :, row] = _pack(codes)
        s[name][..., cut:].unflatten(-1, (page, hd // 16))[pg, :, row] = d.contiguous().view(torch.uint8)
        got[name] = ((codes - 8).float() * d.float().repeat_interleave(32, -1)).half()
    return got


def _rows(s, name):
    """The whole cache of every sequence, f32 [seqs, kvh, positions, hd]; what a missing page holds says nothing."""
    c = s["c"]
    hd, page = c["hd"], c["page"]
    p = s[name][s["table"].clamp(min=0).long()].transpose(1, 2)  # [seqs, kvh, blocks, ...]
    if c["type"] == "f16":
        return p.float().flatten(2, 3)
    cut = page * hd // 2
    b = p[..., :cut].reshape(*p.shape[:-1], page, hd // 8, 4).short()
    lo, hi = b & 15, b >> 4
    e = torch.cat([lo[..., [0, 2, 1, 3]], hi[..., [0, 2, 1, 3]]], -1).reshape(*p.shape[:-1], page, hd)
    d = p[..., cut:].contiguous().view(torch.float16).reshape(*p.shape[:-1], page, hd // 32)
    return ((e - 8).float().unflatten(-1, (-1, 32)) * d.float()[..., None]).flatten(-2).flatten(2, 3)


def _attend(s, q):
    c = s["c"]
    hd, kvh, g, page, mq = c["hd"], c["kvh"], c["g"], c["page"], s["max_q"]
    n = s["table"].shape[1] * page
    k = torch.arange(n, device="cuda")
    q_len = s["q_start"][1:] - s["q_start"][:-1]
    p = (s["kv_len"] - q_len)[:, None] + torch.arange(mq, device="cuda")  # [seqs, mq]
    sees = k <= p[..., None]
    if c["window"]:
        sees &= (k > p[..., None] - c["window"]) | (k < c["sinks"])
    sees &= (s["table"] >= 0).repeat_interleave(page, 1)[:, None]
    sees = sees[:, None].repeat_interleave(g, 2)  # [seqs, 1, mq g, n]
    at = (s["q_start"][:-1, None] + torch.arange(mq, device="cuda")).clamp(max=s["n_tok"] - 1).long()
    rows = q[at].float().reshape(c["seqs"], mq, kvh, g, hd).transpose(1, 2).reshape(c["seqs"], kvh, mq * g, hd)
    w = torch.matmul(rows, _rows(s, "k").transpose(2, 3)) * c["scale"]
    w = w.masked_fill(~sees, float("-inf"))
    top = w.amax(-1, keepdim=True)
    w = torch.exp(w - top.masked_fill(top == float("-inf"), 0.0))
    total = w.sum(-1, keepdim=True)
    o = torch.matmul(w, _rows(s, "v")) / torch.where(total == 0, torch.ones_like(total), total)
    o = o.reshape(c["seqs"], kvh, mq, g, hd).transpose(1, 2).reshape(c["seqs"], mq, kvh * g * hd)
    seq, pos = _tokens(s)
    return o[seq, pos - p[seq, 0]].half()


def _call(s):
    """The framework's calls."""
    if _PKG not in sys.path:
        sys.path.insert(0, _PKG)
    from e4b import kernels as K
    from e4b._lib import DT_F16, DT_F32
    c = s["c"]
    if "kv" not in s:  # the descriptions of cache and batch, which a program keeps beside its buffers
        a = {n: t.data_ptr() for n, t in s.items() if isinstance(t, torch.Tensor)}
        s["kv"] = K.PagedKV(c["type"], c["kvh"], c["hd"], c["page"], s["n_pages"], s["table"].shape[1], k=a["k"],
                            v=a["v"], table=a["table"])
        s["batch"] = K.KvBatch(a["q_start"], a["kv_len"], c["seqs"], s["n_tok"], s["max_q"], s["max_kv"])
        if "x" in s:
            s["prep"] = K.HeadPrep(a["qw"], a["kw"], a["inv"], s["inv"].numel(), EPS)
    kv, qh, qt = s["kv"], c["kvh"] * c["g"], DT_F16 if c["qt"] == "f16" else DT_F32
    got = {}
    if c["kind"] != "attn":
        kv.append_dev(s["batch"], s["prep"], s["x"].data_ptr(), DT_F16 if c["x"] == "f16" else DT_F32, qh,
                      s["q"].data_ptr(), qt)
        got = {"q": s["q"], "k": s["k"], "v": s["v"]}
    if c["kind"] == "append" and c["type"] == "q4":
        kv.gather_dev(s["batch"], s["k_rows"].data_ptr(), s["v_rows"].data_ptr())
        got.update(k=s["k_rows"], v=s["v_rows"])
    if c["kind"] == "append":
        return got
    kv.attn_dev(s["batch"], s["q"].data_ptr(), qt, qh, s["out"].data_ptr(), window=c["window"], sinks=c["sinks"],
                scale=c["scale"])
    return {"out": s["out"]} if c["kind"] == "attn" else {"q": s["q"], "out": s["out"]}


def run(state):
    if own:
        return _call(state)
    if state["c"]["kind"] == "append":
        return _append(state)
    if state["c"]["kind"] == "attn":
        return {"out": _attend(state, state["q"])}
    q = _append(state)["q"]
    return {"q": q, "out": _attend(state, q)}


# ---- what a pass cannot do without ---------------------------------------------------------------------------------

def _seen(lo, hi, window, sinks):
    """(keys that some query at positions lo .. hi sees, sum of the keys that each of them sees)"""
    p = np.arange(lo, hi + 1)
    if not window:
        return hi + 1, int((p + 1).sum())
    first = np.maximum(0, p - window + 1)
    return hi + 1 - int(first[0]) + min(sinks, int(first[0])), int((p - first + 1 + np.minimum(first, sinks)).sum())


def work(case):
    c = case
    hd, kvh, qh = c["hd"], c["kvh"], c["kvh"] * c["g"]
    q_len, kv_len = _lengths(c)
    n, row = sum(q_len), hd * 2 if c["type"] == "f16" else hd // 2 + hd // 16  # bytes of one head's K or V
    q_bytes = n * qh * hd * (2 if c["qt"] == "f16" else 4)
    size, flops = 4 * len(q_len) * 2, 0
    if c["kind"] != "attn":
        size += n * (qh + 2 * kvh) * hd * (2 if c["x"] == "f16" else 4) + q_bytes + 2 * n * kvh * row
        flops += 10 * n * (qh + 2 * kvh) * hd
        if c["kind"] == "append" and c["type"] == "q4":
            size += 2 * n * kvh * (row + 2 * hd)
    if c["kind"] != "append":
        seen = [_seen(k - m, k - 1, c["window"], c["sinks"]) for m, k in zip(q_len, kv_len)]
        size += sum(k for k, _ in seen) * kvh * 2 * row + q_bytes + n * qh * hd * 2
        flops += 4 * hd * qh * sum(p for _, p in seen)
    return {"bytes": size, "flops": flops}


# ---- 64 bits, from the definitions ---------------------------------------------------------------------------------

_DIM_AT = [0, 16, 8, 24, 4, 20, 12, 28]  # bit of each of eight dims in their 32-bit word


def _exact_quantised(x):
    """What 4-bit rows [.., hd] stand for."""
    blocks = x.unflatten(-1, (-1, 32))
    low, high = blocks.amin(-1), blocks.amax(-1)
    first_low = (blocks == low[..., None]).int().argmax(-1)
    first_high = (blocks == high[..., None]).int().argmax(-1)
    big = torch.where((-low > high) | ((-low == high) & (first_low < first_high)), low, high)
    m, e = torch.frexp(big / -8)
    d = torch.ldexp((m * 256).round(), e - 8).half().double()[..., None]
    steps = torch.where(d == 0, torch.zeros_like(blocks), blocks / torch.where(d == 0, torch.ones_like(d), d))
    return (steps.round().clamp(-8, 7) * d).flatten(-2)


def _exact_cache(c, pool):
    """A pool's rows in 64 bits, [n_pages, kvh, page, hd]."""
    if c["type"] == "f16":
        return pool.double()
    hd, page = c["hd"], c["page"]
    words = pool[..., :page * hd // 2].contiguous().view(torch.int32).unflatten(-1, (page, hd // 8))
    codes = torch.stack([(words >> b) & 15 for b in _DIM_AT], -1).flatten(-2)
    d = pool[..., page * hd // 2:].contiguous().view(torch.float16).unflatten(-1, (page, hd // 32)).double()
    return (codes.double() - 8) * d.repeat_interleave(32, -1)


def exact(case, seed):
    c, s = case, prepare(case, seed)
    hd, kvh, g, page = c["hd"], c["kvh"], c["g"], c["page"]
    qh = kvh * g
    q_len, kv_len = _lengths(c)
    pools = {n: s[n] for n in ("k", "v")}
    norm = lambda y: y / ((y ** 2).sum(-1, keepdim=True) / hd + EPS).sqrt()  # noqa: E731

    def turn(y, p):
        n = s["inv"].numel()
        z = torch.polar(torch.ones(1, dtype=torch.float64, device="cuda"), p[:, None] * s["inv"].double())[:, None]
        z = torch.complex(y[..., :n], y[..., hd // 2:hd // 2 + n]) * z
        y = y.clone()
        y[..., :n], y[..., hd // 2:hd // 2 + n] = z.real, z.imag
        return y

    q_all, out_all, k_new, v_new = [], [], [], []
    full = {n: _exact_cache(c, pools[n]) for n in pools} if c["kind"] == "append" and c["type"] == "f16" else None
    at = 0
    for i, (m, n) in enumerate(zip(q_len, kv_len)):
        p = torch.arange(n - m, n, device="cuda", dtype=torch.float64)
        if c["kind"] != "attn":
            x = s["x"][at:at + m].double().reshape(m, -1, hd)
            q = turn(norm(x[:, :qh]) * s["qw"].double(), p)
            new = [turn(norm(x[:, qh:qh + kvh]) * s["kw"].double(), p), norm(x[:, qh + kvh:])]
            if c["type"] == "q4":
                new = [_exact_quantised(y) for y in new]
            k_new.append(new[0])
            v_new.append(new[1])
            if full is not None:
                where = s["table"][i, p.long() // page].long()
                for name, y in zip(("k", "v"), new):
                    full[name][where, :, p.long() % page] = y
        else:
            q = s["q"][at:at + m].double().reshape(m, qh, hd)
        q_all.append(q.reshape(m, -1))
        if c["kind"] != "append":
            if c["kind"] == "step":
                q = q.to(_dtype(c["qt"])).double()  # the queries as the attention reads them
            pages = s["table"][i, :-(-n // page)].long()
            rows = {}
            for j, name in enumerate(("k", "v")):
                r = _exact_cache(c, pools[name][pages]).transpose(0, 1).flatten(1, 2)[:, :n].clone()
                if c["kind"] == "step":
                    y = new[j] if c["type"] == "q4" else new[j].half().double()
                    r[:, n - m:] = y.transpose(0, 1)
                rows[name] = r
            keys = torch.arange(n, device="cuda")
            dist = p.long()[:, None] - keys
            sees = dist >= 0
            if c["window"]:
                sees &= (dist < c["window"]) | (keys < c["sinks"])[None]
            heads = []
            for h in range(qh):
                w = (q[:, h] @ rows["k"][h // g].T) * c["scale"]
                w = torch.softmax(w.masked_fill(~sees, float("-inf")), -1).masked_fill(~sees, 0.0)
                heads.append(w @ rows["v"][h // g])
            out_all.append(torch.stack(heads, 1).reshape(m, -1))
        at += m
    if c["kind"] == "attn":
        return {"out": torch.cat(out_all)}
    if c["kind"] == "step":
        return {"q": torch.cat(q_all), "out": torch.cat(out_all)}
    if c["type"] == "f16":
        return {"q": torch.cat(q_all), "k": full["k"], "v": full["v"]}
    return {"q": torch.cat(q_all), "k": torch.cat(k_new), "v": torch.cat(v_new)}
