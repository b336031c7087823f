"""The paged key/value cache in numpy, 64 bits, from its definitions: pools and
tables as the library lays them out, append, read-back and attention."""
import numpy as np

NONE = 0xFFFFFFFF
DIM_BIT = np.array([0, 16, 8, 24, 4, 20, 12, 28], np.uint32)


def q4_encode(x):
    """Rows [..., hd] -> (codes 0..15, scales f16 [..., hd / 32])."""
    x = np.asarray(x, np.float64)
    b = x.reshape(*x.shape[:-1], -1, 32)
    a = np.take_along_axis(b, np.abs(b).argmax(-1)[..., None], -1)
    m, e = np.frexp(a / -8)
    d = np.clip(np.ldexp(np.rint(m * 256), e - 8), -8160, 8160).astype(np.float16)
    d[~np.isfinite(b).all(-1, keepdims=True)] = np.nan
    with np.errstate(all="ignore"):
        s = np.clip(np.rint(b / d.astype(np.float64)), -8, 7)
    s[~np.isfinite(s)] = 0
    s = np.where((d == 0) | np.isnan(d), 0, s)
    return (s + 8).astype(np.uint32).reshape(x.shape), d[..., 0]


def q4_bytes(codes):
    w = (codes.reshape(*codes.shape[:-1], -1, 8) << DIM_BIT).sum(-1).astype(np.uint32)
    return np.ascontiguousarray(w).view(np.uint8)


class Cache:
    """Host image of a pool pair: rows(page, head, row) in the library's layout."""

    def __init__(self, kind, kvh, hd, page, n_pages, n_seq, stride):
        self.kind, self.kvh, self.hd, self.page, self.n_pages, self.stride = kind, kvh, hd, page, n_pages, stride
        self.table = np.full((n_seq, stride), NONE, np.uint32)
        if kind == "f16":
            self.pools = {n: np.full((n_pages, kvh, page, hd), np.nan, np.float16) for n in "kv"}
        else:  # codes 0xAA and NaN scales: what was never written
            self.codes = {n: np.full((n_pages, kvh, page, hd // 2), 0xAA, np.uint8) for n in "kv"}
            self.scales = {n: np.full((n_pages, kvh, page, hd // 32), np.nan, np.float16) for n in "kv"}

    def bytes(self, n):
        if self.kind == "f16":
            return self.pools[n].view(np.uint8).reshape(-1)
        c = self.codes[n].reshape(self.n_pages, self.kvh, -1)
        s = np.ascontiguousarray(self.scales[n]).view(np.uint8).reshape(self.n_pages, self.kvh, -1)
        return np.ascontiguousarray(np.concatenate([c, s], -1)).reshape(-1)

    def set_bytes(self, n, raw):
        if self.kind == "f16":
            self.pools[n] = raw.view(np.float16).reshape(self.pools[n].shape).copy()
            return
        cut = self.page * self.hd // 2
        r = raw.reshape(self.n_pages, self.kvh, -1)
        self.codes[n] = r[..., :cut].reshape(self.codes[n].shape).copy()
        self.scales[n] = np.ascontiguousarray(r[..., cut:]).view(np.float16).reshape(self.scales[n].shape).copy()

    def page_of(self, seq, pos):
        b = pos // self.page
        if pos < 0 or b >= self.stride or self.table[seq, b] >= self.n_pages:
            return -1
        return int(self.table[seq, b])

    def put(self, n, seq, pos, rows):
        """rows [kvh][hd] in 64 bits"""
        pg, r = self.page_of(seq, pos), pos % self.page
        if pg < 0:
            return
        if self.kind == "f16":
            with np.errstate(over="ignore"):
                self.pools[n][pg, :, r] = rows.astype(np.float16)
        else:
            codes, d = q4_encode(rows)
            self.codes[n][pg, :, r], self.scales[n][pg, :, r] = q4_bytes(codes), d

    def get(self, n, seq, pos):
        """-> [kvh][hd] float64, or None"""
        pg, r = self.page_of(seq, pos), pos % self.page
        if pg < 0:
            return None
        if self.kind == "f16":
            return self.pools[n][pg, :, r].astype(np.float64)
        w = np.ascontiguousarray(self.codes[n][pg, :, r]).view(np.uint32)
        c = ((w[..., None] >> DIM_BIT) & 15).reshape(self.kvh, self.hd).astype(np.float64) - 8
        return c * np.repeat(self.scales[n][pg, :, r].astype(np.float64), 32, -1)

    def fill(self, rng, kv_len, k_std=0.25, first=None):
        """Gives every sequence its pages (in random order) and random rows."""
        need = [-(-int(n) // self.page) for n in kv_len]
        assert sum(need) <= self.n_pages
        order, at = rng.permutation(self.n_pages), 0
        for i, n in enumerate(need):
            self.table[i, :n] = order[at:at + n]
            at += n
            for pos in range(int(kv_len[i])):
                self.put("k", i, pos, k_std * rng.standard_normal((self.kvh, self.hd)))
                self.put("v", i, pos, rng.standard_normal((self.kvh, self.hd)))


def spans(q_len, kv_len):
    """(sequence, first token, first position, tokens) of each sequence"""
    at = 0
    for i, (m, n) in enumerate(zip(q_len, kv_len)):
        yield i, at, int(n) - int(m), int(m)
        at += int(m)


def rms(x, eps):
    return x / np.sqrt((x * x).mean(-1, keepdims=True) + eps)


def rotate(x, pos, inv_freq):
    n, h = len(inv_freq), x.shape[-1] // 2
    y, a = x.copy(), float(pos) * inv_freq.astype(np.float64)
    y[..., :n] = x[..., :n] * np.cos(a) - x[..., h:h + n] * np.sin(a)
    y[..., h:h + n] = x[..., h:h + n] * np.cos(a) + x[..., :n] * np.sin(a)
    return y


def append(cache, q_len, kv_len, x, q_heads, q_norm, k_norm, inv_freq, eps, v_rms=True, v_is_k=False):
    """x [n_tok][heads][hd]; writes the cache, returns q [n_tok][q_heads][hd] (NaN where nothing is written)."""
    x = np.asarray(x, np.float64)
    q = np.full((x.shape[0], q_heads, cache.hd), np.nan)
    g = cache.kvh
    for i, at, p0, m in spans(q_len, kv_len):
        for j in range(m):
            pos, row = p0 + j, x[at + j]
            if pos < 0:
                continue
            norm = lambda y, w: y if w is None else rms(y, eps) * w.astype(np.float64)  # noqa: E731
            q[at + j] = rotate(norm(row[:q_heads], q_norm), pos, inv_freq)
            k = row[q_heads:q_heads + g]
            v = k if v_is_k else row[q_heads + g:q_heads + 2 * g]
            cache.put("k", i, pos, rotate(norm(k, k_norm), pos, inv_freq))
            cache.put("v", i, pos, rms(v, eps) if v_rms else v)
    return q


def attend(cache, q_len, kv_len, q, q_heads, scale, window, sinks):
    """-> (out [n_tok][q_heads][hd], bound [same]): the result and how far a
    correct kernel may be from it.

    bound: the f16 result's half step 2^-11 |out|, the weights' rounding to
    f16 2^-11 sum p |v|, their f16 subnormals' 2^-25 max |v| a key, and twice
    the weights' relative error e sum p |v| from the scores' error e: f32 sums
    of hd products (hd 2^-24 sum |q k|), queries as two f16 (2^-22 sum |q k|),
    scale, maximum and exp2 argument in f32 (8 roundings of a score's size)."""
    q = np.asarray(q, np.float64)
    out, bound = np.zeros_like(q), np.zeros_like(q)
    g = q_heads // cache.kvh
    for i, at, p0, m in spans(q_len, kv_len):
        rows = {n: [cache.get(n, i, p) for p in range(max(p0 + m, 0))] for n in "kv"}
        have = np.array([r is not None for r in rows["k"]], bool)
        if not len(have):
            continue
        zero = np.zeros((cache.kvh, cache.hd))
        K = np.stack([zero if r is None else r for r in rows["k"]])
        V = np.stack([zero if r is None else r for r in rows["v"]])
        p = np.arange(len(have))
        for j in range(m):
            pos = p0 + j
            sees = have & (p <= pos)
            if window:
                sees &= (p > pos - window) | (p < sinks)
            if not sees.any():
                continue
            for h in range(q_heads):
                k, v, x = K[sees, h // g], V[sees, h // g], q[at + j, h]
                s = (k @ x) * scale
                w = np.exp(s - s.max())
                w /= w.sum()
                o = w @ v
                mag = (np.abs(k) @ np.abs(x)) * abs(scale)
                e = (cache.hd * 2.0**-24 + 2.0**-22) * mag.max() + 8 * 2.0**-24 * np.abs(s).max()
                out[at + j, h] = o
                av = w @ np.abs(v)
                bound[at + j, h] = 2.0**-11 * np.abs(o) + (2.0**-11 + 2 * e) * av + \
                    len(s) * 2.0**-25 * np.abs(v).max() + 2.0**-25
    return out, bound
