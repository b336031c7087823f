"""The paged key/value cache on the GPU against its definitions in 64 bits
(paged_ref.py): append, read-back, attention and the three together.

Every pool starts out as NaN (4 bits: NaN scales), so whatever a kernel reads
of rows that no query sees shows up; outputs start out as a mark, so whatever
it writes that is not its own shows up too.

Tolerances.  Appended f16 rows: the rounding's half step, 2^-11 of the value
(2^-25 below the normal range), and 2^-19 of the row's largest value for the
f32 norm and rotation (sum of squares, root and quotient, weight, sine and
cosine, two products and a sum: 16 roundings of 2^-24 are 2^-20; doubled for
the sine's own error); f32 queries the 2^-19 alone.  4-bit rows: the bytes of
the reference.  Attention: the bound that paged_ref.attend derives."""
import ctypes as C

import numpy as np
import pytest

from e4b import _lib
from e4b._lib import DT_F16, DT_F32, E4BError, lib
from e4b.device import DeviceBuffer
from e4b.kernels import HeadPrep, KvBatch, PagedKV, rope_inv_freq
from tests import paged_ref as ref

pytestmark = pytest.mark.gpu

EPS = 1e-6
MARK = 0x7BCD  # an f16 of 63,900: no result here is near it


class Rig:
    """A cache on the host and its copy on the device."""

    def __init__(self, kind, hd, kvh, page, n_seq, kv_max, extra_pages=3, n_pages=None):
        stride = kv_max // page + 2
        self.n_pages = n_pages or n_seq * (kv_max // page + 1) + extra_pages
        self.host = ref.Cache(kind, kvh, hd, page, self.n_pages, n_seq, stride)
        self.dev = PagedKV(kind, kvh, hd, page, self.n_pages, stride, n_seq=n_seq)
        assert self.dev.page_bytes * self.n_pages == self.host.bytes("k").nbytes

    def push(self):
        self.dev.k.upload(self.host.bytes("k"))
        self.dev.v.upload(self.host.bytes("v"))
        self.dev.table.upload(self.host.table)

    def pulled(self, n):
        return (self.dev.k if n == "k" else self.dev.v).download(np.uint8)


def rows_buffer(rows, cols, dtype, pad=0):
    """Marked rows with `pad` more elements between them."""
    a = np.full((rows, cols + pad), MARK, np.uint16) if dtype == np.float16 else \
        np.full((rows, cols + pad), -12345.0, np.float32)
    return DeviceBuffer.from_array(a), a


def run_attn(rig, q_len, kv_len, q, q_heads, qt, window=0, sinks=0, scale=1.0, pad=0, extra_tok=2, stream=None,
             own_ws=False):
    """-> out f16 [n_tok][q_heads][hd]; checks that padding and the tokens behind the batch keep their marks"""
    hd, n = rig.host.hd, sum(q_len)
    dt = np.float16 if qt == DT_F16 else np.float32
    qa = np.full((n + extra_tok, q_heads * hd + pad), np.nan, dt)
    qa[:n, :q_heads * hd] = q.reshape(n, -1)
    qd = DeviceBuffer.from_array(qa)
    od, marks = rows_buffer(n + extra_tok, q_heads * hd, np.float16, pad)
    b = KvBatch.from_lengths(q_len, kv_len, n + extra_tok)
    ws = DeviceBuffer(max(1, rig.dev.attn_ws_bytes(b, qt, q_heads, window, sinks))) if own_ws else None
    rig.dev.attn_dev(b, qd, qt, q_heads, od, window, sinks, scale, q_heads * hd + pad, q_heads * hd + pad, ws,
                     ws.nbytes if ws else 0, stream)
    if stream:
        _lib.check(lib.e4b_stream_sync(stream), "e4b_stream_sync")
    got = od.download(np.uint16).reshape(marks.shape)
    np.testing.assert_array_equal(got[n:], marks[n:])
    np.testing.assert_array_equal(got[:, q_heads * hd:], marks[:, q_heads * hd:])
    return np.ascontiguousarray(got[:n, :q_heads * hd]).view(np.float16).reshape(n, q_heads, hd)


def check_attn(rig, q_len, kv_len, q, q_heads, qt, window=0, sinks=0, scale=1.0, **kw):
    got = run_attn(rig, q_len, kv_len, q, q_heads, qt, window, sinks, scale, **kw).astype(np.float64)
    want, bound = ref.attend(rig.host, q_len, kv_len, q, q_heads, scale, window, sinks)
    assert np.isfinite(got).all()
    off = np.abs(got - want)
    worst = float((off / np.maximum(bound, 1e-30)).max(initial=0))
    print(f"worst error / bound {worst:.3f}", flush=True)
    assert worst <= 1
    return got


def queries(rng, n, q_heads, hd, qt):
    return rng.standard_normal((n, q_heads, hd)).astype(np.float16 if qt == DT_F16 else np.float32)


# (q_len, kv_len, window, sinks)
LENGTHS = {
    "one_token": ([1], [1], 0, 0),
    "decode": ([1] * 6, [1, 2, 31, 33, 64, 300], 0, 0),
    "decode_window": ([1] * 5, [1, 40, 48, 49, 331], 48, 5),
    "empty_ones": ([1, 0, 1, 0, 1], [5, 7, 1, 0, 33], 0, 0),
    "nothing_seen": ([2, 1, 3], [0, 0, 1], 0, 0),
    "more_new_than_kept": ([4, 1], [2, 9], 4, 1),
    "chunks": ([3, 1, 40, 0, 17], [3, 129, 40, 9, 200], 0, 0),
    "chunks_window": ([33, 2, 70], [90, 200, 70], 20, 3),
    "window_1": ([5, 1], [77, 40], 1, 0),
    "window_1_sink": ([5, 1], [77, 40], 1, 1),
    "sinks_past_all": ([7, 1], [50, 20], 8, 1000),
    "window_past_all": ([7, 1], [50, 20], 1000, 2),
    "sinks_meet_window": ([9], [100], 40, 60),
    "sinks_mid_tile": ([1, 9], [500, 420], 33, 37),
}
SHAPES = [("f16", 256, 2, 4, 16), ("q4", 256, 2, 4, 16), ("f16", 512, 1, 8, 32), ("q4", 512, 2, 2, 64),
          ("f16", 128, 3, 3, 128), ("q4", 128, 1, 1, 256)]


@pytest.mark.parametrize("shape", SHAPES, ids=lambda s: "%s-%d-%dx%d-p%d" % s)
@pytest.mark.parametrize("lens", list(LENGTHS))
@pytest.mark.parametrize("qt", [DT_F32, DT_F16], ids=["q32", "q16"])
def test_attention(shape, lens, qt):
    kind, hd, kvh, g, page = shape
    q_len, kv_len, window, sinks = LENGTHS[lens]
    print(shape, lens, qt, flush=True)
    rng = np.random.default_rng(hd + page + len(q_len))
    rig = Rig(kind, hd, kvh, page, len(q_len), max(kv_len))
    rig.host.fill(rng, kv_len)
    rig.push()
    q = queries(rng, sum(q_len), kvh * g, hd, qt)
    check_attn(rig, q_len, kv_len, q, kvh * g, qt, window, sinks, scale=1.0 if qt == DT_F32 else hd**-0.5)


@pytest.mark.parametrize("kind", ["f16", "q4"])
@pytest.mark.parametrize("hd,kvh,g", [(256, 2, 4), (512, 1, 8), (128, 1, 16), (256, 1, 6), (128, 2, 20)])
@pytest.mark.parametrize("q_len,kv,window,sinks", [(1, 2500, 0, 0), (1, 2500, 700, 4), (2, 1777, 0, 0), (130, 700, 0, 0),
                                                   (130, 700, 100, 9), (37, 1500, 0, 0)])
def test_attention_over_long_ones(kind, hd, kvh, g, q_len, kv, window, sinks):
    print(kind, hd, kvh, g, q_len, kv, flush=True)
    rng = np.random.default_rng(kv + q_len)
    rig = Rig(kind, hd, kvh, 64, 1, kv)
    rig.host.fill(rng, [kv])
    rig.push()
    qt = DT_F16 if q_len & 1 else DT_F32
    check_attn(rig, [q_len], [kv], queries(rng, q_len, kvh * g, hd, qt), kvh * g, qt, window, sinks)


@pytest.mark.parametrize("qt", [DT_F32, DT_F16], ids=["q32", "q16"])
@pytest.mark.parametrize("kind", ["f16", "q4"])
def test_attention_of_a_mixed_batch(kind, qt):
    # decoded tokens beside chunks, one long sequence among short ones, rows with gaps between them
    q_len, kv_len = [1, 50, 1, 0, 1, 7, 1], [1900, 80, 12, 30, 64, 411, 1]
    rng = np.random.default_rng(11)
    rig = Rig(kind, 256, 2, 32, len(q_len), max(kv_len))
    rig.host.fill(rng, kv_len)
    rig.push()
    check_attn(rig, q_len, kv_len, queries(rng, sum(q_len), 8, 256, qt), 8, qt, pad=24, extra_tok=70)
    check_attn(rig, q_len, kv_len, queries(rng, sum(q_len), 8, 256, qt), 8, qt, 100, 4, pad=8, extra_tok=0)


@pytest.mark.parametrize("n_seq", [64, 65, 200])
def test_attention_of_many_sequences(n_seq):
    rng = np.random.default_rng(n_seq)
    kv_len = rng.integers(0, 40, n_seq)
    q_len = np.minimum(rng.integers(0, 4, n_seq), kv_len)
    rig = Rig("f16", 128, 1, 16, n_seq, 40)
    rig.host.fill(rng, kv_len)
    rig.push()
    check_attn(rig, list(q_len), list(kv_len), queries(rng, int(q_len.sum()), 2, 128, DT_F32), 2, DT_F32)
    x = rng.standard_normal((int(q_len.sum()), 4, 128)).astype(np.float32)
    check_append(rig, list(q_len), list(kv_len), x, 2, None, None, np.zeros(0, np.float32), DT_F32)


@pytest.mark.parametrize("kind", ["f16", "q4"])
@pytest.mark.parametrize("q_len", [1, 21])
def test_pages_that_are_missing(kind, q_len):
    # entries that name no page: freed ones, ones past the pool, the last one; a window that needs none of them
    rng = np.random.default_rng(5)
    rig = Rig(kind, 256, 2, 16, 1, 400)
    rig.host.fill(rng, [400])
    whole = rig.host.table.copy()
    q = queries(rng, q_len, 8, 256, DT_F32)
    for gone, window, sinks in (([3, 4, 9], 0, 0), ([0, 24], 0, 0), (list(range(25)), 0, 0),
                                (list(range(1, 20)), 60, 16), (list(range(20)), 60, 16)):
        rig.host.table = whole.copy()
        rig.host.table[0, gone] = [ref.NONE, rig.n_pages, 0x80000000][len(gone) % 3]
        rig.push()
        check_attn(rig, [q_len], [400], q, 8, DT_F32, window, sinks)


@pytest.mark.parametrize("kind", ["f16", "q4"])
@pytest.mark.parametrize("q_len", [1, 30])
def test_a_table_that_ends_before_the_sequence(kind, q_len):
    rng = np.random.default_rng(6)
    rig = Rig(kind, 128, 1, 16, 2, 64)
    rig.host.fill(rng, [64, 60])  # every row of the first one's pages
    rig.push()
    kv_len = [rig.host.stride * 16 + 37, 50]  # positions past the table's end have no row
    check_attn(rig, [q_len, 1], kv_len, queries(rng, q_len + 1, 2, 128, DT_F16), 2, DT_F16)


@pytest.mark.parametrize("bad", [np.inf, -np.inf, np.nan])
@pytest.mark.parametrize("q_len", [1, 3, 60])
@pytest.mark.parametrize("kind", ["f16", "q4"])
def test_values_that_are_not_finite_where_they_are_masked(kind, q_len, bad):
    # rows 90 (behind the window), 61 and 99 (seen by some of the chunk's tokens alone) are not finite: who does not
    # see them is as exact as ever, who does gets no finite result
    kv, window, sinks = 100, 12, 2
    rng = np.random.default_rng(8)
    rig = Rig(kind, 256, 1, 32, 1, kv)
    rig.host.fill(rng, [kv])
    rows = [20, 61, 99] if q_len > 1 else [20, 87]
    for n, p in zip("kvv", rows):
        x = rig.host.get(n, 0, p)
        x[:, 40] = bad
        rig.host.put(n, 0, p, x)
    rig.push()
    q = queries(rng, q_len, 4, 256, DT_F16)
    got = run_attn(rig, [q_len], [kv], q, 4, DT_F16, window, sinks, 0.1).astype(np.float64)
    pos = kv - q_len + np.arange(q_len)
    sees = np.zeros(q_len, bool)
    for p in rows:
        sees |= (p <= pos) & ((p > pos - window) | (p < sinks))
    for n, p in zip("kvv", rows):  # the reference without them
        rig.host.put(n, 0, p, np.zeros((1, 256)))
    want, bound = ref.attend(rig.host, [q_len], [kv], q, 4, 0.1, window, sinks)
    clear = ~sees
    assert clear.any()
    assert np.all(np.abs(got - want)[clear] <= bound[clear])
    if q_len > 1:
        assert sees.any()
        for t in np.flatnonzero(sees):  # the dim (4 bits: its block) that holds the value
            assert not np.isfinite(got[t, :, 40]).any(), t


def test_infinite_scores_of_masked_keys_and_large_ones():
    # scores of some thousands, the largest one first, last and in the middle
    rng = np.random.default_rng(9)
    rig = Rig("f16", 128, 1, 16, 1, 200)
    rig.host.fill(rng, [200], k_std=30.0)
    rig.push()
    for q_len in (1, 40):
        check_attn(rig, [q_len], [200], queries(rng, q_len, 4, 128, DT_F16), 4, DT_F16)
        check_attn(rig, [q_len], [200], queries(rng, q_len, 4, 128, DT_F16), 4, DT_F16, scale=0.0)
        check_attn(rig, [q_len], [200], queries(rng, q_len, 4, 128, DT_F16), 4, DT_F16, scale=-0.02)


def test_rows_past_four_gib():
    # a pool of more than 2^32 bytes whose first and last pages are in use
    hd, kvh, page = 512, 8, 256
    pb = 2 * hd * kvh * page
    n_pages = (1 << 32) // pb + 40
    rng = np.random.default_rng(10)
    small = ref.Cache("f16", kvh, hd, page, 2, 1, 3)
    small.fill(rng, [300])
    dev = PagedKV("f16", kvh, hd, page, n_pages, 3, n_seq=1)
    table = np.array([n_pages - 1, 0, ref.NONE], np.uint32)
    dev.table.upload(table)
    for n, buf in (("k", dev.k), ("v", dev.v)):
        raw = small.bytes(n).reshape(2, -1)
        for b in range(2):
            buf.upload(raw[small.table[0, b]], int(table[b]) * pb)
    for q_len in (1, 20):
        q = queries(rng, q_len, 8, hd, DT_F32)
        qd, od = DeviceBuffer.from_array(q), DeviceBuffer(q.size * 2)
        batch = KvBatch.from_lengths([q_len], [300])
        dev.attn_dev(batch, qd, DT_F32, 8, od)
        want, bound = ref.attend(small, [q_len], [300], q, 8, 1.0, 0, 0)
        assert np.all(np.abs(od.download(np.float16).reshape(q.shape).astype(np.float64) - want) <= bound)
    ko, vo = DeviceBuffer(300 * kvh * hd * 2), DeviceBuffer(300 * kvh * hd * 2)
    dev.gather_dev(KvBatch.from_lengths([300], [300]), ko, vo)
    for n, buf in (("k", ko), ("v", vo)):
        want = np.stack([small.get(n, 0, p) for p in range(300)]).astype(np.float16)
        np.testing.assert_array_equal(buf.download(np.uint16), want.view(np.uint16).reshape(-1))


# ---- append and read-back ------------------------------------------------------------------------------------------

def check_append(rig, q_len, kv_len, x, q_heads, qw, kw, inv, qt, v_rms=True, v_is_k=False, pad=0, extra_tok=3,
                 in_place=False):
    hd, kvh, n = rig.host.hd, rig.host.kvh, sum(q_len)
    heads = x.shape[1]
    xa = np.full((n + extra_tok, heads * hd + pad), 3.0, x.dtype)
    xa[:n, :heads * hd] = x.reshape(n, -1)
    xd = DeviceBuffer.from_array(xa)
    dt = np.float16 if qt == DT_F16 else np.float32
    xt = DT_F16 if x.dtype == np.float16 else DT_F32
    if in_place:
        qd, marks, width = xd, xa.copy(), heads * hd + pad
    else:
        qd, marks = rows_buffer(n + extra_tok, q_heads * hd, dt, pad)
        width = q_heads * hd + pad
    dev = [None if w is None else DeviceBuffer.from_array(w) for w in (qw, kw)]
    prep = HeadPrep(dev[0], dev[1], DeviceBuffer.from_array(inv) if len(inv) else None, len(inv), EPS, v_rms, v_is_k)
    rig.dev.append_dev(KvBatch.from_lengths(q_len, kv_len, n + extra_tok), prep, xd, xt, q_heads, qd, qt,
                       heads * hd + pad, width)
    want_q = ref.append(rig.host, q_len, kv_len, x, q_heads, qw, kw, inv, EPS, v_rms, v_is_k)
    got_q = qd.download(np.uint16 if dt == np.float16 else np.float32).reshape(marks.shape)
    same = np.uint16 if marks.dtype == np.float16 else marks.dtype
    written = ~np.isnan(want_q[:, 0, 0]) if q_heads else np.zeros(n, bool)
    marks = marks.view(same)
    np.testing.assert_array_equal(got_q[n:], marks[n:])
    np.testing.assert_array_equal(got_q[:, q_heads * hd:], marks[:, q_heads * hd:])
    np.testing.assert_array_equal(got_q[:n][~written], marks[:n][~written])
    got = got_q[:n][written][:, :q_heads * hd].copy().view(dt).astype(np.float64).reshape(-1, q_heads, hd)
    want = want_q[written]
    half = 2.0**-11 * np.abs(want) + 2.0**-25 if qt == DT_F16 else 0.0
    if want.size:
        assert np.all(np.abs(got - want) <= half + 2.0**-19 * np.abs(want).max(-1, keepdims=True))
    for name in "kv":
        raw, expect = rig.pulled(name), rig.host.bytes(name)
        if rig.host.kind == "q4":
            np.testing.assert_array_equal(raw, expect)
        else:
            a, b = raw.view(np.float16).astype(np.float64), expect.view(np.float16).astype(np.float64)
            np.testing.assert_array_equal(np.isnan(a), np.isnan(b))
            top = np.abs(np.nan_to_num(b)).reshape(-1, hd).max(-1, keepdims=True)
            d = np.abs(np.nan_to_num(a) - np.nan_to_num(b)).reshape(-1, hd)
            # both sides round: two half steps where they fall on either side of a border
            assert np.all(d <= 2.0**-10 * np.abs(np.nan_to_num(b)).reshape(-1, hd) + 2.0**-24 + 2.0**-19 * top)
            rig.host.set_bytes(name, raw)
    return prep


@pytest.mark.parametrize("kind", ["f16", "q4"])
@pytest.mark.parametrize("hd,angles", [(128, 64), (256, 128), (512, 64), (256, 37), (256, 0)])
@pytest.mark.parametrize("xt", [np.float32, np.float16], ids=["x32", "x16"])
def test_append(kind, hd, angles, xt):
    print(kind, hd, angles, xt, flush=True)
    rng = np.random.default_rng(hd + angles)
    q_len, kv_len = [1, 20, 0, 5, 1], [1, 70, 12, 5, 33]
    rig = Rig(kind, hd, 2, 16, 5, 80)
    rig.host.fill(rng, np.array(kv_len) - q_len)
    for i, n in enumerate(kv_len):  # pages for the new rows
        for b in range(-(-n // 16)):
            if rig.host.table[i, b] == ref.NONE:
                rig.host.table[i, b] = next(p for p in range(rig.n_pages) if p not in rig.host.table)
    rig.push()
    x = rng.standard_normal((sum(q_len), 8 + 4, hd)).astype(xt)
    qw, kw = ((1 + 0.1 * rng.standard_normal((2, hd))) * [[1], [0.25]]).astype(np.float32)
    inv = rope_inv_freq(1e4, hd, angles)
    check_append(rig, q_len, kv_len, x, 8, qw, kw, inv, DT_F16 if hd == 256 else DT_F32)
    # without norms, into the same rows again; then with v = k; in place
    check_append(rig, q_len, kv_len, x, 8, None, None, inv, DT_F32, v_rms=False, pad=16)
    check_append(rig, q_len, kv_len, x[:, :10], 8, qw, kw, inv, DT_F16, v_is_k=True, extra_tok=0)
    check_append(rig, q_len, kv_len, x, 8, qw, kw, inv, DT_F16 if xt == np.float16 else DT_F32, in_place=True)


@pytest.mark.parametrize("kind", ["f16", "q4"])
def test_append_where_there_is_no_page(kind):
    # positions before the sequence, past the table, and on entries that name no page write nothing
    rng = np.random.default_rng(3)
    q_len, kv_len = [6, 40, 30], [3, 200, 64]
    rig = Rig(kind, 256, 1, 16, 3, 64)
    rig.host.table[0, 0] = 2
    rig.host.table[1, :4] = [5, ref.NONE, rig.n_pages, 0x7FFFFFFF]
    rig.host.table[2, :4] = [7, 8, 0xFFFFFFFE, 9]
    rig.push()
    x = rng.standard_normal((sum(q_len), 4, 256)).astype(np.float32)
    check_append(rig, q_len, kv_len, x, 2, None, None, rope_inv_freq(1e6, 256, 128), DT_F32)
    ko, marks = rows_buffer(sum(q_len) + 1, 256, np.float16)
    rig.dev.gather_dev(KvBatch.from_lengths(q_len, kv_len, sum(q_len) + 1), ko, None)
    got = ko.download(np.uint16).reshape(marks.shape)
    np.testing.assert_array_equal(got[-1], marks[-1])
    for i, at, p0, m in ref.spans(q_len, kv_len):
        for j in range(m):
            r = rig.host.get("k", i, p0 + j)
            want = np.zeros(256, np.float16) if r is None else r.astype(np.float16).reshape(-1)
            np.testing.assert_array_equal(got[at + j].view(np.float16), want)


@pytest.mark.parametrize("far", [4095, 32767, 1 << 20, (1 << 30) + 12345])
def test_append_at_far_positions(far):
    # one page whose entry is the last of a long table; angles of far positions are exact
    page = 256
    b = far // page
    rng = np.random.default_rng(4)
    dev = PagedKV("f16", 1, 256, page, 1, b + 1, n_seq=1)
    table = np.full(b + 1, ref.NONE, np.uint32)
    table[b] = 0
    dev.table.upload(table)
    x = rng.standard_normal((1, 3, 256)).astype(np.float32)
    inv = rope_inv_freq(1e4, 256, 128)
    xd, qd, iv = DeviceBuffer.from_array(x), DeviceBuffer(1024), DeviceBuffer.from_array(inv)
    dev.append_dev(KvBatch.from_lengths([1], [far + 1]), HeadPrep(None, None, iv, 128, EPS), xd, DT_F32, 1, qd)
    want = ref.rotate(x[0, :1].astype(np.float64), far, inv)
    got = qd.download(np.float32).astype(np.float64)
    assert np.all(np.abs(got - want[0]) <= 2.0**-19 * np.abs(want).max())


@pytest.mark.parametrize("kind", ["f16", "q4"])
def test_append_of_special_values(kind):
    # zeros, ties of the largest magnitude, tiny, huge and not finite values
    hd = 128
    x = np.zeros((7, 2, hd), np.float32)
    x[0, :, 3], x[0, :, 5] = 2.0, -2.0          # the first of two largest, of either sign
    x[1, :, 3], x[1, :, 5] = -2.0, 2.0
    x[2, :, 7] = 1e-7                           # below a step of the scale's type
    x[3, :, :32] = np.linspace(-1e5, 9e4, 32)   # past what f16 holds
    x[4, :, 33], x[4, :, 70] = np.inf, np.nan
    x[5, :, ::2] = 2.0**-20
    x[6] = np.random.default_rng(1).integers(-8, 9, (2, hd)) * 0.5  # quotients halfway between two codes
    rig = Rig(kind, hd, 1, 16, 1, 16)
    rig.host.table[0, 0] = 1
    rig.push()
    with np.errstate(all="ignore"):
        check = ref.append(rig.host, [7], [7], x, 0, None, None, np.zeros(0), EPS, v_rms=False)
    assert check.shape == (7, 0, hd)
    xd = DeviceBuffer.from_array(x)
    rig.dev.append_dev(KvBatch.from_lengths([7], [7]), HeadPrep(None, None, None, 0, EPS, v_rms=False), xd, DT_F32, 0)
    for n in "kv":
        got, want = rig.pulled(n), rig.host.bytes(n)
        if kind == "f16":
            got, want = got.view(np.float16), want.view(np.float16)
            np.testing.assert_array_equal(got, want)
            continue
        cut = 16 * hd // 2
        got, want = got.reshape(rig.n_pages, -1), want.reshape(rig.n_pages, -1)
        np.testing.assert_array_equal(got[:, cut:].copy().view(np.float16), want[:, cut:].copy().view(np.float16))
        np.testing.assert_array_equal(got[:, :cut], want[:, :cut])


def test_read_back_of_whole_sequences():
    rng = np.random.default_rng(13)
    for kind, hd in (("f16", 256), ("q4", 128), ("q4", 256), ("q4", 512)):
        rig = Rig(kind, hd, 2, 32, 3, 90)
        kv_len = [90, 1, 33]
        rig.host.fill(rng, kv_len)
        rig.push()
        k, v = (DeviceBuffer(sum(kv_len) * 2 * hd * 2) for _ in "kv")
        rig.dev.gather_dev(KvBatch.from_lengths(kv_len, kv_len), k, v)
        for n, buf in (("k", k), ("v", v)):
            want = np.stack([rig.host.get(n, i, p) for i in range(3) for p in range(kv_len[i])]).astype(np.float16)
            np.testing.assert_array_equal(buf.download(np.float16), want.reshape(-1))


# ---- together ------------------------------------------------------------------------------------------------------

@pytest.mark.parametrize("kind", ["f16", "q4"])
def test_prompts_and_decoded_tokens_through_one_cache(kind):
    """Two prompts of unlike lengths in chunks, then tokens, each step append
    and attention; pages are handed out as they are needed and the ones behind
    the window are given back and used again."""
    hd, kvh, qh, page, window, sinks = 256, 2, 8, 16, 40, 4
    rng = np.random.default_rng(21)
    rig = Rig(kind, hd, kvh, page, 2, 400, n_pages=14)
    rig.push()
    qw, kw = ((1 + 0.1 * rng.standard_normal((2, hd))) * [[1], [0.25]]).astype(np.float32)
    inv = rope_inv_freq(1e4, hd, 128)
    free, kv = list(range(14)), [0, 0]
    for q_len in [(30, 7), (0, 21), (33, 1), (1, 1), (1, 0), (1, 1), (16, 1), (1, 1), (1, 1)]:
        for i, m in enumerate(q_len):
            for b in range(kv[i] // page, -(-(kv[i] + m) // page)):
                if rig.host.table[i, b] == ref.NONE:
                    rig.host.table[i, b] = free.pop()
            kv[i] += m
        rig.dev.table.upload(rig.host.table)
        n = sum(q_len)
        x = rng.standard_normal((n, qh + 2 * kvh, hd)).astype(np.float32)
        xd, qd, od = DeviceBuffer.from_array(x), DeviceBuffer(n * qh * hd * 4), DeviceBuffer(n * qh * hd * 2)
        b = KvBatch.from_lengths(q_len, kv)
        ws = [DeviceBuffer.from_array(a) for a in (qw, kw, inv)]
        rig.dev.append_dev(b, HeadPrep(ws[0], ws[1], ws[2], 128, EPS), xd, DT_F32, qh, qd)
        rig.dev.attn_dev(b, qd, DT_F32, qh, od, window, sinks)
        ref.append(rig.host, q_len, kv, x, qh, qw, kw, inv, EPS)
        q = qd.download(np.float32).reshape(n, qh, hd)
        for name in "kv":  # what the cache holds, bit for bit (4 bits), or as the append's own test says
            if kind == "q4":
                np.testing.assert_array_equal(rig.pulled(name), rig.host.bytes(name))
            rig.host.set_bytes(name, rig.pulled(name))
        want, bound = ref.attend(rig.host, q_len, kv, q, qh, 1.0, window, sinks)
        got = od.download(np.float16).reshape(n, qh, hd).astype(np.float64)
        assert np.all(np.abs(got - want) <= bound), q_len
        for i in range(2):  # give back what no later token sees
            for blk in range(1, max(0, (kv[i] - window) // page)):
                if rig.host.table[i, blk] != ref.NONE:
                    free.append(int(rig.host.table[i, blk]))
                    rig.host.table[i, blk] = ref.NONE


def test_the_same_call_gives_the_same_bits():
    rng = np.random.default_rng(30)
    rig = Rig("q4", 256, 2, 64, 3, 3000)
    kv_len = [3000, 200, 900]
    rig.host.fill(rng, kv_len)
    rig.push()
    for q_len in ([1, 1, 1], [40, 9, 1]):
        q = queries(rng, sum(q_len), 8, 256, DT_F32)
        a, b = (run_attn(rig, q_len, kv_len, q, 8, DT_F32) for _ in range(2))
        np.testing.assert_array_equal(a.view(np.uint16), b.view(np.uint16))
        c = run_attn(rig, q_len, kv_len, q, 8, DT_F32, own_ws=True)
        np.testing.assert_array_equal(a.view(np.uint16), c.view(np.uint16))
