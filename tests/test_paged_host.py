"""Paged key/value cache: what the library answers without a GPU -- sizes, the
place of a row (missing and bad pages among them) and every refusal."""
import ctypes as C

import numpy as np
import pytest

from e4b import _lib
from e4b._lib import (DT_F16, DT_F32, E4B_EINVAL, E4B_ERANGE, E4B_OK, KV_F16, KV_Q4, HeadPrepC, KvBatchC, PagedKvC,
                      lib)
from tests import paged_ref as ref

P = 1 << 20  # an address that is aligned and never read


def cache(**over):
    d = dict(k=P, v=P, table=P, type=KV_F16, kv_heads=2, head_dim=256, page=32, n_pages=7, table_stride=5)
    d.update(over)
    return PagedKvC(**d)


def batch(**over):
    d = dict(q_start=P, kv_len=P, n_seq=2, n_tok=3, max_q=2, max_kv=40)
    d.update(over)
    return KvBatchC(**d)


def prep(**over):
    d = dict(q_norm=P, k_norm=P, inv_freq=P, rope_angles=128, eps=1e-6, flags=1)
    d.update(over)
    return HeadPrepC(**d)


def append(kv=None, b=None, pr=None, qkv=P, dtype=DT_F32, stride=12 * 256, qh=8, q=P, qt=DT_F32, qs=8 * 256):
    return lib.e4b_k_kv_append(C.byref(kv or cache()), C.byref(b or batch()), C.byref(pr or prep()), qkv, dtype,
                               stride, qh, q, qt, qs, None)


def gather(kv=None, b=None, k=P, v=P):
    return lib.e4b_k_kv_gather(C.byref(kv or cache()), C.byref(b or batch()), k, v, None)


def attn(kv=None, b=None, q=P, qt=DT_F32, qs=8 * 256, qh=8, scale=1.0, window=0, sinks=0, out=P, os=8 * 256, ws=None,
         wb=0):
    return lib.e4b_k_attn_paged(C.byref(kv or cache()), C.byref(b or batch()), q, qt, qs, qh, scale, window, sinks,
                                out, os, ws, wb, None)


@pytest.mark.parametrize("hd", [128, 256, 512])
@pytest.mark.parametrize("page", [16, 64, 256])
def test_page_bytes(hd, page):
    assert lib.e4b_kv_page_bytes(KV_F16, 3, hd, page) == 3 * page * hd * 2
    assert lib.e4b_kv_page_bytes(KV_Q4, 3, hd, page) == 3 * page * (hd // 2 + hd // 32 * 2)


@pytest.mark.parametrize("args", [(2, 2, 256, 32), (-1, 2, 256, 32), (KV_F16, 0, 256, 32), (KV_F16, 257, 256, 32),
                                  (KV_F16, 2, 64, 32), (KV_F16, 2, 192, 32), (KV_Q4, 2, 256, 8), (KV_Q4, 2, 256, 48),
                                  (KV_Q4, 2, 256, 512)])
def test_page_bytes_of_what_is_not_supported(args):
    assert lib.e4b_kv_page_bytes(*args) == 0
    assert "e4b_kv_page_bytes" in _lib.last_error()


def test_row_of_a_position():
    kv = cache(k=None, v=None, table=None)
    row = np.array([3, 0, ref.NONE, 7, 6], np.uint32)  # entry 2 names no page, entry 3 one past the pool
    at = lambda p: lib.e4b_kv_row(C.byref(kv), row.ctypes.data, p)  # noqa: E731
    c = ref.Cache("f16", 2, 256, 32, 7, 1, 5)
    c.table[0] = row
    for p in range(-3, 200):
        pg = c.page_of(0, p)
        assert at(p) == (E4B_ERANGE if pg < 0 else pg * 2 * 32 + p % 32), p
    assert at(0) == 3 * 64 and at(33) == 1 and at(64) == E4B_ERANGE and at(96) == E4B_ERANGE
    assert at(159) == 6 * 64 + 31 and at(160) == E4B_ERANGE and at(2**40) == E4B_ERANGE
    assert lib.e4b_kv_row(C.byref(kv), None, 0) == E4B_EINVAL
    assert lib.e4b_kv_row(C.byref(cache(page=24)), row.ctypes.data, 0) == E4B_EINVAL


def test_rows_past_four_gib():
    n = 200000
    kv = cache(kv_heads=8, head_dim=512, page=256, n_pages=n)
    row = np.array([n - 1], np.uint32)
    kv.table_stride = 1
    assert lib.e4b_kv_row(C.byref(kv), row.ctypes.data, 255) == (n - 1) * 8 * 256 + 255


BAD_CACHE = [dict(type=2), dict(type=-1), dict(kv_heads=0), dict(kv_heads=-2), dict(kv_heads=257), dict(head_dim=64),
             dict(head_dim=0), dict(page=0), dict(page=8), dict(page=33), dict(page=512), dict(n_pages=0),
             dict(table_stride=0), dict(k=None), dict(v=None), dict(table=None), dict(k=P + 8), dict(v=P + 2),
             dict(table=P + 2)]
BAD_BATCH = [dict(n_seq=-1), dict(n_tok=-1), dict(n_seq=65536), dict(n_tok=(1 << 24) + 1), dict(q_start=None),
             dict(kv_len=None), dict(q_start=P + 1), dict(kv_len=P + 2), dict(max_q=0), dict(max_kv=0),
             dict(max_q=-5)]


@pytest.mark.parametrize("call", [append, gather, attn], ids=["append", "gather", "attn"])
@pytest.mark.parametrize("over", BAD_CACHE + BAD_BATCH, ids=str)
def test_refusals_of_every_call(call, over):
    kv, b = (cache(**over), None) if over in BAD_CACHE else (None, batch(**over))
    assert call(kv=kv, b=b) == E4B_EINVAL
    assert "e4b_k_" in _lib.last_error()


@pytest.mark.parametrize("fn", ["e4b_k_kv_append", "e4b_k_attn_paged", "e4b_k_kv_gather"])
def test_null_descriptions(fn):
    c, b = C.byref(cache()), C.byref(batch())
    tail = {"e4b_k_kv_append": (P, 0, 12 * 256, 8, P, 0, 2048, None),
            "e4b_k_attn_paged": (P, 0, 2048, 8, 1.0, 0, 0, P, 2048, None, 0, None), "e4b_k_kv_gather": (P, P, None)}[fn]
    mid = (C.byref(prep()),) if fn == "e4b_k_kv_append" else ()
    assert getattr(lib, fn)(None, b, *mid, *tail) == E4B_EINVAL
    assert getattr(lib, fn)(c, None, *mid, *tail) == E4B_EINVAL
    if mid:
        assert lib.e4b_k_kv_append(c, b, None, *tail) == E4B_EINVAL


@pytest.mark.parametrize("over", [dict(qkv=None), dict(qkv=P + 8), dict(dtype=2), dict(dtype=-1), dict(stride=12 * 256 - 1),
                                  dict(stride=12 * 256 + 2), dict(qh=-1), dict(qh=5000), dict(q=P + 4), dict(qt=7),
                                  dict(qs=2047), dict(qs=2050), dict(qt=DT_F16, qs=2052),
                                  dict(dtype=DT_F16, stride=12 * 256 + 4), dict(pr=prep(rope_angles=-1)),
                                  dict(pr=prep(rope_angles=129)), dict(pr=prep(inv_freq=None)),
                                  dict(pr=prep(q_norm=P + 4)), dict(pr=prep(k_norm=P + 8)),
                                  dict(pr=prep(inv_freq=P + 1)), dict(pr=prep(eps=-1.0)),
                                  dict(pr=prep(eps=float("nan"))), dict(pr=prep(flags=4))], ids=lambda d: str(list(d)))
def test_refusals_of_append(over):
    assert append(**over) == E4B_EINVAL
    assert "e4b_k_kv_append" in _lib.last_error()


def test_rows_without_v_are_shorter():
    assert append(pr=prep(flags=2), stride=10 * 256 - 4) == E4B_EINVAL
    assert append(pr=prep(flags=1), stride=10 * 256) == E4B_EINVAL


@pytest.mark.parametrize("over", [dict(k=None, v=None), dict(k=P + 2), dict(v=P + 8)], ids=str)
def test_refusals_of_gather(over):
    assert gather(**over) == E4B_EINVAL


@pytest.mark.parametrize("over", [dict(q=None), dict(q=P + 8), dict(qt=2), dict(qs=2047), dict(qs=2049), dict(qh=0),
                                  dict(qh=7), dict(qh=-8), dict(scale=float("nan")), dict(scale=float("inf")),
                                  dict(window=-1), dict(sinks=-1), dict(out=None), dict(out=P + 2), dict(os=2040),
                                  dict(os=2052)], ids=str)
def test_refusals_of_attention(over):
    assert attn(**over) == E4B_EINVAL
    assert "e4b_k_attn_paged" in _lib.last_error()


@pytest.mark.parametrize("over", [dict(n_seq=0), dict(n_tok=0), dict(n_seq=0, n_tok=0, q_start=None, kv_len=None)],
                         ids=str)
def test_an_empty_batch_does_nothing(over):
    b = batch(**over)
    assert append(b=b) == E4B_OK and gather(b=b, k=None, v=None) == E4B_OK and attn(b=b, q=None, out=None) == E4B_OK


def test_ws_bytes():
    n = C.c_size_t(7)
    ask = lambda kv, b, *a: lib.e4b_attn_paged_ws_bytes(C.byref(kv), C.byref(b), *a, C.byref(n))  # noqa: E731
    assert ask(cache(), batch(n_seq=0), DT_F32, 8, 0, 0) == E4B_OK and n.value == 0
    assert ask(cache(), batch(), DT_F32, 8, 0, 0) == E4B_OK
    assert ask(cache(), batch(), DT_F32, 7, 0, 0) == E4B_EINVAL
    assert ask(cache(), batch(), 5, 8, 0, 0) == E4B_EINVAL
    assert ask(cache(type=9), batch(), DT_F32, 8, 0, 0) == E4B_EINVAL
    assert lib.e4b_attn_paged_ws_bytes(C.byref(cache()), C.byref(batch()), 0, 8, 0, 0, None) == E4B_EINVAL


def test_reference_codes():
    # the oracle's own quantiser: the largest magnitude is code 0, steps are exact in f16
    rng = np.random.default_rng(3)
    x = rng.standard_normal((40, 256))
    codes, d = ref.q4_encode(x)
    v = (codes.astype(np.float64) - 8) * np.repeat(d.astype(np.float64), 32, -1)
    assert np.array_equal(v.astype(np.float16).astype(np.float64), v)
    step = np.abs(np.repeat(d.astype(np.float64), 32, -1))
    # half a step; one at the value opposite to the largest, which would be code 16; and the step's own rounding
    assert np.all(np.abs(v - x) <= step * (1 + 8 * 2.0**-9) + 1e-12)
    assert np.mean(np.abs(v - x) <= step * 0.5 * (1 + 2.0**-4)) > 0.97
    b = x.reshape(40, 8, 32)
    assert np.all(np.take_along_axis(codes.reshape(40, 8, 32), np.abs(b).argmax(-1)[..., None], -1) == 0)


@pytest.mark.parametrize("call", [append, gather, attn], ids=["append", "gather", "attn"])
def test_batches_past_the_grids(call):
    """A grid holds fewer than 2^32 threads."""
    assert call(b=batch(n_tok=1 << 24)) == E4B_EINVAL and "2^24" in _lib.last_error()
    for n_seq, kvh in ((65535, 33), (8193, 256)):
        kw = {} if call is not attn else dict(qh=kvh, qs=kvh * 256, os=kvh * 256)
        assert call(kv=cache(kv_heads=kvh), b=batch(n_seq=n_seq), **kw) == E4B_EINVAL
        assert "2^21" in _lib.last_error()


def test_rows_past_the_grid_of_attention():
    qh = 4096
    for n_tok, rc in ((1 << 16, E4B_OK), ((1 << 16) + 1, E4B_EINVAL)):
        n = C.c_size_t(0)
        assert lib.e4b_attn_paged_ws_bytes(C.byref(cache()), C.byref(batch(n_tok=n_tok)), DT_F32, qh, 0, 0,
                                           C.byref(n)) == rc
    assert "2^28" in _lib.last_error()


def test_scratch_that_is_too_small_or_not_aligned():
    n = C.c_size_t(0)
    b = batch(n_seq=1, n_tok=1, max_q=1, max_kv=4000)
    assert lib.e4b_attn_paged_ws_bytes(C.byref(cache()), C.byref(b), DT_F32, 8, 0, 0, C.byref(n)) == E4B_OK
    assert n.value > 0
    for ws, size in ((P, n.value - 1), (P, 0), (P + 8, n.value)):
        assert attn(b=b, ws=ws, wb=size) == E4B_EINVAL
        assert "scratch" in _lib.last_error()


def test_scratch_does_not_depend_on_pointers():
    sizes = []
    for over in ({}, dict(q_start=P + 4, kv_len=P + 8)):
        bb, n = batch(n_seq=3, n_tok=900, max_q=400, max_kv=9000, **over), C.c_size_t(0)
        assert lib.e4b_attn_paged_ws_bytes(C.byref(cache()), C.byref(bb), DT_F16, 8, 0, 0, C.byref(n)) == E4B_OK
        sizes.append(n.value)
    assert sizes[0] == sizes[1]
