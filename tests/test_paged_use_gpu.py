"""The paged cache as programs use it: calls captured into graphs and replayed
with other lengths, pages and tokens, on several streams, with batches at the
bounds that they name.

A replay and an eager call of the same batch bounds make the same launches, so
what they leave is compared bit for bit; against the definitions in 64 bits
with the bounds that paged_ref.attend derives."""
import ctypes as C
import os
import subprocess
import sys

import numpy as np
import pytest

from e4b import _lib
from e4b._lib import DT_F16, DT_F32, lib
from e4b.device import DeviceBuffer
from e4b.kernels import HeadPrep, KvBatch, PagedKV, rope_inv_freq
from tests import paged_ref as ref
from tests.test_paged_gpu import MARK, Rig, check_attn, queries
from tests.test_zz_no_alloc import _hip, _ok

pytestmark = pytest.mark.gpu

EPS = 1e-6


class Graph:
    """`calls(stream)` captured on a stream of its own."""

    def __init__(self, calls):
        self.hip, self.st, self.g, self.ge = _hip(), C.c_void_p(), C.c_void_p(), C.c_void_p()
        _ok(self.hip.hipStreamCreate(C.byref(self.st)), "hipStreamCreate")
        _ok(self.hip.hipStreamBeginCapture(self.st, 1), "hipStreamBeginCapture")
        try:
            calls(self.st)
        finally:
            _ok(self.hip.hipStreamEndCapture(self.st, C.byref(self.g)), "hipStreamEndCapture")
        _ok(self.hip.hipGraphInstantiate(C.byref(self.ge), self.g, None, None, 0), "hipGraphInstantiate")

    def replay(self, wait=True):
        _ok(self.hip.hipGraphLaunch(self.ge, self.st), "hipGraphLaunch")
        if wait:
            self.wait()

    def wait(self):
        _ok(self.hip.hipStreamSynchronize(self.st), "hipStreamSynchronize")

    def close(self):
        for f, h in ((self.hip.hipGraphExecDestroy, self.ge), (self.hip.hipGraphDestroy, self.g),
                     (self.hip.hipStreamDestroy, self.st)):
            _ok(f(h), f.__name__)


class Step:
    """Buffers of a step -- append, then attention -- over a cache of its own."""

    def __init__(self, rig, n_seq, n_tok, max_q, max_kv, q_heads, qt, window, sinks, own_ws):
        self.h, self.qh, self.qt, self.window, self.sinks, self.n_tok = rig.host, q_heads, qt, window, sinks, n_tok
        h = rig.host
        self.kv = PagedKV(h.kind, h.kvh, h.hd, h.page, h.n_pages, h.stride, n_seq=n_seq)
        self.q_start, self.kv_len = DeviceBuffer((n_seq + 1) * 4), DeviceBuffer(n_seq * 4)
        self.b = KvBatch(self.q_start, self.kv_len, n_seq, n_tok, max_q, max_kv)
        rng = np.random.default_rng(5)
        w = (1 + 0.1 * rng.standard_normal((2, h.hd))).astype(np.float32)
        self.w = [DeviceBuffer.from_array(a) for a in (w[0], 0.2 * w[1], rope_inv_freq(1e4, h.hd, h.hd // 4))]
        self.prep = HeadPrep(*self.w, h.hd // 4, EPS)
        self.x = DeviceBuffer(n_tok * (q_heads + 2 * h.kvh) * h.hd * 4)
        self.q = DeviceBuffer(n_tok * q_heads * h.hd * (2 if qt == DT_F16 else 4))
        self.out = DeviceBuffer(n_tok * q_heads * h.hd * 2)
        self.ws = DeviceBuffer(max(16, self.kv.attn_ws_bytes(self.b, qt, q_heads, window, sinks))) if own_ws else None
        self.kv.k.upload(h.bytes("k"))
        self.kv.v.upload(h.bytes("v"))

    def put(self, q_len, kv_len, x):
        self.q_start.upload(np.concatenate([[0], np.cumsum(q_len)]).astype(np.int32))
        self.kv_len.upload(np.asarray(kv_len, np.int32))
        self.kv.table.upload(self.h.table)
        self.x.upload(x)
        self.out.upload(np.full(self.out.nbytes // 2, MARK, np.uint16))

    def run(self, stream=None):
        self.kv.append_dev(self.b, self.prep, self.x, DT_F32, self.qh, self.q, self.qt, stream=stream)
        self.kv.attn_dev(self.b, self.q, self.qt, self.qh, self.out, self.window, self.sinks, 1.0, ws=self.ws,
                         ws_bytes=self.ws.nbytes if self.ws else 0, stream=stream)

    def got(self):
        return [self.out.download(np.uint16), self.kv.k.download(np.uint8), self.kv.v.download(np.uint8)]


# (the lengths of each replay: q_len, kv_len), bounds max_q and max_kv of them all
USES = {
    "decode": ([([1, 1, 1, 1, 1], [900, 40, 1, 333, 64]), ([1, 1, 1, 1, 1], [901, 41, 2, 334, 65]),
                ([1, 0, 1, 1, 0], [902, 41, 3, 335, 65]), ([0, 0, 0, 0, 1], [902, 41, 3, 335, 1300]),
                ([1, 1, 1, 1, 1], [1500, 1500, 1500, 1500, 1500])], 1, 1500),
    "prompt": ([([90], [1400]), ([17], [1417]), ([90], [90]), ([1], [5]), ([90], [1500])], 90, 1500),
    "mixed": ([([1, 40, 1, 3], [700, 40, 2, 900]), ([40, 1, 1, 1], [740, 41, 3, 901]), ([0, 0, 40, 5], [9, 9, 1000, 906]),
               ([1, 1, 1, 1], [741, 42, 1001, 907])], 40, 1001),
}


@pytest.mark.parametrize("use", list(USES))
@pytest.mark.parametrize("kind,qt,window", [("f16", DT_F32, 0), ("q4", DT_F32, 100), ("q4", DT_F16, 0), ("f16", DT_F16, 300)])
def test_a_captured_step_replays_with_other_lengths_and_pages(use, kind, qt, window):
    lens, max_q, max_kv = USES[use]
    n_seq, n_tok = len(lens[0][0]), max(sum(q) for q, _ in lens) + 1
    rng = np.random.default_rng(77)
    rig = Rig(kind, 256, 2, 32, n_seq, max_kv, extra_pages=9)
    rig.host.fill(rng, [max_kv] * n_seq)
    sides = [Step(rig, n_seq, n_tok, max_q, max_kv, 8, qt, window, 3 if window else 0, own) for own in (True, False)]
    eager = sides[1]
    eager.put(*lens[0], np.zeros((n_tok, 12, 256), np.float32))
    eager.run()  # (the library's workspace holds it from here on)
    for s in sides:
        s.kv.k.upload(rig.host.bytes("k"))
        s.kv.v.upload(rig.host.bytes("v"))
    graph = Graph(sides[0].run)
    for n, (q_len, kv_len) in enumerate(lens):
        print(f"replay {n}: {q_len} of {kv_len}", flush=True)
        rig.host.table[:, :max_kv // 32] = np.roll(rig.host.table[:, :max_kv // 32], 1, 1)  # the same pages, elsewhere
        x = rng.standard_normal((n_tok, 12, 256)).astype(np.float32)
        for s in sides:
            s.put(q_len, kv_len, x)
        graph.replay()
        eager.run()
        for a, b in zip(sides[0].got(), eager.got()):
            np.testing.assert_array_equal(a, b)
        out = eager.got()[0].reshape(n_tok, -1)
        assert (out[sum(q_len):] == MARK).all() and np.isfinite(out[:sum(q_len)].view(np.float16)).all()
        # and it is the answer: what the cache holds now, and the queries it was asked with
        for name, raw in zip("kv", eager.got()[1:]):
            rig.host.set_bytes(name, raw)
        m = sum(q_len)
        q = eager.q.download(np.float16 if qt == DT_F16 else np.float32).reshape(n_tok, 8, 256)[:m]
        want, bound = ref.attend(rig.host, q_len, kv_len, q, 8, 1.0, window, 3 if window else 0)
        off = np.abs(out[:m].view(np.float16).reshape(m, 8, 256).astype(np.float64) - want)
        assert np.all(off <= bound), float((off / bound).max())
    graph.close()


def test_steps_on_two_streams_at_once():
    """Two captured steps, each with scratch of its own, run side by side."""
    rng = np.random.default_rng(78)
    q_len, kv_len = [1, 60, 1], [2500, 1100, 300]
    rig = Rig("q4", 256, 2, 64, 3, 2500)
    rig.host.fill(rng, kv_len)
    steps = [Step(rig, 3, 62, 60, 2500, 8, DT_F32, 0, 0, True) for _ in range(2)]
    want, graphs = [], []
    for s in steps:
        s.put(q_len, kv_len, rng.standard_normal((62, 12, 256)).astype(np.float32))
        s.run()
        want.append(s.got())
        graphs.append(Graph(s.run))
    assert not np.array_equal(want[0][0], want[1][0])
    for _ in range(4):
        for s in steps:
            s.out.fill(0)
        _lib.check(lib.e4b_sync(), "e4b_sync")
        for g in graphs * 3:
            g.replay(wait=False)
        for g in graphs:
            g.wait()
        for s, w in zip(steps, want):
            for a, b in zip(s.got(), w):
                np.testing.assert_array_equal(a, b)
    for g in graphs:
        g.close()


_CHILD = r"""
import numpy as np
from e4b import _lib
from e4b._lib import DT_F32
from tests.test_paged_gpu import Rig
from tests.test_paged_use_gpu import Graph, Step
rng = np.random.default_rng(79)
rig = Rig("f16", 256, 1, 64, 1, 3000)
rig.host.fill(rng, [3000])
x = rng.standard_normal((1, 4, 256)).astype(np.float32)
lib_ws, own = (Step(rig, 1, 1, 1, 3000, 2, DT_F32, 0, 0, o) for o in (False, True))
assert own.ws.nbytes > 16
for s in (lib_ws, own):
    s.put([1], [3000], x)
try:
    Graph(lib_ws.run)
    raise SystemExit("a first call inside a capture took memory")
except _lib.E4BError as e:
    print(e, flush=True)
    assert "stream capture" in str(e)
g = Graph(own.run)
g.replay()
got = own.got()
lib_ws.run()
for a, b in zip(got, lib_ws.got()):
    np.testing.assert_array_equal(a, b)
g.close()
print("CHILD OK", flush=True)
"""


def test_the_workspace_is_refused_inside_a_capture_and_own_scratch_is_not():
    root = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
    env = dict(os.environ, PYTHONPATH=os.pathsep.join([root, os.path.join(root, "e4b-webgpu_amd"),
                                                       os.environ.get("PYTHONPATH", "")]))
    r = subprocess.run([sys.executable, "-c", _CHILD], cwd=root, env=env, capture_output=True, text=True, timeout=110)
    print(r.stdout, r.stderr[-2000:])
    assert r.returncode == 0 and "CHILD OK" in r.stdout


@pytest.mark.parametrize("kind", ["f16", "q4"])
@pytest.mark.parametrize("max_q,max_kv", [(1, 1), (1, 5000), (2, 40), (40, 1), (64, 64), (7, 100)])
def test_lengths_past_the_bounds_of_the_batch(kind, max_q, max_kv):
    """max_kv below a length: the same answers.  max_q below one: that
    sequence's tokens are right or left as they were, the others' are right."""
    rng = np.random.default_rng(80)
    q_len, kv_len = [1, 40, 0, 1, 2], [1700, 900, 4, 33, 200]
    rig = Rig(kind, 256, 2, 64, 5, 1700)
    rig.host.fill(rng, kv_len)
    rig.push()
    n, qh = sum(q_len), 8
    q = queries(rng, n, qh, 256, DT_F32)
    qd, od = DeviceBuffer.from_array(q), DeviceBuffer.from_array(np.full(n * qh * 256, MARK, np.uint16))
    start = np.concatenate([[0], np.cumsum(q_len)]).astype(np.int32)
    bufs = DeviceBuffer.from_array(start), DeviceBuffer.from_array(np.asarray(kv_len, np.int32))
    rig.dev.attn_dev(KvBatch(*bufs, 5, n, max_q, max_kv), qd, DT_F32, qh, od)
    raw = od.download(np.uint16).reshape(n, qh, 256)
    want, bound = ref.attend(rig.host, q_len, kv_len, q, qh, 1.0, 0, 0)
    off = np.abs(raw.view(np.float16).astype(np.float64) - want)
    right, left = (off <= bound).all((1, 2)), (raw == MARK).all((1, 2))
    for i, m in enumerate(q_len):
        rows = slice(start[i], start[i + 1])
        assert (right[rows] | (left[rows] if m > max_q else False)).all(), (i, m)


def test_the_most_sequences():
    """65535 sequences with one page between them, a KV head a query head."""
    rng = np.random.default_rng(81)
    n, kvh, hd = 65535, 4, 128
    rig = Rig("q4", hd, kvh, 16, 1, 16, n_pages=1)
    rig.host.fill(rng, [16])
    kv = PagedKV("q4", kvh, hd, 16, 1, 1, k=DeviceBuffer.from_array(rig.host.bytes("k")),
                 v=DeviceBuffer.from_array(rig.host.bytes("v")), table=DeviceBuffer.from_array(np.zeros(n, np.uint32)))
    kv_len = (1 + np.arange(n) % 16).astype(np.int32)
    q = queries(rng, 16 * 5, kvh, hd, DT_F16)  # the same ones again and again
    qd = DeviceBuffer.from_array(np.resize(q, (n, kvh, hd)))
    od = DeviceBuffer(n * kvh * hd * 2)
    kv.attn_dev(KvBatch.from_lengths([1] * n, kv_len), qd, DT_F16, kvh, od)
    got = od.download(np.uint16).reshape(n, kvh, hd)
    np.testing.assert_array_equal(got, np.resize(got[:80], got.shape))
    host = ref.Cache("q4", kvh, hd, 16, 1, 80, 1)
    host.codes, host.scales = rig.host.codes, rig.host.scales
    host.table[:] = 0
    want, bound = ref.attend(host, [1] * 80, kv_len[:80], q, kvh, 1.0, 0, 0)
    assert np.all(np.abs(got[:80].view(np.float16).astype(np.float64) - want) <= bound)


@pytest.mark.parametrize("kind", ["f16", "q4"])
@pytest.mark.parametrize("n_seq,kv,q", [(70, 3000, 1), (256, 2500, 1), (130, 2300, 2), (20, 4100, 4)])
def test_ragged_batches_whose_splits_are_dealt_out(kind, n_seq, kv, q):
    rng = np.random.default_rng(n_seq)
    kv_len = [int(x) for x in rng.integers(q, 300, n_seq)]
    for i in rng.integers(0, n_seq, 3):
        kv_len[i] = kv
    kv_len[0] = q
    kv_len[-1] = kv - 1
    rig = Rig(kind, 128, 1, 64, 1, 16, n_pages=3)  # (pages of every sequence but its last ones are shared)
    rig.host = ref.Cache(kind, 1, 128, 64, 50, n_seq, kv // 64 + 2)
    rig.dev = PagedKV(kind, 1, 128, 64, 50, kv // 64 + 2, n_seq=n_seq)
    base = ref.Cache(kind, 1, 128, 64, 50, 1, 50)
    base.fill(rng, [50 * 64])
    for name in ("pools", "codes", "scales"):
        if hasattr(base, name):
            setattr(rig.host, name, getattr(base, name))
    rig.host.table[:, :kv // 64 + 1] = rng.integers(0, 50, (n_seq, kv // 64 + 1))
    rig.push()
    check_attn(rig, [q] * n_seq, kv_len, queries(rng, q * n_seq, 4, 128, DT_F32), 4, DT_F32, scale=0.09)


@pytest.mark.parametrize("kind", ["f16", "q4"])
@pytest.mark.parametrize("window,sinks", [(2**31 - 1, 0), (2**31 - 1, 2**31 - 1), (3, 2**31 - 1)])
def test_the_widest_windows_with_more_new_tokens_than_kept(kind, window, sinks):
    rng = np.random.default_rng(82)
    q_len, kv_len = [4, 40, 1, 90], [1, 9, 30, 70]
    rig = Rig(kind, 128, 2, 16, 4, 80)
    rig.host.fill(rng, kv_len)
    rig.push()
    for qt in (DT_F32, DT_F16):
        check_attn(rig, q_len, kv_len, queries(rng, sum(q_len), 8, 128, qt), 8, qt, window, sinks, scale=0.09)
        check_attn(rig, q_len[:1], kv_len[:1], queries(rng, 4, 8, 128, qt), 8, qt, window, sinks, scale=0.09)


@pytest.mark.parametrize("n", [1, 63, 64, 65, 128, 4096, 4097, 9000])
def test_append_to_many_sequences(n):
    """Every token finds its sequence, with empty ones among them and tokens before the first and behind the last."""
    rng = np.random.default_rng(n)
    hd, skip, behind = 128, 3, 5
    q_len = rng.integers(0, 3, n)
    q_len[rng.integers(n)] = 6
    kv_len = (q_len + rng.integers(0, 10, n)).astype(np.int32)
    start = (skip + np.concatenate([[0], np.cumsum(q_len)])).astype(np.int32)
    n_tok = int(start[-1]) + behind
    table = rng.permutation(n).astype(np.uint32)
    kv = PagedKV("f16", 1, hd, 16, n, 1, table=DeviceBuffer.from_array(table))
    kv.k.fill(0xFF)
    kv.v.fill(0xFF)
    x = rng.standard_normal((n_tok, 2, hd)).astype(np.float32)
    b = KvBatch(DeviceBuffer.from_array(start), DeviceBuffer.from_array(kv_len), n, n_tok, 6, 16)
    kv.append_dev(b, HeadPrep(None, None, None, 0, EPS, v_rms=False), DeviceBuffer.from_array(x), DT_F32, 0)
    want = np.full((2, n, 16, hd), 0xFFFF, np.uint16)
    for i in range(n):
        for j in range(q_len[i]):
            want[:, table[i], kv_len[i] - q_len[i] + j] = x[start[i] + j].astype(np.float16).view(np.uint16)
    np.testing.assert_array_equal(kv.k.download(np.uint16).reshape(n, 16, hd), want[0])
    np.testing.assert_array_equal(kv.v.download(np.uint16).reshape(n, 16, hd), want[1])
    ko, vo = (DeviceBuffer.from_array(np.full((n_tok, hd), MARK, np.uint16)) for _ in "kv")
    kv.gather_dev(b, ko, vo)
    for j, o in enumerate((ko, vo)):
        got = o.download(np.uint16).reshape(n_tok, hd)
        assert (got[:skip] == MARK).all() and (got[n_tok - behind:] == MARK).all()
        np.testing.assert_array_equal(got[skip:n_tok - behind],
                                      x[skip:n_tok - behind, j].astype(np.float16).view(np.uint16))


@pytest.mark.parametrize("kind,hd,kvh,g", [("f16", 256, 8, 2), ("q4", 128, 16, 1), ("q4", 512, 4, 3), ("f16", 128, 256, 1),
                                           ("f16", 512, 8, 8)])
@pytest.mark.parametrize("window", [0, 70])
def test_batches_of_many_units(kind, hd, kvh, g, window):
    """More (sequence, KV head)s than two a CU, with lengths of one token to several tiles for each wave."""
    rng = np.random.default_rng(hd + kvh)
    n = 1300 // kvh
    rig = Rig(kind, hd, kvh, 32, 1, 16, n_pages=2)
    base = ref.Cache(kind, kvh, hd, 32, 12, 1, 12)
    base.fill(rng, [12 * 32])
    base.table = rng.integers(0, 12, (n, 12)).astype(np.uint32)
    base.stride = 12
    rig.host, rig.dev = base, PagedKV(kind, kvh, hd, 32, 12, 12, n_seq=n)
    rig.push()
    kv_len = rng.integers(1, 380 if n < 100 else 130, n)
    kv_len[0], kv_len[-1] = 1, 380
    check_attn(rig, [1] * n, kv_len, queries(rng, n, kvh * g, hd, DT_F32), kvh * g, DT_F32, window, 5 if window else 0,
               scale=hd**-0.5)
