"""The token-side operators together: the example that trains and serves with
them, captured into a HIP graph, and with values that are not finite."""
import ctypes as C
import os
import sys

import numpy as np
import pytest

import pywelvet
from devmem import Stream, _ok, hip
from parity import assert_bit_equal
import test_gpu_adapters as adapters
import test_gpu_embedding as embedding
from test_gpu_adapters import Case
from tokmem import DT, U, Dev, within

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module", autouse=True)
def device():
    pywelvet.init()


@pytest.fixture
def stream():
    s = Stream()
    yield s
    s.sync()
    s.close()


def test_example(capsys):
    """Sixty steps of the example bring the loss and the served answers to the
    teachers' (a simulation in f64 with unquantised weights halves the loss,
    and its last steps answer 4 in 10 rows right, from 3); the first loss is
    the formula's on the mounted weights, within the f32 sums' 1e-4."""
    sys.path.insert(0, os.path.join(os.path.dirname(os.path.abspath(__file__)), "..", "examples"))
    import distill_adapters as ex
    losses, before, after = ex.run(60, say=lambda s: None)
    assert np.isfinite(losses).all()
    assert np.mean(losses[-5:]) < 0.75 * np.mean(losses[:5])
    assert after > before

    rng, W, table, teacher = ex.make()
    student = ex.Student(W, table, rng)
    tokens, ids = rng.integers(0, ex.VOCAB, ex.ROWS), rng.integers(0, ex.TENANTS, ex.ROWS)
    index, values = ex.top(teacher, tokens, ids)
    got = student.step(tokens, ids, index, values)
    z = table[tokens].astype(np.float64) @ student.layer.export_f32().T.astype(np.float64) / ex.TEMPERATURE
    logp = z - z.max(1, keepdims=True)
    logp -= np.log(np.exp(logp).sum(1, keepdims=True))
    t = values.astype(np.float64) / ex.TEMPERATURE
    logq = t - t.max(1, keepdims=True)
    logq -= np.log(np.exp(logq).sum(1, keepdims=True))
    want = ex.TEMPERATURE ** 2 * (np.exp(logq) * (logq - np.take_along_axis(logp, index, 1))).sum() / ex.ROWS
    student.close()
    assert abs(got - want) <= 1e-4 * want


class Graph:
    """What `calls` enqueue on a stream, captured."""

    def __init__(self, stream, calls):
        h = hip()
        vp = C.c_void_p
        h.hipStreamBeginCapture.argtypes = [vp, C.c_int]
        h.hipStreamEndCapture.argtypes = [vp, C.POINTER(vp)]
        h.hipGraphInstantiate.argtypes = [C.POINTER(vp), vp, C.POINTER(vp), C.c_char_p, C.c_size_t]
        h.hipGraphLaunch.argtypes = [vp, vp]
        h.hipGraphExecDestroy.argtypes = h.hipGraphDestroy.argtypes = [vp]
        self.stream, g, x = stream, vp(), vp()
        _ok(h.hipStreamBeginCapture(stream.h, 1), "hipStreamBeginCapture")
        calls()
        _ok(h.hipStreamEndCapture(stream.h, C.byref(g)), "hipStreamEndCapture")
        _ok(h.hipGraphInstantiate(C.byref(x), g, None, None, 0), "hipGraphInstantiate")
        self.g, self.x = g.value, x.value

    def launch(self):
        _ok(hip().hipGraphLaunch(self.x, self.stream.h), "hipGraphLaunch")
        self.stream.sync()

    def close(self):
        _ok(hip().hipGraphExecDestroy(self.x), "hipGraphExecDestroy")
        _ok(hip().hipGraphDestroy(self.g), "hipGraphDestroy")


def put(dev, a):
    a = np.ascontiguousarray(a, dev.dtype)
    assert a.shape == dev.shape
    _ok(hip().hipMemcpy(dev.ptr, a.ctypes.data, a.nbytes, 1), "hipMemcpy H2D")


@pytest.mark.parametrize("n", [3, 40, 400, 2300])
def test_replayed_from_a_graph(stream, n):
    """A captured step (lookups, adapters and distillation both ways, the
    table's gradient) replayed five times on new inputs, with eager calls
    between the replays: every output the eager one, bit for bit."""
    vocab, dim, rank, count, k = 300, 68, 12, 5, 9
    rng = np.random.default_rng(n)
    c = Case("bfloat16", dim, vocab, rank, count, n, junk=False).on_device()
    table = Dev(rng.normal(0, 1, (vocab, dim)).astype(np.float32))
    store = pywelvet.Session(rng.normal(0, 1, (vocab, dim)).astype(np.float32), 1, -1, 4)
    tokens = Dev(np.zeros(n, np.int32))
    index, values = Dev(np.zeros((n, k), np.int32)), Dev(np.zeros((n, k), np.float32))
    eb, db = pywelvet.embedding_backward_bytes(vocab, dim, n), pywelvet.distill_bytes(1, n, vocab, k)
    ews, dws = Dev(np.zeros(max(eb, 16), np.uint8)), Dev(np.zeros(max(db, 16), np.uint8))
    f32 = lambda *s: Dev(np.full(s, np.nan, np.float32))  # noqa: E731
    out = dict(x=f32(n, dim), xs=f32(n, dim), y=f32(n, vocab), h=f32(n, rank), loss=f32(n), dy=f32(n, vocab),
               dx=f32(n, dim), dd=f32(count, rank, dim), du=f32(count, rank, vocab), de=f32(vocab, dim))
    p = {name: d.ptr for name, d in out.items()}

    def calls():
        on = dict(stream=stream.h)
        pywelvet.embedding_forward(1, vocab, dim, table.ptr, tokens.ptr, n, p["x"], **on)
        pywelvet.embedding_store_forward(store, tokens.ptr, n, p["xs"], **on)
        c.a.forward(p["x"], c.d["ids"].ptr, n, c.d["base"].ptr, p["y"], p["h"], **c.ws, **on)
        pywelvet.distill(1, n, vocab, p["y"], k, index.ptr, values.ptr, p["loss"], p["dy"], 2.0, ws=dws.ptr,
                         ws_bytes=db, **on)
        c.a.backward(p["x"], c.d["ids"].ptr, n, p["h"], p["dy"], p["xs"], p["dx"], p["dd"], p["du"], **c.ws, **on)
        pywelvet.embedding_backward(vocab, dim, tokens.ptr, n, p["dx"], p["de"], ws=ews.ptr, ws_bytes=eb, **on)

    def inputs():
        put(tokens, rng.integers(-1, vocab, n))
        put(c.d["ids"], rng.integers(-1, count, n))
        put(c.d["base"], rng.normal(0, 1, (n, vocab)))
        put(index, rng.integers(0, vocab, (n, k)))
        put(values, rng.normal(0, 1, (n, k)))

    inputs()
    calls()
    stream.sync()
    g = Graph(stream, calls)
    for replay in range(5):
        inputs()
        for d in out.values():
            put(d, np.full(d.shape, np.nan, np.float32))
        g.launch()
        got = {name: d.get() for name, d in out.items()}
        for d in out.values():
            put(d, np.full(d.shape, np.nan, np.float32))
        calls()
        stream.sync()
        for name, d in out.items():
            assert_bit_equal(got[name], d.get(), f"{name} of replay {replay}")
            assert np.isfinite(got[name]).all(), name
    g.close()
    store.close()


@pytest.mark.parametrize("n", [20, 300, 2400])
@pytest.mark.parametrize("rank", [1, 20])
@pytest.mark.parametrize("dtype", DT)
def test_adapters_with_values_not_finite(stream, dtype, rank, n):
    """Infinities, NaN and values near the type's end in x and dy: the same
    places come out infinite (with the sign) and NaN as in the formula, what
    does not depend on them stays within its bound."""
    c = Case(dtype, 200, 640, rank, 2, n, ranks=[rank, rank], scales=False, junk=False)
    c.ids[:] = np.arange(n) % 2
    c.x[7, 5], c.x[8, 130], c.x[11, 199] = np.inf, -np.inf, np.nan
    c.dy[6, 5], c.dy[9, 639], c.dy[13, 600] = np.inf, -np.inf, np.nan
    c.x[15, ::16], c.dy[17, ::64] = 2e38, 2e38  # their sums pass the type's end, on the way or for good
    c.on_device()
    with np.errstate(all="ignore"):
        got_y, got_h = c.forward(stream.h)
        h = np.zeros((n, rank), np.float32)
        far = np.zeros(n, bool)
        far[15] = True
        for a, rows, down, up, s in c.groups():
            x = c.x[rows].astype(np.float64)
            want = x @ down.T
            bound = (c.inn / 8 + 64) * 2 * U * (np.abs(x) @ np.abs(down).T)
            near = ~far[rows]
            within(got_h[rows][near], want[near], bound[near], "h")
            h[rows] = want.astype(np.float32)
            y = c.base[rows] + want @ up
            odd = ~np.isfinite(want).all(1) & near
            assert np.array_equal(np.isnan(got_y[rows][odd]), np.isnan(y[odd]))
            assert np.isfinite(got_y[rows][near & ~odd]).all()
        h[[7, 8, 11, 15]] = 1.0  # the backward's own values
        dx, dd, du = c.backward(stream.h, h)
        far[:] = False
        far[17] = True
        for a, rows, down, up, s in c.groups():
            near = ~far[rows]
            x, dy, hh = c.x[rows].astype(np.float64), c.dy[rows].astype(np.float64), h[rows].astype(np.float64)
            g = dy @ up.T
            want = c.dxb[rows] + g @ down
            bad = ~np.isfinite(want).all(1)
            assert bad.sum() >= 1 and np.array_equal(np.isnan(dx[rows][near]), np.isnan(want[near]))
            inf = np.isinf(want) & near[:, None]
            assert np.array_equal(dx[rows][inf], want[inf])
            assert np.isfinite(dx[rows][near & ~bad]).all()
            wu = hh.T @ dy
            clean = np.isfinite(dy).all(0) & (np.abs(dy) < 1e30).all(0)
            bu = (len(rows) + 16) * 2 * U * np.abs(hh).T @ np.abs(dy[:, clean])
            within(du[a][:, clean], wu[:, clean], bu, "dup")
            marked = ~np.isfinite(dy).all(0)
            assert np.array_equal(np.isnan(du[a][:, marked]), np.isnan(wu[:, marked]))
            hits = np.isinf(wu) & marked
            assert np.array_equal(du[a][hits], wu[hits])


# tables of more than 32 MiB: filled first where tokens name few rows, else
# their unnamed rows looked up; results stored past the caches
@pytest.mark.parametrize("vocab,dim,n,extra", [
    (9000, 1027, 200, 3), (20000, 515, 300, 0), (20000, 515, 2400, 5), (20000, 515, 6000, 0), (4200, 2052, 700, 4)])
@pytest.mark.parametrize("accumulate", [False, True])
def test_gradients_of_large_tables(stream, vocab, dim, n, extra, accumulate):
    embedding.test_gradient(stream.h, vocab, dim, n, extra, accumulate)


@pytest.mark.parametrize("dtype", DT)
@pytest.mark.parametrize("dim,extra", [(515, 0), (516, 3), (2048, 4)])
def test_lookups_of_large_results(stream, dtype, dim, extra):
    embedding.test_lookup(stream.h, dtype, 300, dim, 9_000_000 // dim + 7, extra, 2.0)


# more than 2048 rows are always sorted by their adapters; the last two shapes'
# rows pass 32 MiB
@pytest.mark.parametrize("dtype", DT)
@pytest.mark.parametrize("shape", [
    (1001, 777, 5, 4, 2100, "mixed", 0), (130, 70, 33, 7, 2300, "mixed", 2), (260, 196, 20, 9, 2200, "mixed", 4),
    (96, 1028, 100, 3, 2500, "mixed", 0), (3, 2, 4, 2, 2100, "mixed", 1), (513, 257, 16, 2, 4200, "sorted", 1),
    (64, 68, 4, 200, 4100, "mixed", 0), (600, 4100, 16, 1, 2100, "sorted", 0), (4100, 600, 33, 5, 2200, "mixed", 3)],
    ids=lambda s: "-".join(map(str, s)))
def test_many_rows_of_adapters(stream, dtype, shape):
    adapters.test_forward_and_backward(stream.h, dtype, shape)


def test_many_rows_of_adapters_elsewhere(stream):
    """Without bases, added to gradients, without adapters, with another
    tenant's NaN and in place, on sorted rows."""
    adapters.test_without_bases_scales_or_h(stream.h, 2200)
    adapters.test_accumulates(stream.h, 2300)
    adapters.test_rows_without_an_adapter(stream.h, 2400)
    adapters.test_tenants_do_not_meet(stream.h, 2500)
    c = Case("float16", 100, 84, 8, 3, 2100).on_device()
    y, h = c.forward(stream.h)
    dx, _, _ = c.backward(stream.h, h)
    yb, xb = Dev(c.base), Dev(c.dxb)
    c.a.forward(c.d["x"].ptr, c.d["ids"].ptr, c.n, yb.ptr, yb.ptr, stream=stream.h, **c.ws)
    assert_bit_equal(yb.get(), y, "y")
    c.a.backward(None, c.d["ids"].ptr, c.n, None, c.d["dy"].ptr, d_dx_base=xb.ptr, d_dx=xb.ptr, stream=stream.h, **c.ws)
    assert_bit_equal(xb.get(), dx, "dx")


@pytest.mark.parametrize("n,count", [(64, 1), (130, 1), (256, 1), (200, 2), (1300, 3)])
@pytest.mark.parametrize("rank", [3, 24, 40])
def test_long_runs_row_by_row(stream, n, count, rank):
    """Few adapters with many rows each, below the sorting's threshold."""
    adapters.test_forward_and_backward(stream.h, "bfloat16", (132, 200, rank, count, n, "mixed", 0))


@pytest.mark.parametrize("given", ["dx", "ddown", "dup"])
@pytest.mark.parametrize("n", [6, 300, 2200])
def test_one_gradient_alone(stream, n, given):
    """Each of the backward's outputs by itself; of rows that go one by one
    with the bits that it has beside the others."""
    c = Case("bfloat16", 140, 264, 12, 5, n).on_device()
    _, h = c.forward(stream.h)
    outs = dict(zip(("dx", "ddown", "dup"), c.backward(stream.h, h)))
    dh, out = Dev(h), Dev(np.full(outs[given].shape, np.nan, np.float32))
    c.a.backward(c.d["x"].ptr if given == "ddown" else None, c.d["ids"].ptr, n, dh.ptr if given == "dup" else None,
                 c.d["dy"].ptr, d_dx_base=c.d["dxb"].ptr if given == "dx" else None, stream=stream.h,
                 **{"d_" + given: out.ptr}, **c.ws)
    got = out.get()
    if n <= 2048:
        assert_bit_equal(got, outs[given], given)
    outs[given] = got
    adapters.check_backward(c, outs["dx"], outs["ddown"], outs["dup"], h)
