"""welvet_hip_int8_*: the layer against f64.  The sum is exact; pre is a
conversion, a product of two scales, an fma with an f32 bias: 4 U of
|product| + |bias|.  A row's bits must not depend on the batch it is in."""
import numpy as np
import pytest

import pywelvet
from devmem import Stream
from parity import assert_bit_equal
from rows8ref import ACT_ERR, ACTS, TINY, Rows, act, codes_of
from test_gpu_rows8 import HALF_ULP, LEAST, matrix
from tokmem import DT, U, Big, Dev, to_bits, to_f64, within

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module", autouse=True)
def device():
    pywelvet.init()


@pytest.fixture
def stream():
    s = Stream()
    yield s.h
    s.sync()
    s.close()


def expected(xc, xs, wc, ws, bias, name):
    total = xc.astype(np.float64) @ wc.T.astype(np.float64)  # whole, below 2^53
    with np.errstate(invalid="ignore"):
        product = total * (xs.astype(np.float64)[:, None] * ws.astype(np.float64))
    b = np.zeros(wc.shape[0]) if bias is None else bias
    pre = product + b
    err = 4 * U * (np.abs(product) + np.abs(b)) + TINY
    post = act(pre, name)
    slope = 2 * np.abs(pre) + 2 * err if name == "relu2" else 1.2
    return pre, err, post, slope * err + ACT_ERR * (np.abs(pre) + (np.abs(post) if name == "relu2" else 1))


def run(stream, layer, dtype, n, ptr, rows=None, x_stride=None, pre=True, post=True, extra=0):
    item = to_bits(np.zeros(1), dtype).dtype
    a, b = (Dev(np.full((n, layer.out + extra), 5, item)) for _ in range(2))
    ws = Dev(np.full(layer.workspace_bytes(n), 0xFF, np.uint8))
    layer.forward(DT[dtype], n, ptr, rows=rows, d_pre=a.ptr if pre else None, d_post=b.ptr if post else None,
                  x_stride=x_stride, pre_stride=layer.out + extra, post_stride=layer.out + extra, ws=ws.ptr,
                  ws_bytes=ws.nbytes, stream=stream)
    ws.get()
    a, b = a.get(), b.get()
    assert (a[:, layer.out:] == 5).all() and (b[:, layer.out:] == 5).all()
    return a[:, :layer.out], b[:, :layer.out]


SHAPES = [(1, 1, 1), (1, 17, 5), (3, 1001, 777), (2, 64, 16), (16, 128, 100), (17, 500, 33), (33, 4096, 48),
          (64, 777, 129), (65, 100, 130), (100, 1001, 777), (129, 64, 257), (300, 2000, 300), (700, 130, 5000),
          (1, 11008, 64), (40, 20000, 32), (4200, 192, 2100), (20, 4200, 1040), (64, 4200, 1040), (19, 1000, 4500),
          (50, 300, 20000), (130, 2000, 8300),
          (5, 1600, 21000), (2, 1600, 21001), (128, 300, 66000), (3, 700, 9000)]


@pytest.mark.parametrize("dtype", DT)
@pytest.mark.parametrize("n,inn,out", SHAPES)
def test_forward(stream, dtype, n, inn, out):
    rng = np.random.default_rng([n, inn, out])
    W = rng.normal(0, inn ** -0.5, (out, inn)).astype(np.float32)
    bias = rng.normal(0, 0.5, out) if n % 2 else None
    name = ACTS[(n + out) % len(ACTS)]
    extra, shift = inn % 3, out % 4
    with pywelvet.Int8Layer(W, pywelvet.ACT[name], bias) as layer:
        wc, wscale = layer.weights()
        want, wanted = codes_of(W)
        assert np.array_equal(wc, want)
        assert_bit_equal(wscale, wanted, "channel scales")
        d, ptr, x = matrix(rng.normal(0, 1, (n, inn)) * np.exp(rng.normal(0, 1, (n, 1))), dtype, extra, shift)
        rows = Rows(n, inn, 1)
        pre, post = run(stream, layer, dtype, n, ptr, rows.desc, inn + extra, extra=out % 2)
        xc, xs = rows.get()
        want, wanted = codes_of(x)
        assert np.array_equal(xc, want)
        assert_bit_equal(xs, wanted, "row scales")
        b = None if bias is None else bias.astype(np.float32).astype(np.float64)
        wp, ep, wq, eq = expected(xc, xs, wc, wscale, b, name)
        within(to_f64(pre, dtype), wp, ep * 1.01 + HALF_ULP[dtype] * np.abs(wp) + LEAST[dtype], "pre")
        within(to_f64(post, dtype), wq, eq * 1.01 + HALF_ULP[dtype] * np.abs(wq) + LEAST[dtype], "post")
        # without the rows, one output at a time, and from the rows
        assert_bit_equal(run(stream, layer, dtype, n, ptr, None, inn + extra, post=False)[0], pre, "pre alone")
        assert_bit_equal(run(stream, layer, dtype, n, ptr, None, inn + extra, pre=False)[1], post, "post alone")
        again = Dev(np.zeros_like(post))
        ws = Dev(np.zeros(layer.workspace_bytes(n), np.uint8))
        layer.product(DT[dtype], n, rows.desc, d_post=again.ptr, ws=ws.ptr, ws_bytes=ws.nbytes, stream=stream)
        assert_bit_equal(again.get(), post, "from rows")


@pytest.mark.parametrize("inn,out", [(777, 300), (4096, 520), (11008, 64), (11008, 400), (1600, 21000)])
def test_a_row_has_the_same_bits_in_every_batch(stream, inn, out):
    rng = np.random.default_rng([inn, out])
    x = rng.normal(0, 1, (1100, inn)).astype(np.float32)
    d = Dev(x)
    with pywelvet.Int8Layer(rng.normal(0, 0.02, (out, inn)), pywelvet.ACT["gelu"], rng.normal(0, 1, out)) as layer:
        _, whole = run(stream, layer, "float32", 1100, d.ptr)
        for n in (1, 2, 3, 5, 16, 17, 32, 50, 64, 65, 128, 200, 256, 400, 1000):
            assert_bit_equal(run(stream, layer, "float32", n, d.ptr)[1], whole[:n], f"{n} rows")


def test_the_largest_sum(stream):
    """in = 131072 with every code at 127 reaches 2^31 - 2^21 or so, exact in 32 bits."""
    inn = 131072
    W = np.ones((3, inn), np.float32)
    W[1] = -1
    with pywelvet.Int8Layer(W) as layer:
        for n in (1, 70):
            d = Dev(np.full((n, inn), 127, np.float32))
            pre, _ = run(stream, layer, "float32", n, d.ptr)
            want = np.float64(np.float32(1) / np.float32(127)) * 127 * 127 * inn
            within(pre, np.tile([want, -want, want], (n, 1)), 4 * U * want, "pre")
    with pytest.raises(pywelvet.WelvetError) as e:
        pywelvet.Int8Layer(np.zeros((1, inn + 1), np.float32))
    assert e.value.code == 1


def test_long_sums_of_many_channels(stream):
    """129 tiles of channels, whose sums are long enough to be split in three all the same."""
    inn, out, rng = 13000, 16500, np.random.default_rng(9)
    w = rng.integers(-127, 128, (out, inn), dtype=np.int8)
    c = np.zeros((100, 13008), np.int8)
    c[:, :inn] = rng.integers(-127, 128, (100, inn))
    scales, ws = rng.uniform(0.5, 1, 100).astype(np.float32), rng.uniform(0.5, 1, out).astype(np.float32)
    # whole numbers below 2^53: exact in f64
    sums = np.concatenate([c[:, :inn].astype(np.float64) @ w[o:o + 1500].T.astype(np.float64)
                           for o in range(0, out, 1500)], 1)
    want = sums * scales.astype(np.float64)[:, None] * ws.astype(np.float64)
    codes, sc = Dev(c), Dev(scales)
    with pywelvet.Int8Layer.from_codes(w, ws) as layer:
        for n in (1, 60, 100):
            pre = Dev(np.zeros((n, out), np.float32))
            work = Dev(np.full(layer.workspace_bytes(n), 0xFF, np.uint8))
            layer.product(1, n, pywelvet.rows8(codes.ptr, 13008, sc.ptr), d_pre=pre.ptr, ws=work.ptr,
                          ws_bytes=work.nbytes, stream=stream)
            work.get()
            within(pre.get(), want[:n], 4 * U * np.abs(want[:n]), f"{n} rows")


@pytest.mark.parametrize("n", [2, 9, 70])
def test_rows_past_32_bits(stream, n):
    """The last row of x, of post and of the rows left behind begins past 2^32 values
    (of codes: bytes), and has the bits that it has beside the others."""
    inn, out, rng = 100, 300, np.random.default_rng(n)
    stride = (2 ** 32 // (n - 1) + 64) // 16 * 16
    x = rng.normal(0, 1, (n, inn)).astype(np.float32)
    with pywelvet.Int8Layer(rng.normal(0, 0.1, (out, inn)), pywelvet.ACT["gelu"]) as layer:
        d = Dev(x)
        want = run(stream, layer, "float32", n, d.ptr)[1]
        rows, scales = Big(stride * n), Dev(np.zeros(n, np.float32))
        far, post = Big(4 * (stride * (n - 1) + inn)), Big(4 * (stride * (n - 1) + out))
        for r in range(n):
            far.put(4 * stride * r, x[r])
        ws = Dev(np.full(layer.workspace_bytes(n), 0xFF, np.uint8))
        for kept in (None, pywelvet.rows8(rows.ptr, stride, scales.ptr)):
            layer.forward(1, n, far.ptr, rows=kept, d_post=post.ptr, x_stride=stride, post_stride=stride, ws=ws.ptr,
                          ws_bytes=ws.nbytes, stream=stream)
            ws.get()
            for r in range(n):
                assert_bit_equal(post.get(4 * stride * r, out, np.float32), want[r], f"row {r}")
        codes, _ = codes_of(x)
        assert np.array_equal(rows.get(stride * (n - 1), inn, np.int8), codes[n - 1])
        for b in (rows, far, post):
            b.free()


def test_codes_past_the_width_do_not_matter(stream):
    rng = np.random.default_rng(5)
    for n, inn, out in ((3, 33, 20), (40, 77, 20), (200, 100, 300)):
        codes = rng.integers(-127, 128, (n, inn))
        scales = rng.uniform(0.5, 1, n).astype(np.float32)
        with pywelvet.Int8Layer(rng.normal(0, 1, (out, inn))) as layer:
            got = []
            for fill in (0, 127):
                rows = Rows(n, inn, 1)
                host = np.full((n, rows.stride), fill, np.int8)
                host[:, :inn] = codes
                rows.codes = Dev(host)
                s = Dev(scales)
                rows.desc = pywelvet.rows8(rows.codes.ptr, rows.stride, s.ptr)
                y, ws = Dev(np.zeros((n, out), np.float32)), Dev(np.zeros(layer.workspace_bytes(n), np.uint8))
                layer.product(1, n, rows.desc, d_post=y.ptr, ws=ws.ptr, ws_bytes=ws.nbytes, stream=stream)
                got.append(y.get())
            assert_bit_equal(got[0], got[1], f"{n} rows of {inn}")


def test_rows_and_channels_that_are_not_finite_or_zero(stream):
    rng = np.random.default_rng(6)
    for n in (5, 100):
        x, W = rng.normal(0, 1, (n, 60)).astype(np.float32), rng.normal(0, 1, (40, 60)).astype(np.float32)
        x[1], x[2, 3], x[3, 59] = 0, np.nan, np.inf
        W[4], W[5, 0] = 0, -np.inf
        d = Dev(x)
        with pywelvet.Int8Layer(W, bias=np.arange(40)) as layer:
            pre, _ = run(stream, layer, "float32", n, d.ptr)
        assert np.isnan(pre[2:4]).all() and np.isnan(pre[:, 5]).all()
        fine = np.delete(np.delete(pre, [2, 3], 0), 5, 1)
        assert np.isfinite(fine).all()
        assert np.array_equal(np.delete(pre[1], 5), np.delete(np.arange(40), 5))
        assert (np.delete(pre[:, 4], [2, 3]) == 4).all()


@pytest.mark.parametrize("dtype", [0, 1, 3, 4, 9, 13, 26, 33])
def test_mount_from_a_session(stream, dtype):
    """The layer holds what the session's store decodes to, its bias and its activation."""
    rng = np.random.default_rng(dtype)
    W, bias = rng.normal(0, 0.3, (48, 70)).astype(np.float32), rng.normal(0, 1, 48)
    x = rng.normal(0, 1, (9, 70)).astype(np.float32)
    with pywelvet.Session(W, 9, pywelvet.ACT["silu"], dtype, bias) as s:
        values = s.export_f32()
        codes, scales = codes_of(values)
        with pywelvet.Int8Layer.from_session(s) as layer, pywelvet.Int8Layer(values, 1, bias) as other, \
                pywelvet.Int8Layer.from_codes(codes, scales, 1, bias) as third:
            for a, b in zip(layer.weights(), other.weights()):
                assert_bit_equal(a, b, "weights")
            d = Dev(x)
            for a, b in zip(run(stream, layer, "float32", 9, d.ptr), run(stream, other, "float32", 9, d.ptr)):
                assert_bit_equal(a, b, "outputs")
            assert_bit_equal(run(stream, third, "float32", 9, d.ptr)[1], run(stream, other, "float32", 9, d.ptr)[1],
                             "from codes")


def test_two_streams_share_a_layer(stream):
    rng = np.random.default_rng(8)
    x = [rng.normal(0, 1, (n, 512)).astype(np.float32) for n in (3, 90)]
    with pywelvet.Int8Layer(rng.normal(0, 1, (640, 512))) as layer:
        ds = [Dev(a) for a in x]
        want = [run(stream, layer, "float32", len(a), d.ptr)[1] for a, d in zip(x, ds)]
        other = Stream()
        ys = [Dev(np.zeros((len(a), 640), np.float32)) for a in x]
        wss = [Dev(np.zeros(layer.workspace_bytes(len(a)), np.uint8)) for a in x]
        for _ in range(10):
            for d, y, ws, at, a in zip(ds, ys, wss, (stream, other.h), x):
                layer.forward(1, len(a), d.ptr, d_post=y.ptr, ws=ws.ptr, ws_bytes=ws.nbytes, stream=at)
        for y, w in zip(ys, want):
            assert_bit_equal(y.get(), w, "overlapping calls")
        other.close()
