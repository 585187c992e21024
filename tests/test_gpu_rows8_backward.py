"""welvet_hip_rows8_backward: a layer's backward from 8-bit activations against f64.

Bounds.  The activations' values are rounded once (U |pre|, U of x), act' is
within 64 U, dpre one rounding more and then its type's.  A product's terms
carry that, one rounding of the scale's product and what the f16 parts leave:
2^-22 or 2^-11 of a term for two or one (each part is within 2^-11 of what is
left), and f16's last place, half of 2^-24, where the largest |dy| scale
times what |act'| can be (below 1.3, or 2 |pre| <= 254 scales) lies from 2^14
on: 2^-39 of it.  A sum of K terms in f32 is within (P K + 8) U of the sum of
their magnitudes."""
import numpy as np
import pytest

import pywelvet
from devmem import Stream
from parity import assert_bit_equal
from rows8ref import ACTS, PRIME_ERR, Rows, act, act_prime, codes_of, values
from test_gpu_rows8 import HALF_ULP, LEAST, matrix
from tokmem import DT, U, Big, Dev, to_bits, to_f64, within

pytestmark = pytest.mark.gpu
PARTS = {"float32": (2, 2), "float16": (2, 2), "bfloat16": (2, 1)}


@pytest.fixture(scope="module", autouse=True)
def device():
    pywelvet.init()


@pytest.fixture
def stream():
    s = Stream()
    yield s.h
    s.sync()
    s.close()


class Case:
    def __init__(self, dtype, n, inn, out, name, seed=0, layer=True, extra=0, shift=0):
        rng = np.random.default_rng([n, inn, out, seed])
        self.dtype, self.n, self.inn, self.out, self.name, self.extra = dtype, n, inn, out, name, extra
        self.xc, self.xs = codes_of(rng.normal(0, 1, (n, inn)).astype(np.float32) if n else np.zeros((0, inn)))
        self.pc, self.ps = codes_of((rng.normal(0, 2, (n, out)) * np.exp(rng.normal(0, 1, (n, 1)))).astype(np.float32)
                                    if n else np.zeros((0, out)))
        self.x8, self.pre8 = Rows(n, inn, 1, self.xc, self.xs), Rows(n, out, 0, self.pc, self.ps)
        self.d, self.dy_ptr, self.dy = matrix(rng.normal(0, 1, (n, out)) * 1e-2, dtype, extra, shift)
        self.layer = pywelvet.Int8Layer(rng.normal(0, 1, (out, inn)) * np.exp(rng.normal(0, 1, (out, 1)))) if layer else None
        self.item = to_bits(np.zeros(1), dtype).dtype
        self.ws = Dev(np.full(max(16, pywelvet.rows8_backward_bytes(DT[dtype], n, inn, out)), 0xFF, np.uint8))

    def run(self, stream, dpre=True, dx=True, dw=True, base=None, ws=None, in_place=False):
        e = self.extra
        a, b = Dev(np.full((self.n, self.out + e), 5, self.item)), Dev(np.full((self.n, self.inn + e), 5, self.item))
        c = Dev(np.full((self.out, self.inn), 3.0, np.float32) if base is None else base)
        ws = self.ws if ws is None else ws
        pywelvet.rows8_backward(
            pywelvet.ACT[self.name], DT[self.dtype], self.n, self.inn, self.out, self.dy_ptr,
            pre=None if self.name == "linear" else self.pre8.desc, x=self.x8.desc if dw else None,
            layer=self.layer if dx else None, d_dpre=(self.dy_ptr if in_place else a.ptr) if dpre else None,
            d_dx=b.ptr if dx else None, d_dw=c.ptr if dw else None, accumulate=base is not None,
            dy_stride=self.out + e, dpre_stride=self.out + e, dx_stride=self.inn + e, ws=ws.ptr, ws_bytes=ws.nbytes,
            stream=stream)
        ws.get()
        a, b = a.get(), b.get()
        assert (a[:, self.out:] == 5).all() and (b[:, self.inn:] == 5).all()
        return (a[:, :self.out] if dpre else None, b[:, :self.inn] if dx else None, c.get() if dw else None)

    def want(self):
        pre = values(self.pc, self.ps)
        prime = act_prime(pre, self.name)
        dpre = self.dy * prime
        smooth = self.name in ("silu", "gelu", "tanh", "sigmoid")
        err = np.abs(self.dy) * (PRIME_ERR + U * np.abs(pre) if smooth else 0) + 3 * U * np.abs(dpre)
        x = values(self.xc, self.xs)
        return dpre, err, x

    def check(self, stream, base=None, **kw):
        dpre, dx, dw = self.run(stream, base=base, **kw)
        want, err, x = self.want()
        half, pw, px = HALF_ULP[self.dtype], *PARTS[self.dtype]
        steep = 256.0 * self.ps if self.name == "relu2" else np.full(self.n, 1.3)
        if dpre is not None and not kw.get("in_place"):
            within(to_f64(dpre, self.dtype), want, err + half * (np.abs(want) + err) + LEAST[self.dtype], "dpre")
        if dw is not None:
            total, ab, more = want.T @ x, np.abs(want).T @ np.abs(x), err.T @ np.abs(x)
            b = 0 if base is None else base
            least = 2.0 ** -39 * np.abs(steep[:, None] * self.dy * self.xs[:, None]).max(0, initial=0)
            more = more + least[:, None] * np.abs(self.xc).sum(0)
            within(dw, total + b, more + ab * (2.0 ** (-11 * pw) + (pw * self.n + 12) * U)
                   + U * np.abs(total + b) * 2 + 1e-36, "dw")
        if dx is not None:
            wc, ws = self.layer.weights()
            W = values(wc, ws)
            total, ab, more = want @ W, np.abs(want) @ np.abs(W), err @ np.abs(W)
            least = 2.0 ** -39 * np.abs(steep[:, None] * self.dy * ws).max(1, initial=0)
            more = more + least[:, None] * np.abs(wc.astype(np.float64)).sum(0)
            bound = more + ab * (2.0 ** (-11 * px) + (px * self.out + 12) * U)
            within(to_f64(dx, self.dtype), total, bound * 1.01 + half * np.abs(total) + LEAST[self.dtype] * 2, "dx")
        return dpre, dx, dw


SHAPES = [(1, 1, 1), (1, 40, 70), (3, 17, 5), (31, 64, 64), (32, 65, 63), (33, 100, 129), (100, 1001, 777),
          (65, 300, 260), (256, 512, 1100), (700, 130, 33), (2100, 200, 128), (64, 600, 4100), (40, 130, 2050), (130, 8300, 1100),
          (1100, 2100, 1000), (130, 8300, 3300), (3300, 2100, 1000)]


@pytest.mark.parametrize("dtype", DT)
@pytest.mark.parametrize("n,inn,out", SHAPES)
def test_backward(stream, dtype, n, inn, out):
    case = Case(dtype, n, inn, out, ACTS[(n + inn) % len(ACTS)], extra=out % 3, shift=inn % 4)
    dpre, dx, dw = case.check(stream)
    again = case.run(stream)
    for a, b, what in zip(again, (dpre, dx, dw), ("dpre", "dx", "dw")):
        assert_bit_equal(a, b, what + " of a second run")
    for k, what in enumerate(("dpre", "dx", "dw")):  # each alone has the same bits
        only = case.run(stream, dpre=k == 0, dx=k == 1, dw=k == 2)
        assert_bit_equal(only[k], (dpre, dx, dw)[k], what + " alone")
    base = np.random.default_rng(1).normal(0, 1, (out, inn)).astype(np.float32)
    case.check(stream, base=base)
    case.run(stream, dx=False, dw=False, in_place=True)
    placed = case.d.get()[inn % 4:].reshape(n, out + case.extra)[:, :out]
    assert_bit_equal(placed, dpre, "dpre in dy's place")


# up to eight rows go another way: columns past a block's 512 and 1024, channels past its 512, odd sizes
FEW = [(1, 1025, 1600), (2, 513, 100), (3, 2051, 1031), (4, 1024, 520), (5, 7, 3000), (7, 515, 31), (8, 1000, 2049),
       (9, 1000, 2049), (16, 515, 700), (17, 515, 700)]


@pytest.mark.parametrize("dtype", DT)
@pytest.mark.parametrize("n,inn,out", FEW)
def test_few_rows(stream, dtype, n, inn, out):
    case = Case(dtype, n, inn, out, ACTS[(n + inn) % len(ACTS)], 8, extra=out % 3, shift=inn % 4)
    first = case.check(stream)
    for k in range(3):
        assert_bit_equal(case.run(stream, dpre=k == 0, dx=k == 1, dw=k == 2)[k], first[k], "alone")
    base = np.random.default_rng(2).normal(0, 1, (out, inn)).astype(np.float32)
    case.check(stream, base=base)
    placed = case.run(stream, in_place=True)
    assert_bit_equal(case.d.get()[inn % 4:].reshape(n, out + case.extra)[:, :out], first[0], "dpre in dy's place")
    assert_bit_equal(placed[1], first[1], "dx, dpre in dy's place")
    assert_bit_equal(placed[2], first[2], "dw, dpre in dy's place")


@pytest.mark.parametrize("dtype", DT)
@pytest.mark.parametrize("n", [2, 70, 200])
def test_dpre_in_the_place_of_dy_with_both_products(stream, dtype, n):
    case = Case(dtype, n, 130, 140, "silu", 9)
    first = case.run(stream)
    placed = case.run(stream, in_place=True)
    assert_bit_equal(case.d.get().reshape(n, 140), first[0], "dpre")
    for k in (1, 2):
        assert_bit_equal(placed[k], first[k], "products")


@pytest.mark.parametrize("dtype", DT)
def test_few_rows_that_are_not_finite(stream, dtype):
    case = Case(dtype, 5, 50, 60, "linear", 5)
    dy = case.dy.copy()
    dy[2, 9] = np.inf
    case.d, case.dy_ptr, case.dy = matrix(dy, dtype)
    dpre, dx, dw = case.run(stream)
    dx, dw = to_f64(dx, dtype), dw.astype(np.float64)
    assert not np.isfinite(dx[2]).any() and np.isfinite(np.delete(dx, 2, 0)).all()
    assert not np.isfinite(dw[9]).any() and np.isfinite(np.delete(dw, 9, 0)).all()
    case.xs[3] = np.nan
    case.x8 = Rows(5, 50, 1, case.xc, case.xs)
    assert np.isnan(case.run(stream)[2]).all()


@pytest.mark.parametrize("dtype", DT)
@pytest.mark.parametrize("name", ACTS)
def test_every_activation(stream, dtype, name):
    Case(dtype, 70, 90, 110, name, 1).check(stream)


@pytest.mark.parametrize("dtype", DT)
def test_large_tiles(stream, dtype):
    """Sizes past 256 x 256 tiles on every side, none of them a multiple."""
    Case(dtype, 2900, 2900, 2900, "silu", 2, extra=1).check(stream)


def test_gradients_against_differences(stream):
    """The layer's own loss sum(dy act(x W^T)) at the values held, differentiated numerically."""
    case = Case("float32", 6, 20, 9, "gelu", 3)
    wc, ws = case.layer.weights()
    W, x = values(wc, ws), values(case.xc, case.xs)
    pre = x @ W.T * 0.1
    case.pc, case.ps = codes_of(pre.astype(np.float32))
    case.pre8 = Rows(6, 9, 0, case.pc, case.ps)
    dpre, dx, dw = case.run(stream)
    p, step = values(case.pc, case.ps), 1e-5
    d = case.dy * (act(p + step, "gelu") - act(p - step, "gelu")) / (2 * step)
    # differences are off by step^2 / 6 of a third derivative of at most 3 and f64's rounding over the step
    size = np.abs(case.dy)
    within(dpre, d, 1e-5 * size, "dpre")
    within(dx, d @ W, 1e-5 * size @ np.abs(W) + 1e-6 * np.abs(d) @ np.abs(W), "dx")
    within(dw, d.T @ x, 1e-5 * size.T @ np.abs(x) + 1e-6 * np.abs(d).T @ np.abs(x), "dw")


@pytest.mark.parametrize("n", [5, 17, 140])
def test_rows_past_32_bits(stream, n):
    """The last rows of dy, dpre, dx begin past 2^32 values and the activations' past
    2^32 bytes; all have the bits that they have beside the others."""
    case = Case("bfloat16", n, 100, 130, "silu", 10)
    first = case.run(stream)
    stride = (2 ** 32 // (n - 1) + 160) // 16 * 16
    dy, dpre, dx = (Big(2 * (stride * (n - 1) + w)) for w in (130, 130, 100))
    x8, pre8 = Big(stride * n), Big(stride * n)
    bits = case.d.get().reshape(n, 130)
    for r in range(n):
        dy.put(2 * stride * r, bits[r])
        for to, codes in ((x8, case.xc), (pre8, case.pc)):
            to.put(stride * r, codes[r].astype(np.int8))
    xs, ps, dw = Dev(case.xs), Dev(case.ps), Dev(np.zeros((130, 100), np.float32))
    pywelvet.rows8_backward(
        pywelvet.ACT["silu"], 3, n, 100, 130, dy.ptr, pre=pywelvet.rows8(pre8.ptr, stride, ps.ptr),
        x=pywelvet.rows8(x8.ptr, stride, xs.ptr), layer=case.layer, d_dpre=dpre.ptr, d_dx=dx.ptr, d_dw=dw.ptr,
        dy_stride=stride, dpre_stride=stride, dx_stride=stride, ws=case.ws.ptr, ws_bytes=case.ws.nbytes, stream=stream)
    case.ws.get()
    for r in range(n):
        assert_bit_equal(dpre.get(2 * stride * r, 130, np.uint16), first[0][r], f"dpre {r}")
        assert_bit_equal(dx.get(2 * stride * r, 100, np.uint16), first[1][r], f"dx {r}")
    assert_bit_equal(dw.get(), first[2], "dw")
    for b in (dy, dpre, dx, x8, pre8):
        b.free()


def test_no_rows(stream):
    case = Case("float32", 0, 30, 20, "silu", 4)
    ones = np.ones((20, 30), np.float32)
    assert (case.run(stream, dpre=False, dx=False, dw=True)[2] == 0).all()
    assert_bit_equal(case.run(stream, dpre=False, dx=False, dw=True, base=ones)[2], ones, "added to")


def test_values_that_are_not_finite(stream):
    """A NaN row of the input makes dw NaN; an infinite gradient reaches its own
    row of dx and its own channel of dw, and nothing else; other rows and channels stay."""
    for dtype in DT:
        case = Case(dtype, 40, 50, 60, "linear", 5)
        dy = case.dy.copy()
        dy[7, 9] = np.inf
        case.d, case.dy_ptr, case.dy = matrix(dy, dtype)
        dpre, dx, dw = case.run(stream)
        dx, dw = to_f64(dx, dtype), dw.astype(np.float64)
        assert not np.isfinite(dx[7]).any() and np.isfinite(np.delete(dx, 7, 0)).all()
        assert not np.isfinite(dw[9]).any() and np.isfinite(np.delete(dw, 9, 0)).all()
        # inf times a code: infinite where the code is not 0, as the formula has it
        some = case.xc[7] != 0
        assert np.isinf(dw[9][some]).all() and np.isnan(dw[9][~some]).all()
        case = Case(dtype, 40, 50, 60, "linear", 5)
        case.xs[3] = np.nan
        case.x8 = Rows(40, 50, 1, case.xc, case.xs)
        dpre, dx, dw = case.run(stream)
        assert np.isnan(dw).all() and np.isfinite(to_f64(dx, dtype)).all()


def test_a_smaller_batch_in_the_same_workspace(stream):
    big = Case("bfloat16", 300, 130, 140, "silu", 6)
    for n in (299, 64, 33, 1):
        case = Case("bfloat16", n, 130, 140, "silu", 7)
        want = case.check(stream)
        got = case.run(stream, ws=big.ws)
        for a, b in zip(got, want):
            assert_bit_equal(a, b, f"{n} rows")
