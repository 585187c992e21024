"""welvet_hip_rows8_*: rows in 8 bits and SwiGLU between them, against f64.

Codes and scales are whole: they have to be equal.  h = silu(gate) up is two
products of a sigmoid within 8 U: 10 U of |h|, and what the exponential leaves
out below 2^-126.  Of 16-bit types the exponential's argument is rounded to
f32, U |gate| of it and so of the sigmoid, and taken times a rounded log2 e, as
much again.  Its code is off by at most half a step of its own row and
what h is off; the scale by 11 U."""
import numpy as np
import pytest

import pywelvet
from devmem import Stream
from parity import assert_bit_equal
from rows8ref import PRIME_ERR, TINY, Rows, act, act_prime, codes_of, values
from tokmem import DT, U, Dev, strided, to_bits, to_f64, within

pytestmark = pytest.mark.gpu
HALF_ULP = {"float32": U, "float16": 2.0 ** -11, "bfloat16": 2.0 ** -8}
LEAST = {"float32": TINY, "float16": 2.0 ** -24, "bfloat16": TINY}


@pytest.fixture(scope="module", autouse=True)
def device():
    pywelvet.init()


@pytest.fixture
def stream():
    s = Stream()
    yield s.h
    s.sync()
    s.close()


def matrix(x, dtype, extra=0, shift=0):
    """x on the device in rows of `extra` more values, `shift` values past an alignment of 16."""
    bits = to_bits(x, dtype)
    d = Dev(np.concatenate([np.zeros(shift, bits.dtype), strided(bits, extra).reshape(-1)]))
    return d, d.ptr + shift * bits.dtype.itemsize, to_f64(bits, dtype)


SHAPES = [(1, 1), (3, 7), (2, 8), (5, 15), (4, 16), (3, 17), (300, 100), (100, 777), (7, 1001), (5, 1024), (3, 1025),
          (2, 4096), (4, 8192), (3, 8193), (2, 11008), (1, 40000), (2, 33001)]


@pytest.mark.parametrize("dtype", DT)
@pytest.mark.parametrize("n,width", SHAPES)
def test_store_and_load(stream, dtype, n, width):
    rng = np.random.default_rng([n, width])
    extra, shift = (n + width) % 3, width % 4
    d, ptr, x = matrix(rng.normal(0, 1, (n, width)) * np.exp(rng.normal(0, 2, (n, 1))), dtype, extra, shift)
    rows = Rows(n, width, extra)
    pywelvet.rows8_store(DT[dtype], n, width, ptr, rows.desc, x_stride=width + extra, stream=stream)
    codes, scales = rows.get()
    want, ws = codes_of(x)
    assert_bit_equal(scales, ws, "scales")
    assert np.array_equal(codes, want)
    back = Dev(np.full((n, width + extra), 5, to_bits(np.zeros(1), dtype).dtype))
    pywelvet.rows8_load(DT[dtype], n, width, rows.desc, back.ptr, x_stride=width + extra, stream=stream)
    got = back.get()
    assert (got[:, width:] == 5).all()
    v = values(want, ws)
    within(to_f64(got[:, :width], dtype), v, HALF_ULP[dtype] * np.abs(v) * (1 + U) + U * np.abs(v) + LEAST[dtype], "loaded")


def test_codes_next_to_a_half(stream):
    """Values on, just above and just below (k + 1/2) scale for scales of every
    kind of mantissa: the exact quotient decides, ties go to the even code."""
    rng = np.random.default_rng(3)
    rows, width = 64, 1 + 3 * 127
    x = np.zeros((rows, width), np.float32)
    for r in range(rows):
        top = np.float32(127 * 2.0 ** (r - 32)) if r % 2 else np.float32(rng.uniform(1, 2) * 2.0 ** (r - 30))
        s = np.float64(np.float32(top / np.float32(127)))
        half = ((np.arange(127) + 0.5) * s).astype(np.float32)
        x[r, 0] = top
        x[r, 1:] = np.concatenate([half, np.nextafter(half, np.float32(0)), np.nextafter(half, np.float32(np.inf))])
    x[:, 1:] *= np.where(rng.random((rows, width - 1)) < 0.5, -1, 1)
    d, rows8 = Dev(x), Rows(rows, width)
    pywelvet.rows8_store(1, rows, width, d.ptr, rows8.desc, stream=stream)
    codes, scales = rows8.get()
    want, ws = codes_of(x)
    assert_bit_equal(scales, ws, "scales")
    assert np.array_equal(codes, want)


def test_rows_at_the_ends_of_f32(stream):
    """Zeros, the smallest floats, the largest, and rows that are not finite."""
    tiny = np.float32(1e-45)
    x = np.zeros((12, 40), np.float32)
    x[1] = np.arange(40) * tiny
    x[2] = np.arange(40) * tiny * 1000
    x[3] = np.arange(40) * np.float32(1e-37)
    x[4] = np.linspace(-3.4e38, 3.4e38, 40)
    x[5, 7] = np.nan
    x[6, 39] = -np.inf
    x[7] = -0.0
    x[8] = np.linspace(-1, 1, 40) * 2.0 ** -101
    x[9] = np.linspace(-1, 1, 40) * 2.0 ** -93
    x[10, 0] = tiny
    x[11] = np.linspace(-1, 1, 40) * 127 * 2.0 ** -149
    d, rows = Dev(x), Rows(12, 40)
    pywelvet.rows8_store(1, 12, 40, d.ptr, rows.desc, stream=stream)
    codes, scales = rows.get()
    want, ws = codes_of(x)
    assert np.array_equal(scales, ws, equal_nan=True)
    assert np.array_equal(codes, want)
    back = Dev(np.zeros((12, 40), np.float32))
    pywelvet.rows8_load(1, 12, 40, rows.desc, back.ptr, stream=stream)
    got = back.get()
    assert np.isnan(got[5:7]).all() and np.isfinite(got[[0, 1, 2, 3, 4, 7, 8, 9, 10, 11]]).all()


def swiglu_in(rng, n, width):
    gate, up = rng.normal(0, 2, (n, width)), rng.normal(0, 1, (n, width))
    gate[:, ::7] *= 20
    return gate, up


@pytest.mark.parametrize("dtype", DT)
@pytest.mark.parametrize("n,width", SHAPES)
def test_swiglu(stream, dtype, n, width):
    rng = np.random.default_rng([n, width, 1])
    extra, shift = width % 3, n % 4
    gate, up = swiglu_in(rng, n, width)
    (_g, pg, gate), (_u, pu, up) = matrix(gate, dtype, extra, shift), matrix(up, dtype, 1, 0)
    g8, u8, h8 = Rows(n, width, 1), Rows(n, width), Rows(n, width, 2)
    h = Dev(np.full((n, width + 3), 5, to_bits(np.zeros(1), dtype).dtype))
    kw = dict(gate_stride=width + extra, up_stride=width + 1, stream=stream)
    pywelvet.rows8_swiglu(DT[dtype], n, width, pg, pu, g8.desc, u8.desc, h8.desc, h.ptr, h_stride=width + 3, **kw)
    want = act(gate, "silu") * up
    err = (10 + (0 if dtype == "float32" else 2 * np.abs(gate))) * U * np.abs(want) + TINY * np.abs(gate * up)
    got = h.get()
    assert (got[:, width:] == 5).all()
    within(to_f64(got[:, :width], dtype), want, err * 2 + HALF_ULP[dtype] * np.abs(want) + LEAST[dtype], "h")
    for rows, x in ((g8, gate), (u8, up)):
        codes, scales = rows.get()
        wc, ws = codes_of(x)
        assert_bit_equal(scales, ws, "scales")
        assert np.array_equal(codes, wc)
    codes, scales = h8.get()
    top = np.abs(want).max(1) / 127
    off = np.max(err / (np.abs(want) + TINY), axis=1, initial=0)  # the largest value's own
    within(scales, top, (off + U) * top + TINY, "h's scales")
    within(values(codes, scales), want, (0.5001 + 128 * (off[:, None] + U)) * top[:, None] + err + TINY, "h's codes")
    # the outputs one by one have the same bits
    for k, rows in enumerate((g8, u8, h8)):
        only = Rows(n, width)
        ask = [None, None, None]
        ask[k] = only.desc
        pywelvet.rows8_swiglu(DT[dtype], n, width, pg, pu, *ask, **kw)
        assert np.array_equal(only.get()[0], rows.get()[0])
        assert_bit_equal(only.get()[1], rows.get()[1], "scales")


@pytest.mark.parametrize("dtype", DT)
@pytest.mark.parametrize("n,width", SHAPES)
def test_swiglu_backward(stream, dtype, n, width):
    rng = np.random.default_rng([n, width, 2])
    gate, up = swiglu_in(rng, n, width)
    (gc, gs), (uc, us) = codes_of(to_f64(to_bits(gate, dtype), dtype)), codes_of(to_f64(to_bits(up, dtype), dtype))
    g8, u8 = Rows(n, width, 1, gc, gs), Rows(n, width, 0, uc, us)
    extra, shift = n % 3, width % 4
    d, ptr, dh = matrix(rng.normal(0, 1, (n, width)) * 1e-2, dtype, extra, shift)
    item = to_bits(np.zeros(1), dtype).dtype
    dg, du = Dev(np.full((n, width + 1), 5, item)), Dev(np.full((n, width + 2), 5, item))
    call = lambda a, b, **kw: pywelvet.rows8_swiglu_backward(  # noqa: E731
        DT[dtype], n, width, g8.desc, u8.desc, ptr, a, b, dh_stride=width + extra, stream=stream, **kw)
    call(dg.ptr, du.ptr, dgate_stride=width + 1, dup_stride=width + 2)
    g, u = values(gc, gs), values(uc, us)
    wg, wu = dh * u * act_prime(g, "silu"), dh * act(g, "silu")
    got_g, got_u = dg.get(), du.get()
    assert (got_g[:, width:] == 5).all() and (got_u[:, width:] == 5).all()
    # the values themselves are rounded once: u by U, g by U |g|, which moves silu'(g) by at most U |g| / 2
    within(to_f64(got_g[:, :width], dtype), wg, np.abs(dh * u) * (PRIME_ERR + U * np.abs(g))
           + HALF_ULP[dtype] * np.abs(wg) * 1.001 + LEAST[dtype], "dgate")
    within(to_f64(got_u[:, :width], dtype), wu, np.abs(dh * g) * 12 * U + np.abs(wu) * (U * np.abs(g) + 4 * U)
           + HALF_ULP[dtype] * np.abs(wu) * 1.001 + LEAST[dtype], "dup")
    for gate_there in (True, False):  # one of them in dh's place
        e, there, _ = matrix(dh, dtype, extra, shift)
        other = Dev(np.zeros((n, width), item))
        pywelvet.rows8_swiglu_backward(DT[dtype], n, width, g8.desc, u8.desc, there,
                                       there if gate_there else other.ptr, other.ptr if gate_there else there,
                                       dh_stride=width + extra, dgate_stride=width + (extra if gate_there else 0),
                                       dup_stride=width + (0 if gate_there else extra), stream=stream)
        placed = e.get()[shift:].reshape(n, width + extra)[:, :width]
        first, second = (placed, other.get()) if gate_there else (other.get(), placed)
        assert_bit_equal(first, got_g[:, :width], "dgate in place")
        assert_bit_equal(second, got_u[:, :width], "dup in place")


def test_swiglu_gradient_against_differences(stream):
    """dgate and dup are the differences of sum(dh h) at the values the rows hold."""
    rng = np.random.default_rng(9)
    n, width = 3, 50
    gate, up, dh = rng.normal(0, 2, (n, width)), rng.normal(0, 1, (n, width)), rng.normal(0, 1, (n, width))
    (gc, gs), (uc, us) = codes_of(gate.astype(np.float32)), codes_of(up.astype(np.float32))
    g8, u8, d = Rows(n, width, 0, gc, gs), Rows(n, width, 0, uc, us), Dev(dh.astype(np.float32))
    dg, du = Dev(np.zeros((n, width), np.float32)), Dev(np.zeros((n, width), np.float32))
    pywelvet.rows8_swiglu_backward(1, n, width, g8.desc, u8.desc, d.ptr, dg.ptr, du.ptr, stream=stream)
    g, u, step = values(gc, gs), values(uc, us), 1e-5
    h = lambda g, u: act(g, "silu") * u  # noqa: E731
    # a central difference is off by step^2 / 6 of the third derivative (below 1 for silu) and by f64's rounding
    within(dg.get(), dh * (h(g + step, u) - h(g - step, u)) / (2 * step), 1e-5 * (np.abs(dh * u) + 1e-3), "dgate")
    within(du.get(), dh * (h(g, u + step) - h(g, u - step)) / (2 * step), 1e-5 * (np.abs(dh * g) + 1e-3), "dup")


def test_rows_past_32_bits(stream):
    """A row whose codes and values begin past 2^32 bytes: strides count in 64 bits."""
    from tokmem import Big
    width, stride = 100, 1 << 30
    codes, x, scales = Big(5 * stride), Big(4 * (4 * stride + width)), Dev(np.zeros(5, np.float32))
    rng = np.random.default_rng(4)
    want = rng.normal(0, 1, (5, width)).astype(np.float32)
    for r in range(5):
        x.put(4 * stride * r, want[r])
    rows = pywelvet.rows8(codes.ptr, stride, scales.ptr)
    pywelvet.rows8_store(1, 5, width, x.ptr, rows, x_stride=stride, stream=stream)
    c, s = codes_of(want)
    assert_bit_equal(scales.get(), s, "scales")
    for r in range(5):
        assert np.array_equal(codes.get(stride * r, width, np.int8), c[r])
    codes.free()
    x.free()
