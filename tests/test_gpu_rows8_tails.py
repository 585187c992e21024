"""SiLU, sigmoid, tanh-form GELU and SwiGLU where e^x is near the smallest floats:
answers that are themselves above 2^-126 keep their digits.

Bounds, relative to the sigmoid z of argument a (x, or GELU's 2 u, whose four
roundings are 4 U |a|): 8 U for its exponential, sum and reciprocal; of 16-bit types
2 U |a| more, as the exponential's argument and log2 e are rounded; 2^-149, the last
place below 2^-126, twice; then a rounding each of x z, of up and of the type."""
import numpy as np
import pytest

import pywelvet
from devmem import Stream
from rows8ref import Rows, sigmoid, values
from test_gpu_rows8 import HALF_ULP
from tokmem import DT, U, Dev, to_bits, to_f64, within

pytestmark = pytest.mark.gpu
LAST = 2.0 ** -149
SMALL = {"float32": LAST, "float16": 2.0 ** -24, "bfloat16": 2.0 ** -133}
A = 2 * np.sqrt(2 / np.pi)


@pytest.fixture(scope="module", autouse=True)
def device():
    pywelvet.init()


@pytest.fixture
def stream():
    s = Stream()
    yield s.h
    s.sync()
    s.close()


def arg(x, name):
    return A * (x + 0.044715 * x ** 3) if name == "gelu" else x


def z_err(x, name, dtype):
    """What the sigmoid is off by, of itself."""
    a = np.abs(arg(x, name))
    return (8 + (4 * a if name == "gelu" else 0) + (2 * a if dtype != "float32" else 0)) * U


def tail(name):
    return np.linspace(-11.5, -7.5, 1001) if name == "gelu" else np.linspace(-108, -60, 1001)


@pytest.mark.parametrize("dtype", DT)
@pytest.mark.parametrize("name", ["silu", "sigmoid", "gelu"])
@pytest.mark.parametrize("n", [1, 20, 200])
def test_answers(stream, dtype, name, n):
    x, one = tail(name), np.ones((1001, 1), np.int8)
    posts = {}
    with pywelvet.Int8Layer.from_codes(one, x, pywelvet.ACT[name]) as layer:
        for t in {"float32", dtype}:
            item = to_bits(np.zeros(1), t).dtype
            d, pre, post = Dev(to_bits(np.ones((n, 1)), t)), Dev(np.zeros((n, 1001), item)), Dev(np.zeros((n, 1001), item))
            ws = Dev(np.zeros(layer.workspace_bytes(n), np.uint8))
            layer.forward(DT[t], n, d.ptr, d_pre=pre.ptr, d_post=post.ptr, ws=ws.ptr, ws_bytes=ws.nbytes, stream=stream)
            posts[t] = to_f64(post.get(), t)
            if t == "float32":
                x = pre.get().astype(np.float64)  # what the activation saw, in every type
    z = sigmoid(arg(x, name))
    size = np.ones_like(x) if name == "sigmoid" else np.abs(x)
    err = size * (z * z_err(x, name, dtype) + 2 * LAST) + U * size * z
    want = z if name == "sigmoid" else x * z
    within(posts[dtype], want, err * 1.01 + HALF_ULP[dtype] * np.abs(want) + SMALL[dtype], name)


@pytest.mark.parametrize("dtype", DT)
@pytest.mark.parametrize("name", ["silu", "sigmoid", "gelu"])
def test_answers_do_not_depend_on_their_neighbours(stream, dtype, name):
    """Values on both sides of what the 16-bit types' quick sigmoid takes, in rows that
    one value a lane, eight a lane and a split sum's join answer: the same bits."""
    x = np.random.default_rng(1).permutation(np.concatenate([tail(name), np.linspace(-3, 3, 40)]))
    got = []
    with pywelvet.Int8Layer.from_codes(np.repeat(np.ones((1041, 1), np.int8), 6000, 1), x / 6000,
                                       pywelvet.ACT[name]) as layer:
        for n in (1, 3, 20, 100, 3000):
            d, post = Dev(to_bits(np.ones((n, 6000)), dtype)), Dev(np.zeros((n, 1041), to_bits(np.zeros(1), dtype).dtype))
            ws = Dev(np.zeros(layer.workspace_bytes(n), np.uint8))
            layer.forward(DT[dtype], n, d.ptr, d_post=post.ptr, ws=ws.ptr, ws_bytes=ws.nbytes, stream=stream)
            rows = post.get()
            assert np.array_equal(rows, np.tile(rows[:1], (n, 1)))
            got.append(rows[0])
    for g in got[1:]:
        assert np.array_equal(g, got[0])


@pytest.mark.parametrize("dtype", ["float32", "bfloat16"])  # float16 holds nothing as large as these `up`
def test_swiglu(stream, dtype):
    n, width = 3, 1001
    gate = to_f64(to_bits(np.tile(np.linspace(-100, -80, width), (n, 1)), dtype), dtype)
    up = to_f64(to_bits(np.tile([[1e3], [1e20], [3e30]], (1, width)), dtype), dtype)
    g, u, h = Dev(to_bits(gate, dtype)), Dev(to_bits(up, dtype)), Dev(np.zeros((n, width), to_bits(np.zeros(1), dtype).dtype))
    h8 = Rows(n, width)
    pywelvet.rows8_swiglu(DT[dtype], n, width, g.ptr, u.ptr, h=h8.desc, d_h=h.ptr, stream=stream)
    z = sigmoid(gate)
    want = gate * z * up
    err = (np.abs(gate) * (z * (z_err(gate, "silu", dtype) + U) + 2 * LAST) * up + U * np.abs(want)) * 1.01
    within(to_f64(h.get(), dtype), want, err + HALF_ULP[dtype] * np.abs(want) + SMALL[dtype], "h")
    codes, scales = h8.get()
    top, k = np.abs(want).max(1), np.abs(want).argmax(1)
    off = err[np.arange(n), k]
    within(scales, top / 127, (off + U * top) / 127 + LAST, "h's scales")
    # half a step of the row's scale, and of it what the scale is off by
    within(values(codes, scales), want, (0.5001 * top / 127 + off + U * top)[:, None] + err, "h's codes")


@pytest.mark.parametrize("name", ["silu", "sigmoid", "tanh", "gelu"])
@pytest.mark.parametrize("n", [3, 20])
def test_derivatives(stream, name, n):
    """dpre of gradients of 1e30, so that what is below 2^-126 of act' counts."""
    out, rng = 254, np.random.default_rng(n)
    codes = np.tile(np.concatenate([np.arange(-127, 0), np.arange(1, 128)]), (n, 1))
    scales = (rng.uniform(0.9, 1, n) * (11.5 if name == "gelu" else 54 if name == "tanh" else 108) / 127).astype(np.float32)
    pre8, d = Rows(n, out, 0, codes, scales), Dev(np.full((n, out), 1e30, np.float32))
    dpre = Dev(np.zeros((n, out), np.float32))
    pywelvet.rows8_backward(pywelvet.ACT[name], 1, n, 10, out, d.ptr, pre=pre8.desc, d_dpre=dpre.ptr, stream=stream)
    dy = np.float64(np.float32(1e30))
    x = (codes.astype(np.float32) * scales[:, None]).astype(np.float64)  # rounded once, as the kernel has it
    a = 2 * x if name == "tanh" else arg(x, name)
    z, co = sigmoid(a), sigmoid(-a)
    rel, steep = z_err(x, name, "float32") + 4 * U, A * (1 + 0.134145 * x ** 2)
    if name == "silu":
        want, parts = z + x * z * co, z + np.abs(x * z * co)
        least = 2 * LAST * (1 + np.abs(x))
    elif name == "gelu":  # and six roundings of its polynomial and the constants'
        want, parts, rel = z + x * z * co * steep, z + np.abs(x * z * co * steep), rel + 8 * U
        least = 2 * LAST * (1 + np.abs(x) * steep)
    else:
        want = parts = z * co * (4 if name == "tanh" else 1)
        least = 8 * LAST
    within(dpre.get(), dy * want, dy * (parts * 2 * rel + least) * 1.01 + U * dy * np.abs(want), name)
