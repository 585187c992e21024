"""Results in their inputs' place, where the 8-bit operators allow it, have the bits
that they have elsewhere."""
import numpy as np
import pytest

import pywelvet
from devmem import Stream
from parity import assert_bit_equal
from test_gpu_rows8 import matrix, swiglu_in
from tokmem import DT, Dev, to_bits

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


@pytest.mark.parametrize("dtype", DT)
@pytest.mark.parametrize("n,width", [(3, 7), (100, 777), (3, 1025), (2, 8193), (2, 33001)])
@pytest.mark.parametrize("place", ["gate", "up"])
def test_swiglu(stream, dtype, n, width, place):
    gate, up = swiglu_in(np.random.default_rng([n, width]), n, width)
    (g, pg, _), (u, pu, _) = matrix(gate, dtype, 1), matrix(up, dtype, 2)
    h = Dev(np.zeros((n, width), to_bits(np.zeros(1), dtype).dtype))
    kw = dict(gate_stride=width + 1, up_stride=width + 2, stream=stream)
    pywelvet.rows8_swiglu(DT[dtype], n, width, pg, pu, d_h=h.ptr, **kw)
    want, where = h.get(), (g, pg, 1) if place == "gate" else (u, pu, 2)
    pywelvet.rows8_swiglu(DT[dtype], n, width, pg, pu, d_h=where[1], h_stride=width + where[2], **kw)
    assert_bit_equal(where[0].get().reshape(n, width + where[2])[:, :width], want, "h")


# by one launch from x and by the few-row kernel, where x is free and where it is not,
# and in tiles; widths of one and of several blocks
@pytest.mark.parametrize("dtype", DT)
@pytest.mark.parametrize("n,inn,out", [(1, 1000, 1000), (3, 520, 1040), (4, 4096, 4096), (2, 2000, 40), (9, 300, 300),
                                       (100, 700, 700)])
@pytest.mark.parametrize("place", ["pre", "post"])
def test_a_layer(stream, dtype, n, inn, out, place):
    """pre or post where x is, and beginning inside it."""
    rng = np.random.default_rng([n, inn, out])
    stride = max(inn, out) + 5
    x = np.zeros((n, stride))
    x[:, :inn] = rng.normal(0, 1, (n, inn))
    bits = to_bits(x, dtype)
    room = np.zeros((n + 1) * stride, bits.dtype)
    room[:n * stride] = bits.reshape(-1)
    with pywelvet.Int8Layer(rng.normal(0, inn ** -0.5, (out, inn)), pywelvet.ACT["silu"], rng.normal(0, 1, out)) as layer:
        ws = Dev(np.zeros(layer.workspace_bytes(n), np.uint8))
        on = dict(x_stride=stride, pre_stride=stride, post_stride=stride, ws=ws.ptr, ws_bytes=ws.nbytes, stream=stream)
        d, pre, post = Dev(room), Dev(room), Dev(room)
        layer.forward(DT[dtype], n, d.ptr, d_pre=pre.ptr, d_post=post.ptr, **on)
        want = [a.get()[:n * stride].reshape(n, stride)[:, :out] for a in (pre, post)]
        for shift in (0, min(inn, 600) - 1):
            for both in (True, False):
                d, other = Dev(room), Dev(room)
                at = d.ptr + shift * bits.dtype.itemsize
                a, b = (at, other.ptr if both else None) if place == "pre" else (other.ptr if both else None, at)
                layer.forward(DT[dtype], n, d.ptr, d_pre=a, d_post=b, **on)
                ws.get()
                k = place == "post"
                assert_bit_equal(d.get()[shift:shift + n * stride].reshape(n, stride)[:, :out], want[k], place)
                if both:
                    assert_bit_equal(other.get()[:n * stride].reshape(n, stride)[:, :out], want[not k], "the other")
