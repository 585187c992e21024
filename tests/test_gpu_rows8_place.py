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
