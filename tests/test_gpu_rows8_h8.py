"""SwiGLU's product in 8 bits against f64, row by row.

h before its codes is within (10, of 16-bit types 10 + 2 |gate|) U of itself and
2^-148 |gate up|: two products of a sigmoid within 8 U, whose argument a 16-bit type's
is rounded in.  The scale is the largest |h| over 127: between the largest value less
what it is off and the largest that any can be.  A code is the nearest of h over that
scale, so the value it stands for is within half a step of h."""
import numpy as np
import pytest

import pywelvet
from devmem import Stream
from rows8ref import Rows, act, values
from test_gpu_rows8 import SHAPES, matrix, swiglu_in
from tokmem import DT, U, Dev, to_bits, to_f64, within

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module", autouse=True)
def device():
    pywelvet.init()


@pytest.mark.parametrize("alone", [True, False])
@pytest.mark.parametrize("dtype", DT)
@pytest.mark.parametrize("n,width", SHAPES)
def test_h8(dtype, n, width, alone):
    rng = np.random.default_rng([n, width, 3])
    gate, up = swiglu_in(rng, n, width)
    s, (g, pg, gate), (u, pu, up) = Stream(), matrix(gate, dtype), matrix(up, dtype)
    h8, others, h = Rows(n, width, 1), [Rows(n, width) for _ in range(2)], Dev(np.zeros((n, width), to_bits(np.zeros(1), dtype).dtype))
    ask = (None, None, h8.desc, None) if alone else (others[0].desc, others[1].desc, h8.desc, h.ptr)
    pywelvet.rows8_swiglu(DT[dtype], n, width, pg, pu, *ask, stream=s.h)
    s.sync()
    want = act(gate, "silu") * up
    rel = (10 + 2 * np.abs(gate) * (dtype != "float32")) * U
    assert rel.max() < 1e-4  # a bound that tells h from another row, or from zeros
    err = rel * np.abs(want) + 2.0 ** -148 * np.abs(gate * up)
    codes, scales = h8.get()
    sc, at = scales.astype(np.float64), np.abs(want).argmax(1)
    least = (np.abs(want) - err)[np.arange(n), at] / 127
    most = (np.abs(want) + err).max(1) / 127
    assert (sc >= least * (1 - 2 * U)).all() and (sc <= most * (1 + 2 * U)).all()
    assert (np.abs(codes).max(1) == 127).all()
    within(values(codes, scales), want, sc[:, None] * (0.5 + 256 * U) + err, "h's codes")
    s.close()
