"""dw and dx have the same bits whichever other outputs are asked for, where the tiles
that take them differ: dw alone in 256 x 256 tiles and beside dx in 128 x 128, dx of few
rows in 64 x 128 with its sum split and beside dw in 128 x 128."""
import numpy as np
import pytest

import pywelvet
from devmem import Stream
from parity import assert_bit_equal
from test_gpu_rows8_backward import Case
from tokmem import DT

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module", autouse=True)
def device():
    pywelvet.init()


@pytest.mark.parametrize("dtype", DT)
@pytest.mark.parametrize("n,inn,out", [(256, 4096, 4096), (300, 4100, 4090), (64, 4096, 4096)])
def test_the_same_bits_alone(dtype, n, inn, out):
    s, case = Stream(), Case(dtype, n, inn, out, "gelu", 11)
    base = np.random.default_rng(3).normal(0, 1, (out, inn)).astype(np.float32)
    dpre, dx, dw = case.run(s.h)
    assert_bit_equal(case.run(s.h, dx=False)[2], dw, "dw without dx")
    assert_bit_equal(case.run(s.h, dx=False, dpre=False)[2], dw, "dw alone")
    assert_bit_equal(case.run(s.h, dw=False)[1], dx, "dx without dw")
    both, alone = case.run(s.h, base=base)[2], case.run(s.h, base=base, dx=False, dpre=False)[2]
    assert_bit_equal(alone, both, "dw added to")
    s.sync()
    s.close()
