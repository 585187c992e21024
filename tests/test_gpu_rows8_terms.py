"""What a product of the backward from 8-bit rows keeps of its terms, in every type.

Channels come in threes with one row of codes, gradients d, d and -d, and scales
a, b and a + b, all exact in f32: every sum dx is 0, and what a kernel answers is its
terms' rounding.  The bound is the one of the backward's other tests: 2^-22 of a term
for its two f16 parts, 2^-39 of the token's largest |dy| scale times 1.3 for their last
place, and (2 K + 12) U of the terms' magnitudes for the f32 sum of two parts of K
terms and a term's own roundings."""
import numpy as np
import pytest

import pywelvet
from devmem import Stream
from rows8ref import Rows, codes_of
from tokmem import DT, U, Dev, to_bits, to_f64, within

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module", autouse=True)
def device():
    pywelvet.init()


# few rows, tiles of 64 and of 128 rows with split sums and without, and 256 x 256 tiles
@pytest.mark.parametrize("dtype", DT)
@pytest.mark.parametrize("with_dw", [False, True])
@pytest.mark.parametrize("n,inn,out", [(5, 130, 63), (20, 130, 63), (60, 200, 1701), (200, 130, 63), (200, 200, 1701),
                                       (4200, 4200, 255)])
def test_dx_of_terms_that_cancel(dtype, with_dw, n, inn, out):
    rng = np.random.default_rng([n, inn, out])
    a, b = (1 + rng.integers(0, 2 ** 20, out // 3) * 2.0 ** -20 for _ in range(2))
    scales = np.stack([a, b, a + b], 1).reshape(-1).astype(np.float32)
    assert np.array_equal(scales.reshape(-1, 3)[:, 2].astype(np.float64), a + b)
    codes = np.repeat(rng.integers(-127, 128, (out // 3, inn)).astype(np.int8), 3, axis=0)
    d = to_f64(to_bits(rng.normal(0, 1e-2, (n, out // 3)), dtype), dtype)
    dy = np.stack([d, d, -d], 2).reshape(n, out)
    item = to_bits(np.zeros(1), dtype).dtype
    s, grad, dx = Stream(), Dev(to_bits(dy, dtype)), Dev(np.full((n, inn), 5, item))
    xc, xs = codes_of(rng.normal(0, 1, (n, inn)).astype(np.float32))
    rows, dw = Rows(n, inn, 0, xc, xs), Dev(np.zeros((out, inn), np.float32))
    ws = Dev(np.full(pywelvet.rows8_backward_bytes(DT[dtype], n, inn, out), 0xFF, np.uint8))
    with pywelvet.Int8Layer.from_codes(codes, scales) as layer:
        pywelvet.rows8_backward(-1, DT[dtype], n, inn, out, grad.ptr, x=rows.desc if with_dw else None, layer=layer,
                                d_dx=dx.ptr, d_dw=dw.ptr if with_dw else None, ws=ws.ptr, ws_bytes=ws.nbytes, stream=s.h)
        s.sync()
    ws.get()
    terms, w = np.abs(dy * scales), np.abs(codes.astype(np.float64))
    least = 2.0 ** -39 * 1.3 * terms.max(1, initial=0)
    bound = terms @ w * (2.0 ** -22 + (2 * out + 12) * U) + least[:, None] * w.sum(0)
    smallest = {"float32": 2.0 ** -126, "float16": 2.0 ** -24, "bfloat16": 2.0 ** -126}[dtype]
    # what is left is rounded to the type: half a step of it, at most the bound's own half
    half = {"float32": U, "float16": 2.0 ** -11, "bfloat16": 2.0 ** -8}[dtype]
    within(to_f64(dx.get(), dtype), np.zeros((n, inn)), bound * (1 + half) + smallest, "dx")
    s.close()
