"""Terms far below the largest of their channel or token in the backward from 8-bit
rows: the one power of two that both share leaves them f16 parts near and below its
smallest normal, which keep 2^-39 of the bound as documented.

One token (dw) or channel (dx) is 2^20 to 2^36 above the others, and its codes are 0
but in one column, so that every other column's sum is of the small terms alone.  The
bound is the documented one: 2^-22 of a term, 2^-39 of 1.3 times the largest for each,
(2 K + 12) U of the terms' magnitudes."""
import numpy as np
import pytest

import pywelvet
from devmem import Stream
from rows8ref import Rows
from tokmem import DT, U, Dev, to_bits, to_f64, within

pytestmark = pytest.mark.gpu
SMALLEST = {"float32": 2.0 ** -149, "float16": 2.0 ** -24, "bfloat16": 2.0 ** -133}
HALF = {"float32": U, "float16": 2.0 ** -11, "bfloat16": 2.0 ** -8}


@pytest.fixture(scope="module", autouse=True)
def device():
    pywelvet.init()


@pytest.mark.parametrize("dtype", DT)
@pytest.mark.parametrize("above", [20, 28, 36])
@pytest.mark.parametrize("n,inn,out", [(20, 70, 90), (100, 70, 90), (300, 200, 130), (40, 64, 2600)])
def test_small_terms(dtype, above, n, inn, out):
    rng = np.random.default_rng([n, inn, out, above])
    s = Stream()
    xc, wc = rng.integers(-127, 128, (n, inn)), rng.integers(-127, 128, (out, inn))
    xs, ws = (rng.uniform(0.5, 1, k).astype(np.float32) * np.float32(2.0 ** -above) for k in (n, out))
    xc[3], wc[5] = 0, 0
    xc[3, 0] = wc[5, 0] = 127
    xs[3] = ws[5] = 1
    dy = to_f64(to_bits(rng.normal(0, 1, (n, out)), dtype), dtype)
    x8, d = Rows(n, inn, 0, xc, xs), Dev(to_bits(dy, dtype))
    dx, dw = Dev(np.zeros((n, inn), to_bits(np.zeros(1), dtype).dtype)), Dev(np.zeros((out, inn), np.float32))
    work = Dev(np.zeros(pywelvet.rows8_backward_bytes(DT[dtype], n, inn, out), np.uint8))
    with pywelvet.Int8Layer.from_codes(wc, ws) as layer:
        pywelvet.rows8_backward(-1, DT[dtype], n, inn, out, d.ptr, x=x8.desc, layer=layer, d_dx=dx.ptr, d_dw=dw.ptr,
                                ws=work.ptr, ws_bytes=work.nbytes, stream=s.h)
        s.sync()
    work.get()
    tw, tx = dy * xs[:, None].astype(np.float64), dy * ws.astype(np.float64)
    aw, ax = np.abs(xc).astype(np.float64), np.abs(wc).astype(np.float64)
    least_w, least_x = (2.0 ** -39 * 1.3 * np.abs(t).max(k) for t, k in ((tw, 0), (tx, 1)))
    want = tw.T @ xc
    within(dw.get(), want, np.abs(tw).T @ aw * (2.0 ** -22 + (2 * n + 12) * U) + least_w[:, None] * aw.sum(0)
           + U * np.abs(want), "dw")
    want = tx @ wc
    bound = np.abs(tx) @ ax * (2.0 ** -22 + (2 * out + 12) * U) + least_x[:, None] * ax.sum(0)
    within(to_f64(dx.get(), dtype), want, bound * 1.01 + HALF[dtype] * np.abs(want) + SMALLEST[dtype], "dx")
    s.close()
