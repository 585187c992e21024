"""A Dense session that keeps its activations in 8 bits: its own forward on device
pointers, x and pre stored as rows, dpre and dw from them without an integer layer, and
dx by a session of the transposed weights.

dpre is within 64 U + U |pre| of |dy| of its formula at the values held, dw within
2^-22 + (2 n + 12) U of its terms' magnitudes and 2^-39 of the channel's largest (two f16
parts); dx is a Dense forward, 1e-5 of the terms' magnitudes."""
import numpy as np
import pytest

import pywelvet
from devmem import Stream
from rows8ref import PRIME_ERR, Rows, act_prime, codes_of, values
from tokmem import U, Dev, within

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module", autouse=True)
def device():
    pywelvet.init()


@pytest.mark.parametrize("dtype", [1, 3, 4, 13, 26])
@pytest.mark.parametrize("n", [4, 50, 300])
def test_a_dense_step(dtype, n):
    rng = np.random.default_rng([dtype, n])
    inn, out, s = 160, 96, Stream()
    x, dy = rng.normal(0, 1, (n, inn)).astype(np.float32), rng.normal(0, 1e-2, (n, out)).astype(np.float32)
    with pywelvet.Session(rng.normal(0, 0.1, (out, inn)), n, pywelvet.ACT["silu"], dtype, rng.normal(0, 1, out)) as layer:
        W = layer.export_f32()
        with pywelvet.Session(np.ascontiguousarray(W.T), n, -1, 1) as back:
            d, g, pre, post, dpre, dx, spare, dw = (Dev(a) for a in (
                x, dy, *(np.zeros(sh, np.float32) for sh in ((n, out), (n, out), (n, out), (n, inn), (n, inn), (out, inn)))))
            x8, pre8 = Rows(n, inn), Rows(n, out)
            layer.forward_device(d.ptr, pre.ptr, post.ptr, s.h)
            pywelvet.rows8_store(1, n, inn, d.ptr, x8.desc, stream=s.h)
            pywelvet.rows8_store(1, n, out, pre.ptr, pre8.desc, stream=s.h)
            ws = Dev(np.zeros(pywelvet.rows8_backward_bytes(1, n, inn, out), np.uint8))
            pywelvet.rows8_backward(pywelvet.ACT["silu"], 1, n, inn, out, g.ptr, pre=pre8.desc, x=x8.desc, d_dpre=dpre.ptr,
                                    d_dw=dw.ptr, ws=ws.ptr, ws_bytes=ws.nbytes, stream=s.h)
            back.forward_device(dpre.ptr, dx.ptr, spare.ptr, s.h)
            s.sync()
            ws.get()
    (xc, xs), (pc, ps) = x8.get(), pre8.get()
    for got, a in (((xc, xs), x), ((pc, ps), pre.get())):
        want = codes_of(a)
        assert np.array_equal(got[0], want[0]) and np.array_equal(got[1], want[1])
    p, xv = values(pc, ps), values(xc, xs)
    want = dy * act_prime(p, "silu")
    err = np.abs(dy) * (PRIME_ERR + U * np.abs(p)) + 4 * U * np.abs(want)
    within(dpre.get(), want, err, "dpre")
    least = 2.0 ** -39 * 1.3 * np.abs(dy * xs[:, None]).max(0).astype(np.float64)
    within(dw.get(), want.T @ xv, err.T @ np.abs(xv) + np.abs(want).T @ np.abs(xv) * (2.0 ** -22 + (2 * n + 12) * U)
           + least[:, None] * np.abs(xc).sum(0), "dw")
    got = dpre.get().astype(np.float64)
    within(dx.get(), got @ W, 1e-5 * np.abs(got) @ np.abs(W) + 1e-30, "dx")
    s.close()
