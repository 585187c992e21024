"""A row of 8-bit codes that stands for a NaN or an infinity (its scale is NaN)
poisons what reads it, whatever the activation: the layer's answers, and what the
backward takes from pre-activations kept so.  Other rows stay finite."""
import numpy as np
import pytest

import pywelvet
from devmem import Stream
from rows8ref import ACTS, Rows, codes_of
from tokmem import DT, Dev, to_bits, to_f64

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


# one launch from x, few rows, tiles with their sums split, whole ones
@pytest.mark.parametrize("n,inn,out", [(3, 60, 70), (10, 60, 70), (70, 5000, 70), (300, 60, 70)])
@pytest.mark.parametrize("name", ACTS)
@pytest.mark.parametrize("dtype", DT)
def test_answers(stream, dtype, name, n, inn, out):
    rng = np.random.default_rng(n)
    x = rng.normal(0, 1, (n, inn)).astype(np.float32)
    x[1, 5], x[n - 1, inn - 1] = np.nan, -np.inf
    bad = np.isin(np.arange(n), (1, n - 1))
    d, item = Dev(to_bits(x, dtype)), to_bits(np.zeros(1), dtype).dtype
    post = Dev(np.zeros((n, out), item))
    with pywelvet.Int8Layer(rng.normal(0, 0.1, (out, inn)), pywelvet.ACT[name], rng.normal(0, 1, out)) as layer:
        ws = Dev(np.zeros(layer.workspace_bytes(n), np.uint8))
        layer.forward(DT[dtype], n, d.ptr, d_post=post.ptr, ws=ws.ptr, ws_bytes=ws.nbytes, stream=stream)
    got = to_f64(post.get(), dtype)
    assert np.isnan(got[bad]).all() and np.isfinite(got[~bad]).all()


@pytest.mark.parametrize("n", [5, 40, 300])
@pytest.mark.parametrize("name", [a for a in ACTS if a != "linear"])
@pytest.mark.parametrize("dtype", DT)
def test_gradients(stream, dtype, name, n):
    rng = np.random.default_rng(n)
    inn, out, r = 50, 60, 3
    (xc, xs), (pc, ps) = (codes_of(rng.normal(0, 1, (n, w)).astype(np.float32)) for w in (inn, out))
    pc[r], ps[r] = 0, np.nan
    x8, pre8 = Rows(n, inn, 0, xc, xs), Rows(n, out, 0, pc, ps)
    item = to_bits(np.zeros(1), dtype).dtype
    dy = rng.normal(0, 1, (n, out))
    dy[r, ::2] = 0  # nothing times NaN is NaN
    d = Dev(to_bits(dy, dtype))
    dpre, dx, dw = Dev(np.zeros((n, out), item)), Dev(np.zeros((n, inn), item)), Dev(np.zeros((out, inn), np.float32))
    ws = Dev(np.zeros(pywelvet.rows8_backward_bytes(DT[dtype], n, inn, out), np.uint8))
    with pywelvet.Int8Layer(rng.normal(0, 0.1, (out, inn))) as layer:
        pywelvet.rows8_backward(pywelvet.ACT[name], DT[dtype], n, inn, out, d.ptr, pre=pre8.desc, x=x8.desc, layer=layer,
                                d_dpre=dpre.ptr, d_dx=dx.ptr, d_dw=dw.ptr, ws=ws.ptr, ws_bytes=ws.nbytes, stream=stream)
        for a in (dpre, dx):
            got = to_f64(a.get(), dtype)
            assert np.isnan(got[r]).all() and np.isfinite(np.delete(got, r, 0)).all()
        assert np.isnan(dw.get()).all()
