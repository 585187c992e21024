"""welvet_hip_adapters_*: both directions against f64 products.

Bounds.  A value of h (or g) is an f32 sum of K products in chains of at most
K / 8 + 64 additions (a wave takes an eighth of K or less, then the waves and
splits are added), so it lies within (K / 8 + 64) 2^-24 of the products'
absolute sum.  y adds at most rank + 8 further roundings and what h was off;
the factors' gradients are sums over n rows of products of h (or g).  Each is
doubled for second-order terms.  Norm-wise, random roundings stay far below
that: 1e-6 of the result's norm is asked, 3e-6 where two such sums follow one
another."""
import numpy as np
import pytest

import pywelvet
from devmem import Stream
from parity import assert_bit_equal
from tokmem import DT, U, Dev, strided, to_bits, to_f64, within

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


class Case:
    """Inputs on the host and device, and the f64 results."""

    def __init__(self, dtype, inn, out, rank, count, n, order="mixed", ranks=None, scales=True, extra=0, seed=0,
                 junk=True):
        rng = np.random.default_rng([inn, out, rank, count, n, seed])
        self.dtype, self.inn, self.out, self.rank, self.count, self.n, self.extra = dtype, inn, out, rank, count, n, extra
        self.ranks = rng.integers(0, rank + 1, count).astype(np.int32) if ranks is None else np.asarray(ranks, np.int32)
        self.scales = rng.uniform(0.5, 2, count).astype(np.float32) if scales else None
        live = np.arange(rank)[None] < self.ranks[:, None]
        down, up = rng.normal(0, 1, (count, rank, inn)), rng.normal(0, 1, (count, rank, out))
        if junk:  # what lies past an adapter's rank is not to be read
            down[~live], up[~live] = np.nan, np.inf
        self.down, self.up = to_bits(down, dtype), to_bits(up, dtype)
        ids = rng.integers(0, count, n).astype(np.int32)
        if order == "mixed":
            bad = rng.random(n) < 0.15
            ids[bad] = rng.choice([-1, count, np.iinfo(np.int32).max, np.iinfo(np.int32).min], bad.sum())
        else:
            ids = np.sort(ids)
        self.ids = ids
        self.x, self.base = rng.normal(0, 1, (n, inn)).astype(np.float32), rng.normal(0, 1, (n, out)).astype(np.float32)
        self.dy, self.dxb = rng.normal(0, 1, (n, out)).astype(np.float32), rng.normal(0, 1, (n, inn)).astype(np.float32)

    def factors(self, a):
        r = self.ranks[a]
        return to_f64(self.down[a, :r], self.dtype), to_f64(self.up[a, :r], self.dtype), \
            float(self.scales[a]) if self.scales is not None else 1.0

    def groups(self):
        for a in range(self.count):
            rows = np.nonzero(self.ids == a)[0]
            yield (a, rows, *self.factors(a))

    def on_device(self):
        self.d = {k: Dev(strided(getattr(self, k), self.extra)) for k in ("x", "base", "dy", "dxb")}
        self.d.update({k: Dev(getattr(self, k)) for k in ("down", "up", "ids", "ranks")})
        if self.scales is not None:
            self.d["scales"] = Dev(self.scales)
        self.a = pywelvet.Adapters(DT[self.dtype], self.count, self.rank, self.inn, self.out, self.d["down"].ptr,
                                   self.d["up"].ptr, d_ranks=self.d["ranks"].ptr,
                                   d_scales=self.d["scales"].ptr if self.scales is not None else None)
        nb = self.a.workspace_bytes(self.n)
        self.d["ws"] = Dev(np.full(max(nb, 1), 0xFF, np.uint8))
        self.ws = dict(ws=self.d["ws"].ptr, ws_bytes=nb)
        self.strides = dict(x_stride=self.inn + self.extra)
        return self

    def forward(self, stream, base=True, h=True):
        y, hh = Dev(np.full((self.n, self.out + self.extra), 9.0, np.float32)), Dev(
            np.full((self.n, self.rank), np.nan, np.float32))
        self.a.forward(self.d["x"].ptr, self.d["ids"].ptr, self.n, self.d["base"].ptr if base else None, y.ptr,
                       d_h=hh.ptr if h else None, x_stride=self.inn + self.extra, base_stride=self.out + self.extra,
                       y_stride=self.out + self.extra, stream=stream, **self.ws)
        got = y.get()
        self.d["ws"].get()
        assert (got[:, self.out:] == 9.0).all()
        return got[:, :self.out], hh.get()

    def backward(self, stream, h, accumulate=None, dxb=True):
        dx = Dev(np.full((self.n, self.inn + self.extra), 9.0, np.float32))
        first = np.nan if accumulate is None else accumulate
        dd = Dev(np.full((self.count, self.rank, self.inn), first, np.float32))
        du = Dev(np.full((self.count, self.rank, self.out), first, np.float32))
        dh = Dev(h)
        self.a.backward(self.d["x"].ptr, self.d["ids"].ptr, self.n, dh.ptr, self.d["dy"].ptr,
                        d_dx_base=self.d["dxb"].ptr if dxb else None, d_dx=dx.ptr, d_ddown=dd.ptr, d_dup=du.ptr,
                        accumulate=accumulate is not None, x_stride=self.inn + self.extra,
                        dy_stride=self.out + self.extra, dx_base_stride=self.inn + self.extra,
                        dx_stride=self.inn + self.extra, stream=stream, **self.ws)
        got = dx.get()
        self.d["ws"].get()
        assert (got[:, self.inn:] == 9.0).all()
        return got[:, :self.inn], dd.get(), du.get()


def norm_close(got, want, rel, what):
    d, w = np.linalg.norm(got.astype(np.float64) - want), np.linalg.norm(want)
    assert d <= rel * w + 1e-30, f"{what}: {d / max(w, 1e-30):.3e} of the norm"


def check_forward(c, y, h, base=True):
    wy, wh = (c.base if base else np.zeros_like(c.base)).astype(np.float64), np.zeros((c.n, c.rank))
    by, bh = np.abs(wy) * 4 * U, np.zeros((c.n, c.rank))
    chain = (c.inn / 8 + 64) * 2 * U
    for a, rows, down, up, s in c.groups():
        r = len(down)
        if not r or not len(rows):
            continue
        x = c.x[rows].astype(np.float64)
        wh[rows, :r], bh[rows, :r] = x @ down.T, chain * (np.abs(x) @ np.abs(down).T)
        wy[rows] += s * wh[rows, :r] @ up
        by[rows] += s * (bh[rows, :r] + (r + 8) * 2 * U * np.abs(wh[rows, :r])) @ np.abs(up) + 2 * U * np.abs(wy[rows])
    if h is not None:
        within(h, wh, bh, "h")
        norm_close(h, wh, 1e-6, "h")
    within(y, wy, by, "y")
    norm_close(y, wy, 3e-6, "y")
    return wh


def check_backward(c, dx, dd, du, h, start=0.0, dxb=True):
    wx = (c.dxb if dxb else np.zeros_like(c.dxb)).astype(np.float64)
    wd, wu = np.full((c.count, c.rank, c.inn), float(start)), np.full((c.count, c.rank, c.out), float(start))
    bx, bd, bu = np.abs(wx) * 4 * U, np.abs(wd) * 4 * U, np.abs(wu) * 4 * U
    chain = (c.out / 8 + 64) * 2 * U
    for a, rows, down, up, s in c.groups():
        r = len(down)
        if not r or not len(rows):
            continue
        x, dy, hh = c.x[rows].astype(np.float64), c.dy[rows].astype(np.float64), h[rows, :r].astype(np.float64)
        g, bg = dy @ up.T, chain * (np.abs(dy) @ np.abs(up).T)
        wx[rows] += s * g @ down
        bx[rows] += s * (bg + (r + 8) * 2 * U * np.abs(g)) @ np.abs(down) + 2 * U * np.abs(wx[rows])
        sums = (len(rows) + 16) * 2 * U
        wd[a, :r] += s * g.T @ x
        bd[a, :r] += s * (bg + sums * np.abs(g)).T @ np.abs(x) + 2 * U * np.abs(wd[a, :r])
        wu[a, :r] += s * hh.T @ dy
        bu[a, :r] += s * sums * np.abs(hh).T @ np.abs(dy) + 2 * U * np.abs(wu[a, :r])
    within(dx, wx, bx, "dx")
    within(dd, wd, bd, "ddown")
    within(du, wu, bu, "dup")
    norm_close(dx, wx, 3e-6, "dx")
    norm_close(dd, wd, 3e-6, "ddown")
    norm_close(du, wu, 1e-6, "dup")


SHAPES = [  # inn, out, rank, count, n, order, extra
    (1, 1, 1, 1, 1, "mixed", 0), (64, 64, 16, 3, 1, "sorted", 0), (1001, 777, 5, 4, 3, "mixed", 0),
    (256, 512, 8, 1, 17, "sorted", 0), (4096, 1024, 16, 48, 64, "mixed", 0), (130, 70, 33, 7, 128, "mixed", 2),
    (260, 196, 20, 9, 129, "mixed", 4), (2048, 512, 64, 4, 300, "sorted", 0), (96, 1028, 100, 3, 513, "mixed", 0),
    (64, 68, 4, 200, 1500, "mixed", 0), (513, 257, 16, 2, 1100, "sorted", 1), (320, 64, 32, 5, 5000, "mixed", 0),
    (8, 8, 256, 2, 40, "mixed", 0)]


@pytest.mark.parametrize("dtype", DT)
@pytest.mark.parametrize("shape", SHAPES, ids=lambda s: "-".join(map(str, s)))
def test_forward_and_backward(stream, dtype, shape):
    inn, out, rank, count, n, order, extra = shape
    c = Case(dtype, inn, out, rank, count, n, order, extra=extra).on_device()
    y, h = c.forward(stream)
    check_forward(c, y, h)
    dx, dd, du = c.backward(stream, h)
    check_backward(c, dx, dd, du, h)
    y2, h2 = c.forward(stream)
    again = c.backward(stream, h)
    for a, b, what in ((y, y2, "y"), (h, h2, "h"), *zip((dx, dd, du), again, ("dx", "ddown", "dup"))):
        assert_bit_equal(b, a, f"{what} of a second run")


@pytest.mark.parametrize("n", [5, 200])
def test_without_bases_scales_or_h(stream, n):
    c = Case("float32", 128, 96, 16, 3, n, scales=False).on_device()
    y, _ = c.forward(stream, base=False, h=False)
    h = check_forward(c, y, None, base=False).astype(np.float32)
    dx, dd, du = c.backward(stream, h, dxb=False)
    check_backward(c, dx, dd, du, h, dxb=False)


@pytest.mark.parametrize("n", [40, 700])
def test_accumulates(stream, n):
    c = Case("bfloat16", 132, 260, 12, 6, n).on_device()
    _, h = c.forward(stream)
    dx, dd, du = c.backward(stream, h, accumulate=0.75)
    check_backward(c, dx, dd, du, h, start=0.75)


@pytest.mark.parametrize("n", [9, 600])
def test_rows_without_an_adapter(stream, n):
    """No row with an adapter: the base comes back bit for bit, gradients are zero."""
    c = Case("float16", 72, 100, 8, 3, n)
    c.ids[:] = np.where(np.arange(n) % 2, -1, 3)
    c.on_device()
    y, h = c.forward(stream)
    assert_bit_equal(y, c.base, "y")
    assert_bit_equal(h, np.zeros((n, 8), np.float32), "h")
    dx, dd, du = c.backward(stream, h)
    assert_bit_equal(dx, c.dxb, "dx")
    assert not dd.any() and not du.any()
    _, dd, du = c.backward(stream, h, accumulate=2.0)
    assert (dd == 2.0).all() and (du == 2.0).all()


def test_no_rows(stream):
    c = Case("float32", 20, 24, 4, 2, 1).on_device()
    dd, du = Dev(np.full((2, 4, 20), np.nan, np.float32)), Dev(np.full((2, 4, 24), np.nan, np.float32))
    c.a.backward(None, None, 0, None, None, d_ddown=dd.ptr, d_dup=du.ptr, stream=stream)
    assert not dd.get().any() and not du.get().any()
    c.a.forward(None, None, 0, None, None, stream=stream)


@pytest.mark.parametrize("n", [24, 400])
def test_tenants_do_not_meet(stream, n):
    """NaN and infinities in one adapter's factors and rows leave every other row and gradient as it was."""
    clean, dirty = (Case("bfloat16", 64, 128, 16, 4, n, ranks=[16, 16, 16, 16], seed=2, junk=False) for _ in range(2))
    bad = dirty.ids == 1
    dirty.down[1], dirty.up[1] = 0x7FC0, 0x7F80
    dirty.x[bad], dirty.dy[bad] = np.nan, np.inf
    got = []
    for c in (clean, dirty):
        c.on_device()
        y, h = c.forward(stream)
        got.append((y, h, *c.backward(stream, h)))
    rest = ~(clean.ids == 1)
    assert rest.any() and bad.any()
    for i, what in enumerate(("y", "h", "dx")):
        assert_bit_equal(got[1][i][rest], got[0][i][rest], what)
        assert not np.isfinite(got[1][i][bad]).all()
    for i, what in ((3, "ddown"), (4, "dup")):
        assert_bit_equal(got[1][i][[0, 2, 3]], got[0][i][[0, 2, 3]], what)


def test_in_place(stream):
    """y over base and dx over dx_base: the same bits."""
    for n in (6, 300):
        c = Case("float32", 100, 84, 8, 3, n).on_device()
        y, h = c.forward(stream)
        dx, _, _ = c.backward(stream, h)
        yb, xb, dh = Dev(c.base), Dev(c.dxb), Dev(h)
        c.a.forward(c.d["x"].ptr, c.d["ids"].ptr, n, yb.ptr, yb.ptr, stream=stream, **c.ws)
        assert_bit_equal(yb.get(), y, "y")
        c.a.backward(None, c.d["ids"].ptr, n, None, c.d["dy"].ptr, d_dx_base=xb.ptr, d_dx=xb.ptr, stream=stream, **c.ws)
        assert_bit_equal(xb.get(), dx, "dx")


def test_gradients_against_differences(stream):
    """L = <dy, y> is linear in x, in the down and in the up factors, so its
    difference over a whole step is the gradient's product with the step, up
    to f32 roundings of y (1e-5 of the products' absolute sum)."""
    c = Case("float32", 48, 40, 8, 3, 150, ranks=[8, 5, 0], seed=4, junk=False).on_device()
    y0, h = c.forward(stream)
    dx, dd, du = c.backward(stream, h, dxb=False)
    rng = np.random.default_rng(1)
    for name, grad in (("x", dx), ("down", dd), ("up", du)):
        old = getattr(c, name)
        step = rng.normal(0, 1, old.shape).astype(np.float32)
        setattr(c, name, old + step)
        y1, _ = c.on_device().forward(stream)
        moved = (old + step).astype(np.float64) - old
        setattr(c, name, old)
        prod = c.dy * (y1.astype(np.float64) - y0)
        assert abs(prod.sum() - (grad * moved).sum()) <= 1e-5 * np.abs(prod).sum(), name


def test_a_dense_layer_s_adapters(stream):
    """Beside a mounted FP8 layer: its Linear output plus the adapters', as the
    f64 product of the decoded weights and the merged update has it."""
    rng = np.random.default_rng(8)
    inn, out, n = 256, 192, 6
    c = Case("bfloat16", inn, out, 8, 2, n, seed=6)
    W = rng.normal(0, 0.5, (out, inn)).astype(np.float32)
    with pywelvet.Session(W, n, dtype=4) as s:
        Wd = s.export_f32().astype(np.float64)
        x = Dev(c.x)
        pre, post = (Dev(np.zeros((n, out), np.float32)) for _ in range(2))
        s.forward_device(x.ptr, pre.ptr, post.ptr, stream)
        c.on_device()
        c.a.forward(x.ptr, c.d["ids"].ptr, n, post.ptr, post.ptr, stream=stream, **c.ws)
        got = post.get()
    want = c.x.astype(np.float64) @ Wd.T
    for a, rows, down, up, scale in c.groups():
        want[rows] += scale * (c.x[rows].astype(np.float64) @ down.T) @ up
    assert np.abs(got - want).max() <= 1e-5 * np.abs(want).max()


def test_refusals(stream):
    c = Case("float32", 16, 12, 4, 2, 200).on_device()
    y = Dev(np.zeros((200, 12), np.float32))

    def fwd(x=c.d["x"].ptr, ids=c.d["ids"].ptr, n=200, y=y.ptr, a=c.a, **kw):
        kw = {**c.ws, **kw}
        return a.forward(x, ids, n, c.d["base"].ptr, y, stream=stream, status=True, **kw).code

    def stack(dtype=1, count=2, rank=4, inn=16, out=12, down=c.d["down"].ptr):
        return pywelvet.Adapters(dtype, count, rank, inn, out, down, c.d["up"].ptr)
    assert fwd() == 0
    assert fwd(a=stack(dtype=4)) == 2
    for a in (stack(count=0), stack(rank=0), stack(rank=257), stack(inn=0), stack(out=-1), stack(down=None),
              stack(down=c.d["down"].ptr + 2)):
        assert fwd(a=a) == 1
    assert fwd(x=None) == 1 and fwd(ids=None) == 1 and fwd(y=None) == 1 and fwd(n=-1) == 1
    assert fwd(x_stride=15) == 1 and fwd(y_stride=11) == 1 and fwd(base_stride=11) == 1
    assert fwd(ws_bytes=0) == 1 and fwd(ws=None) == 1 and fwd(y=y.ptr + 1) == 1

    def bwd(**kw):
        kw = {**c.ws, **kw}
        return c.a.backward(c.d["x"].ptr, c.d["ids"].ptr, 200, y.ptr, c.d["dy"].ptr, stream=stream, status=True, **kw).code
    dx = Dev(np.zeros((200, 16), np.float32))
    assert bwd() == 1  # no output
    assert bwd(d_dx=dx.ptr) == 0
    assert bwd(d_dx=dx.ptr, dx_stride=15) == 1 and bwd(d_dx=dx.ptr, dy_stride=11) == 1
    assert bwd(d_dx=dx.ptr, ws_bytes=16) == 1
    with pytest.raises(pywelvet.WelvetError):
        stack(rank=0).workspace_bytes(4)


def needed(call):
    """The bytes that a refused call names, 0 where it takes none."""
    st = call(ws=None, ws_bytes=0)
    return int(st.message.split(b" bytes")[0].split()[-1]) if st.code else 0


@pytest.mark.parametrize("dtype,inn,out,rank,count,n", [
    ("float32", 1001, 777, 5, 4, 3), ("bfloat16", 4096, 1024, 16, 8, 64), ("float16", 2048, 512, 64, 4, 300),
    ("bfloat16", 130, 3000, 33, 7, 2100), ("float32", 320, 64, 32, 5, 5000), ("float16", 513, 257, 16, 2, 2049)])
def test_workspaces_of_the_needed_size(stream, dtype, inn, out, rank, count, n):
    """The named workspace serves smaller batches too, so may be larger than
    this one needs; nothing is written past what it needs."""
    c = Case(dtype, inn, out, rank, count, n).on_device()
    y, h = c.forward(stream)
    dx, dd, du = c.backward(stream, h)
    o = [Dev(np.full(a.shape, np.nan, np.float32)) for a in (y, h, dx, dd, du)]
    dh = Dev(h)
    calls = (lambda **ws: c.a.forward(c.d["x"].ptr, c.d["ids"].ptr, n, c.d["base"].ptr, o[0].ptr, o[1].ptr,
                                      stream=stream, status=True, **ws),
             lambda **ws: c.a.backward(c.d["x"].ptr, c.d["ids"].ptr, n, dh.ptr, c.d["dy"].ptr, c.d["dxb"].ptr, o[2].ptr,
                                       o[3].ptr, o[4].ptr, stream=stream, status=True, **ws))
    for call in calls:
        need = needed(call)
        assert need <= c.a.workspace_bytes(n)
        ws = Dev(np.full(need, 0xFF, np.uint8))
        assert call(ws=ws.ptr, ws_bytes=need).code == 0
        ws.get()
    for got, want, what in zip(o, (y, h, dx, dd, du), ("y", "h", "dx", "ddown", "dup")):
        assert_bit_equal(got.get(), want, what)


@pytest.mark.parametrize("n", [40, 2200])
@pytest.mark.parametrize("rank", [12, 20, 64])
@pytest.mark.parametrize("dtype,power", [("float32", 100), ("float16", 12), ("bfloat16", 12), ("bfloat16", 22),
                                         ("bfloat16", 100)])
def test_small_activations(stream, dtype, power, rank, n):
    """Activations and gradients near the type's least normal values (some
    below, whose last bits count) through large factors: as near, norm-wise, as
    ordinary ones."""
    c = Case(dtype, 200, 640, rank, 2, n, ranks=[rank, rank - 3], scales=False, junk=False)
    factor = 2.0 ** power
    for name in ("down", "up"):
        setattr(c, name, to_bits(to_f64(getattr(c, name), dtype) * factor, dtype))
    c.x, c.dy = c.x * np.float32(1e-37), c.dy * np.float32(1e-37)
    c.on_device()
    _, h = c.forward(stream, base=False)
    down = c.down
    c.down = to_bits(to_f64(down, dtype) / factor, dtype)  # dx of the size of g
    c.on_device()
    dx, _, _ = c.backward(stream, h, dxb=False)
    far = 2.0 ** 100
    for a, rows, back, up, s in c.groups():
        want = far * (c.x[rows].astype(np.float64) @ to_f64(down[a, :len(back)], dtype).T)
        norm_close(far * h[rows, :len(back)].astype(np.float64), want, 1e-6, "h")
        want = far * (c.dy[rows].astype(np.float64) @ up.T) @ back
        norm_close(far * dx[rows].astype(np.float64), want, 3e-6, "dx")


@pytest.mark.parametrize("dtype", ["bfloat16", "float16"])
def test_dx_of_sorted_rows_does_not_depend_on_dup(stream, dtype):
    """dx alone has the bits that it has beside dup, also where the gradients
    hold values whose products are looked at again."""
    c = Case(dtype, 140, 264, 12, 5, 2201)
    c.dy[np.random.default_rng(3).random(c.dy.shape) < 0.01] *= np.float32(1e-37)
    c.on_device()
    _, h = c.forward(stream)
    dx, _, _ = c.backward(stream, h)
    out = Dev(np.full(dx.shape, np.nan, np.float32))
    c.a.backward(None, c.d["ids"].ptr, c.n, None, c.d["dy"].ptr, d_dx_base=c.d["dxb"].ptr, d_dx=out.ptr, stream=stream,
                 **c.ws)
    assert_bit_equal(out.get(), dx, "dx")
