"""welvet_hip_distill: loss and gradient against the definition in f64.

Bounds.  With t = (z - m) / T, an exponential's argument is rounded once
(2^-24 of |t| log2 e) after a common shift, the hardware's exponential is
within 1 ulp, and a row's sum of up to 2^17 terms in chains of at most 1024
adds with pairwise joins is within 1100 2^-24, so p is within
(2 |t| + 1200) 2^-24 of itself, q within 64 2^-24 (its exponent is formed in
f64 and rounded to f32, magnitudes up to 40) and the gradient within that of
w T (m p + q), plus half an ulp of its type.  The loss is summed in f64 from
log q in f32 (half an ulp of magnitudes up to 64) and the sum's logarithm:
within 1300 2^-24 of w T^2 sum q (1 + |log q - log p|)."""
import numpy as np
import pytest

import pywelvet
from devmem import Stream
from parity import assert_bit_equal
from tokmem import DT, U, Big, Dev, strided, to_bits, to_f64, within

pytestmark = pytest.mark.gpu
HALF_ULP = {"float32": U, "float16": 2.0 ** -11, "bfloat16": 2.0 ** -8}
LEAST = {"float32": 2.0 ** -126, "float16": 2.0 ** -24, "bfloat16": 2.0 ** -126}  # below: steps of this, or zero


@pytest.fixture(scope="module", autouse=True)
def device():
    pywelvet.init()


@pytest.fixture
def stream():
    s = Stream()
    yield s.h
    s.sync()
    s.close()


def inputs(rng, dtype, n, vocab, k, absent=0.1):
    z = rng.normal(0, 2, (n, vocab))
    k = min(k, vocab)
    index = np.stack([rng.permutation(vocab)[:k] for _ in range(n)]).astype(np.int32)
    teacher = -np.sort(-rng.normal(9, 2, (n, k)), 1).astype(np.float32)
    np.put_along_axis(z, index.astype(np.int64), teacher * 0.8, 1)
    gone = rng.random((n, k)) < absent
    index = np.where(gone & (rng.random((n, k)) < 0.5), rng.choice([-1, vocab, np.iinfo(np.int32).max], (n, k)), index)
    teacher = np.where(gone & (index >= 0) & (index < vocab), np.float32(-np.inf), teacher)
    return to_bits(z, dtype), index.astype(np.int32), teacher.astype(np.float32)


def run(stream, dtype, z, index, teacher, T=1.0, weight=None, lse=None, loss=True, grad=True, extra=0, dextra=None,
        in_place=False, shift=0):
    n, vocab = z.shape
    dextra = extra if dextra is None else dextra
    item = z.dtype.itemsize
    lead = np.zeros(shift, z.dtype)  # moves the first row off a 16-byte boundary
    d_z = Dev(np.concatenate([lead, strided(z, extra).reshape(-1)]))
    d_i, d_t = Dev(index), Dev(teacher)
    d_w, d_l = (Dev(a.astype(np.float32)) if a is not None else None for a in (weight, lse))
    out = Dev(np.full(n, 77.0, np.float32))
    sentinel = 0x4040 if z.dtype == np.uint16 else 3.0
    d_g = d_z if in_place else Dev(np.full((n, vocab + dextra), sentinel, z.dtype))
    nb = pywelvet.distill_bytes(DT[dtype], n, vocab, index.shape[1])
    ws = Dev(np.full(max(nb, 1), 0xFF, np.uint8))
    pywelvet.distill(DT[dtype], n, vocab, d_z.ptr + shift * item, index.shape[1], d_i.ptr, d_t.ptr,
                     d_loss=out.ptr if loss else None,
                     d_dlogits=(d_g.ptr + (shift * item if in_place else 0)) if grad else None, temperature=T,
                     d_weight=d_w.ptr if d_w else None, d_teacher_lse=d_l.ptr if d_l else None,
                     logits_stride=vocab + extra, dlogits_stride=vocab + dextra, ws=ws.ptr, ws_bytes=nb, stream=stream)
    ws.get()
    got = d_g.get()
    if in_place:
        got = got[shift:].reshape(n, vocab + extra)
    elif grad:
        assert (got[:, vocab:] == sentinel).all()
    return out.get() if loss else None, got[:, :vocab] if grad else None


def exact(dtype, z, index, teacher, T, weight, lse):
    """loss, gradient and their bounds."""
    n, vocab = z.shape
    z, T = to_f64(z, dtype), float(np.float32(T))
    weight = np.ones(n) if weight is None else weight.astype(np.float32).astype(np.float64)
    losses, grads, bl, bg = np.zeros(n), np.zeros((n, vocab)), np.zeros(n), np.zeros((n, vocab))
    for r in range(n):
        live = (index[r] >= 0) & (index[r] < vocab) & (teacher[r] != -np.inf)
        if weight[r] == 0 or not live.any():
            continue
        at, l = index[r][live].astype(np.int64), teacher[r][live].astype(np.float64) / T
        norm = l.max() + np.log(np.exp(l - l.max()).sum()) if lse is None else float(np.float32(lse[r]))
        logq = l - norm
        q = np.exp(logq)
        t = (z[r] - z[r].max()) / T
        logp = t - np.log(np.exp(t).sum())
        p = np.exp(logp)
        losses[r] = weight[r] * T * T * (q * (logq - logp[at])).sum()
        bl[r] = abs(weight[r]) * T * T * 1300 * U * (q * (1 + np.abs(logq - logp[at]))).sum()
        grads[r] = p * q.sum()
        size, qs = grads[r] * (2 * np.abs(np.maximum(t, -1e4)) + 1200) * U, np.zeros(vocab)
        np.add.at(qs, at, q)
        grads[r] = weight[r] * T * (grads[r] - qs)
        bg[r] = abs(weight[r]) * T * (size + 64 * U * qs) * (1 + HALF_ULP[dtype]) + HALF_ULP[dtype] * np.abs(grads[r]) \
            + LEAST[dtype]
    return losses, grads, bl, bg


def check(stream, dtype, z, index, teacher, T=1.0, weight=None, lse=None, **kw):
    loss, grad = run(stream, dtype, z, index, teacher, T, weight, lse, **kw)
    wl, wg, bl, bg = exact(dtype, z, index, teacher, T, weight, lse)
    if loss is not None:
        within(loss, wl, bl, "loss")
    if grad is not None:
        within(to_f64(grad, dtype), wg, bg, "gradient")
    return loss, grad


# n below 256 splits long rows; vocab 50257 puts rows on every alignment
SHAPES = [(1, 1, 1), (1, 8, 3), (3, 1001, 20), (2, 32000, 64), (1, 131072, 256), (5, 50257, 100), (300, 1000, 16),
          (257, 4099, 64), (260, 9000, 1024), (4, 4096, 1), (7, 70000, 1000)]


@pytest.mark.parametrize("dtype", DT)
@pytest.mark.parametrize("n,vocab,k", SHAPES)
def test_loss_and_gradient(stream, dtype, n, vocab, k):
    rng = np.random.default_rng([n, vocab, k])
    z, index, teacher = inputs(rng, dtype, n, vocab, k)
    weight = np.where(rng.random(n) < 0.2, 0, rng.uniform(0.5, 2, n))
    T = (1.0, 2.0, 0.7)[(n + k) % 3]
    loss, grad = check(stream, dtype, z, index, teacher, T, weight)
    again = run(stream, dtype, z, index, teacher, T, weight)
    assert_bit_equal(again[0], loss, "loss of a second run")
    assert_bit_equal(again[1], grad, "gradient of a second run")
    only, _ = run(stream, dtype, z, index, teacher, T, weight, grad=False)
    assert_bit_equal(only, loss, "the loss alone")
    _, only = run(stream, dtype, z, index, teacher, T, weight, loss=False)
    assert_bit_equal(only, grad, "the gradient alone")
    _, placed = run(stream, dtype, z, index, teacher, T, weight, in_place=True)
    assert_bit_equal(placed, grad, "the gradient in the logits' place")


@pytest.mark.parametrize("dtype", DT)
@pytest.mark.parametrize("n", [3, 270])
def test_teacher_s_own_sum(stream, dtype, n):
    """The teacher's log-sum given: q keeps the mass of its top entries."""
    rng = np.random.default_rng(n)
    z, index, teacher = inputs(rng, dtype, n, 5000, 30, absent=0)
    lse = np.log(np.exp(teacher.astype(np.float64) / 1.5).sum(1)) + rng.uniform(0, 1, n)
    check(stream, dtype, z, index, teacher, 1.5, None, lse)


@pytest.mark.parametrize("dtype", DT)
@pytest.mark.parametrize("extra,dextra,shift", [(8, 8, 0), (3, 3, 0), (0, 5, 0), (1, 1, 3), (4, 0, 1)])
@pytest.mark.parametrize("n", [3, 256])
def test_strides_and_alignments(stream, dtype, extra, dextra, shift, n):
    rng = np.random.default_rng(extra + dextra + n)
    z, index, teacher = inputs(rng, dtype, n, 8221, 9)
    check(stream, dtype, z, index, teacher, extra=extra, dextra=dextra, shift=shift)


@pytest.mark.parametrize("n", [2, 256])
def test_repeated_indices(stream, n):
    """Entries of one index add up, wherever they stand."""
    rng = np.random.default_rng(n)
    z, index, teacher = inputs(rng, "float32", n, 9000, 40, absent=0)
    index[:, 10:20] = index[:, :1]
    index[:, 39] = index[:, 5]
    check(stream, "float32", z, index, teacher)


@pytest.mark.parametrize("dtype", DT)
@pytest.mark.parametrize("n", [4, 256])
def test_masked_logits(stream, dtype, n):
    """Parts of the vocabulary masked with -inf and with the type's lowest value, whole rows of either."""
    rng = np.random.default_rng(5)
    z, index, teacher = inputs(rng, dtype, n, 8200, 12, absent=0)
    lowest = {"float32": np.finfo(np.float32).min, "float16": np.float16(-65504), "bfloat16": np.uint16(0xFF7F)}[dtype]
    minus = np.uint16(0xFF80) if dtype == "bfloat16" else -np.inf
    named = np.zeros(z.shape, bool)
    np.put_along_axis(named, index.astype(np.int64), True, 1)
    z[0][~named[0] & (rng.random(8200) < 0.5)] = minus
    z[1][~named[1] & (rng.random(8200) < 0.9)] = lowest
    z[2] = lowest
    check(stream, dtype, z, index, teacher, T=0.8)
    z[3] = minus  # no finite logit: p = 0, the loss infinite
    loss, grad = run(stream, dtype, z, index, teacher)
    assert np.isposinf(loss[3])
    got, q = to_f64(grad[3], dtype), np.exp(teacher[3].astype(np.float64) - teacher[3].max())
    want = np.zeros(8200)
    want[index[3]] = -q / q.sum()
    within(got, want, 64 * U * np.abs(want) + HALF_ULP[dtype] * np.abs(want) + LEAST[dtype], "gradient")
    z[3][index[3][1:]] = to_bits(np.ones(11), dtype)  # one named logit still -inf
    loss, grad = run(stream, dtype, z, index, teacher)
    assert np.isposinf(loss[3]) and np.isfinite(to_f64(grad[3], dtype)).all()


@pytest.mark.parametrize("dtype", DT)
@pytest.mark.parametrize("n", [6, 256])
@pytest.mark.parametrize("T", [2.0, 0.002])
def test_logits_of_any_magnitude(stream, dtype, n, T):
    """Rows masked throughout with the type's lowest value or a large one, and
    rows whose logits lie around a large value of either sign, also the one (2^24
    T / log2 e) where the kernels change the form of their exponents, so that a
    row has threads on both sides.  The differences to the maximum are rounded
    once more there: 3 |t| 2^-24, below the bound's 1200 where p is not zero."""
    rng = np.random.default_rng(9)
    z, index, teacher = inputs(rng, dtype, n, 8200, 12, absent=0)
    teacher = teacher * np.float32(min(T, 1.0))  # teacher / T as spread as elsewhere
    lowest = {"float32": np.finfo(np.float32).min, "float16": np.float16(-65504), "bfloat16": np.uint16(0xFF7F)}[dtype]
    top = 65504 if dtype == "float16" else 3e38
    edge = 2.0 ** 24 * T / 1.4426950408889634
    z[0] = lowest
    for row, at in ((1, -1e30), (2, 3e9), (3, edge), (4, -edge)):
        at = np.clip(at, -top, top)
        z[row] = to_bits(np.clip(at + T * rng.uniform(-8, 8, 8200), -top, top), dtype)
    check(stream, dtype, z, index, teacher, T=T)


@pytest.mark.parametrize("n", [3, 256])
def test_rows_left_out(stream, n):
    """Weight 0 or no entry: zeros, whatever the logits; NaN logits stay in their own row."""
    rng = np.random.default_rng(6)
    z, index, teacher = inputs(rng, "bfloat16", n, 8192, 8, absent=0)
    weight = np.ones(n)
    weight[0] = 0
    index[1] = -1
    z[0, ::3], z[1] = 0x7FC0, 0x7FC0
    loss, grad = check(stream, "bfloat16", z, index, teacher, 1.0, weight)
    assert loss[0] == 0 and loss[1] == 0 and not grad[:2].any()
    z[1, 5], index[1] = 0x7FC0, np.arange(8)
    loss, grad = run(stream, "bfloat16", z, index, teacher, 1.0, weight)
    assert np.isnan(loss[1]) and np.isnan(to_f64(grad[1], "bfloat16")).all() and np.isfinite(loss[2:]).all()


def test_gradient_against_differences(stream):
    """Central differences of the f32 loss along random directions: a step of
    h = 2^-6 leaves h^2 / 6 of a third derivative (below 1e-3 here) and the
    loss's rounding over 2 h."""
    rng = np.random.default_rng(7)
    z, index, teacher = inputs(rng, "float32", 2, 300, 10, absent=0)
    _, grad = run(stream, "float32", z, index, teacher, 1.3)
    h = np.float32(2.0 ** -6)
    for _ in range(4):
        v = rng.choice([-1.0, 1.0], z.shape).astype(np.float32)
        up, _ = run(stream, "float32", z + h * v, index, teacher, 1.3, grad=False)
        down, _ = run(stream, "float32", z - h * v, index, teacher, 1.3, grad=False)
        got = (up.astype(np.float64) - down) / (2 * h)
        np.testing.assert_allclose(got, (grad.astype(np.float64) * v).sum(1), atol=2e-3)


def test_rows_past_32_bits(stream):
    """Rows that start more than 2^32 bytes and 2^31 elements apart."""
    rng = np.random.default_rng(11)
    z, index, teacher = inputs(rng, "bfloat16", 2, 4000, 6)
    stride = (1 << 31) + 64
    big = Big(stride * 2 + 4000 * 2)
    try:
        big.put(0, z[0])
        big.put(stride * 2, z[1])
        d_i, d_t, out = Dev(index), Dev(teacher), Dev(np.zeros(2, np.float32))
        nb = pywelvet.distill_bytes(3, 2, 4000, 6)
        ws = Dev(np.zeros(max(nb, 1), np.uint8))
        pywelvet.distill(3, 2, 4000, big.ptr, 6, d_i.ptr, d_t.ptr, d_loss=out.ptr, d_dlogits=big.ptr,
                         logits_stride=stride, dlogits_stride=stride, ws=ws.ptr, ws_bytes=nb, stream=stream)
        loss = out.get()
        grad = np.stack([big.get(r * stride * 2, 4000, np.uint16) for r in range(2)])
    finally:
        big.free()
    wl, wg, bl, bg = exact("bfloat16", z, index, teacher, 1.0, None, None)
    within(loss, wl, bl, "loss")
    within(to_f64(grad, "bfloat16"), wg, bg, "gradient")


def test_refusals(stream):
    z, i, t, o = (Dev(np.zeros(64, a)) for a in (np.float32, np.int32, np.float32, np.float32))
    big = Dev(np.zeros(1 << 16, np.uint8))

    def call(dtype=1, n=2, vocab=16, k=3, logits=z.ptr, index=i.ptr, teacher=t.ptr, **kw):
        kw = {**dict(d_loss=o.ptr, ws=big.ptr, ws_bytes=1 << 16), **kw}
        return pywelvet.distill(dtype, n, vocab, logits, k, index, teacher, stream=stream, status=True, **kw).code
    assert call() == 0
    assert call(dtype=0) == 2
    assert call(n=0, logits=None, index=None, teacher=None) == 0
    assert call(n=-1) == 1 and call(vocab=0) == 1 and call(k=0) == 1 and call(k=1025) == 1
    assert call(logits=None) == 1 and call(index=None) == 1 and call(teacher=None) == 1 and call(d_loss=None) == 1
    for T in (0.0, -1.0, np.inf, np.nan, 1e-45):
        assert call(temperature=T) == 1
    assert call(logits_stride=15) == 1 and call(d_dlogits=o.ptr, dlogits_stride=15) == 1
    assert call(logits=z.ptr + 1) == 1
    need = pywelvet.distill_bytes(1, 2, 32000, 3)
    assert need > 0 and call(vocab=32000, ws_bytes=need - 1) == 1 and call(vocab=32000, ws=None) == 1


def test_smallest_temperature(stream):
    """Where log2(e) / T is just a float: the larger logit has all of p."""
    z, index = np.array([[0.5, 0.25, 0.5, -1.0]], np.float32), np.array([[1]], np.int32)
    _, grad = run(stream, "float32", z, index, np.zeros((1, 1), np.float32), 4.3e-39, np.array([2.0 ** 126]))
    T = float(np.float32(4.3e-39))
    within(grad, 2.0 ** 126 * T * np.array([[0.5, -1.0, 0.5, 0.0]]), 64 * U, "gradient")


@pytest.mark.parametrize("given", [False, True])
@pytest.mark.parametrize("odd", [np.nan, np.inf])
@pytest.mark.parametrize("n", [4, 256])
def test_teacher_s_values_not_finite(stream, n, odd, given):
    """A NaN or infinite teacher logit makes its row's q, so its loss and its
    whole gradient, NaN (with the teacher's own sum given, an infinite logit's
    q is infinite: the named column is NaN, the others infinite); so does a row
    without a finite student logit beside it (0 times NaN).  Other rows keep
    theirs, bit for bit."""
    rng = np.random.default_rng(12)
    z, index, teacher = inputs(rng, "float32", n, 4100, 8, absent=0)
    lse = np.full(n, 14.0) if given else None
    clean = run(stream, "float32", z, index, teacher, 1.3, None, lse)
    teacher[1, 3] = teacher[2, 0] = odd
    z[2] = -np.inf
    loss, grad = run(stream, "float32", z, index, teacher, 1.3, None, lse)
    rest = np.arange(n) % n != 1
    rest[2] = False
    assert_bit_equal(loss[rest], clean[0][rest], "loss")
    assert_bit_equal(grad[rest], clean[1][rest], "gradient")
    if given and odd == np.inf:
        named = np.zeros(4100, bool)
        named[index[1, 3]] = True
        assert np.isnan(grad[1][named]).all()
        # p below the float's range is 0, and 0 times infinity NaN
        assert (np.isposinf(grad[1][~named]) | np.isnan(grad[1][~named])).all()
    else:
        assert np.isnan(loss[1]) and np.isnan(grad[1]).all()
    assert not np.isfinite(loss[2]) and np.isnan(grad[2]).all()


@pytest.mark.parametrize("n,vocab,k", [(1, 32000, 20), (37, 9000, 1000), (170, 50257, 64), (255, 4099, 3)])
def test_workspaces_of_the_needed_size(stream, n, vocab, k):
    """The named workspace serves smaller batches too, so may be larger than
    this one needs; nothing is written past what it needs."""
    rng = np.random.default_rng(n)
    z, index, teacher = inputs(rng, "bfloat16", n, vocab, k)
    loss, grad = run(stream, "bfloat16", z, index, teacher)
    d_z, d_i, d_t, out, d_g = (Dev(a) for a in (z, index, teacher, np.zeros(n, np.float32), np.zeros_like(z)))

    def call(**ws):
        return pywelvet.distill(3, n, vocab, d_z.ptr, k, d_i.ptr, d_t.ptr, out.ptr, d_g.ptr, stream=stream,
                                status=True, **ws)
    need = int(call(ws=None, ws_bytes=0).message.split(b" bytes")[0].split()[-1])
    assert 0 < need <= pywelvet.distill_bytes(3, n, vocab, k)
    ws = Dev(np.full(need, 0xFF, np.uint8))
    assert call(ws=ws.ptr, ws_bytes=need).code == 0
    ws.get()
    assert_bit_equal(out.get(), loss, "loss")
    assert_bit_equal(d_g.get(), grad, "gradient")
