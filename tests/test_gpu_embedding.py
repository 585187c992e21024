"""welvet_hip_embedding_*: lookups bit for bit, gradients against f64 sums.

The lookup rounds once (scale times an exact value), so it is compared bit for
bit.  A gradient element is an f32 sum of m values times the scale: each value
passes at most m additions and one product, so it lies within (m + 1) 2^-24 of
the values' absolute sum (twice that is allowed for second-order terms)."""
import numpy as np
import pytest

import pywelvet
from devmem import Stream
from oracle import DTYPE_NAMES
from parity import assert_bit_equal
from tokmem import DT, U, Big, Dev, strided, to_bits, to_f64, within

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


def tokens_of(rng, vocab, n, pad=0.1):
    """Skewed tokens, a tenth padding of several kinds."""
    t = np.minimum(np.exp(rng.uniform(0, np.log(vocab + 1), n)).astype(np.int64) - 1, vocab - 1)
    t = rng.permutation(vocab)[t].astype(np.int32)
    bad = rng.random(n) < pad
    t[bad] = rng.choice([-1, vocab, np.iinfo(np.int32).min, np.iinfo(np.int32).max], bad.sum())
    return t


@pytest.mark.parametrize("dtype", DT)
@pytest.mark.parametrize("vocab,dim,n,extra,scale", [
    (1, 1, 1, 0, 1.0), (50, 64, 1, 0, 8.0), (1000, 777, 33, 0, 1.5), (1000, 1024, 100, 4, 32.0),
    (37, 4100, 5, 3, -0.5), (300, 256, 20001, 0, 16.0), (300, 333, 9001, 1, 2.0)])
def test_lookup(stream, dtype, vocab, dim, n, extra, scale):
    rng = np.random.default_rng(vocab * dim + n)
    table = to_bits(rng.normal(0, 1, (vocab, dim)), dtype)
    tok = tokens_of(rng, vocab, n)
    d_t, d_k = Dev(strided(table, extra)), Dev(tok)
    out = Dev(np.full((n, dim + extra), 7.0, np.float32))
    pywelvet.embedding_forward(DT[dtype], vocab, dim, d_t.ptr, d_k.ptr, n, out.ptr, scale=scale,
                               table_stride=dim + extra, out_stride=dim + extra, stream=stream)
    got = out.get()
    ok = (tok >= 0) & (tok < vocab)
    want = np.zeros((n, dim), np.float32)
    want[ok] = to_f64(table, dtype)[tok[ok]].astype(np.float32) * np.float32(scale)
    assert_bit_equal(got[:, :dim], want, "rows")
    assert (got[:, dim:] == 7.0).all()


def test_lookup_special_values_and_unaligned_pointers(stream):
    """NaN, infinities, subnormals and -0 come through; a table that starts
    off a 16-byte boundary takes the element-wise path with the same bits."""
    for dtype in DT:
        row = to_bits(np.array([[np.nan, np.inf, -np.inf, -0.0, 1e-40, -6e-8, 65504, 1]], np.float32), dtype)
        flat = np.concatenate([np.zeros(1, row.dtype), row.reshape(-1)])
        d_t, d_k = Dev(flat), Dev(np.zeros(1, np.int32))
        out = Dev(np.zeros(9, np.float32))
        pywelvet.embedding_forward(DT[dtype], 1, 8, d_t.ptr + row.itemsize, d_k.ptr, 1, out.ptr + 4, stream=stream)
        got = out.get()[1:]
        want = to_f64(row, dtype)[0].astype(np.float32)
        assert np.isnan(got[0]) and np.isnan(want[0])
        assert_bit_equal(got[1:], want[1:], dtype)


def test_lookup_past_32_bits(stream):
    """A table of more than 2^32 bytes and 2^31 elements: its last rows."""
    vocab, dim = 270_000, 8192
    table = Big(vocab * dim * 2)
    try:
        rng = np.random.default_rng(3)
        rows = to_bits(rng.normal(0, 1, (2, dim)), "bfloat16")
        table.put((vocab - 2) * dim * 2, rows)
        d_k, out = Dev(np.array([vocab - 1, vocab - 2], np.int32)), Dev(np.zeros((2, dim), np.float32))
        pywelvet.embedding_forward(3, vocab, dim, table.ptr, d_k.ptr, 2, out.ptr, stream=stream)
        assert_bit_equal(out.get(), to_f64(rows[::-1], "bfloat16").astype(np.float32), "last rows")
    finally:
        table.free()


@pytest.mark.parametrize("dtype", range(34), ids=DTYPE_NAMES)
def test_store_lookup(stream, dtype):
    """Rows of a mounted layer's store are its exported rows times the scale,
    at a width whose sub-byte rows start inside bytes."""
    rng = np.random.default_rng(dtype)
    W = rng.normal(0, 1, (41, 67)).astype(np.float32)
    tok = np.array([0, 40, -1, 7, 41, 7], np.int32)
    with pywelvet.Session(W, 1, dtype=dtype) as s:
        values = s.export_f32()
        d_k, out = Dev(tok), Dev(np.zeros((6, 70), np.float32))
        pywelvet.embedding_store_forward(s, d_k.ptr, 6, out.ptr, scale=3.0, out_stride=70, stream=stream)
        got = out.get()
    want = np.zeros((6, 67), np.float32)
    for i, t in enumerate(tok):
        if 0 <= t < 41:
            want[i] = values[t] * np.float32(3.0)
    assert_bit_equal(got[:, :67], want, DTYPE_NAMES[dtype])
    assert (got[:, 67:] == 0).all()


def gradient(stream, vocab, dim, tok, dout, scale, start=None, extra=0):
    """The gradient from sentinel-filled (or `start`) memory, checked for its padding columns."""
    n = tok.size
    d_k, d_o = Dev(tok), Dev(strided(dout, extra))
    first = np.full((vocab, dim), np.nan, np.float32) if start is None else start
    table = Dev(strided(first, extra, 5.0))
    nb = pywelvet.embedding_backward_bytes(vocab, dim, n)
    ws = Dev(np.full(max(nb, 1), 0xFF, np.uint8))
    pywelvet.embedding_backward(vocab, dim, d_k.ptr, n, d_o.ptr, table.ptr, scale=scale, accumulate=start is not None,
                                dout_stride=dim + extra, dtable_stride=dim + extra, ws=ws.ptr, ws_bytes=nb,
                                stream=stream)
    got = table.get()
    ws.get()
    assert (got[:, dim:] == 5.0).all()
    return got[:, :dim]


def exact_gradient(vocab, dim, tok, dout, scale):
    want, size, count = np.zeros((vocab, dim)), np.zeros((vocab, dim)), np.zeros(vocab)
    ok = (tok >= 0) & (tok < vocab)
    np.add.at(want, tok[ok], dout[ok].astype(np.float64))
    np.add.at(size, tok[ok], np.abs(dout[ok].astype(np.float64)))
    np.add.at(count, tok[ok], 1)
    s = float(np.float32(scale))
    return want * s, size * abs(s), count


# n: the direct route up to 256, one sorted chunk up to 4096, joined chunks above
@pytest.mark.parametrize("vocab,dim,n,extra", [
    (1, 1, 1, 0), (50, 64, 7, 0), (1001, 777, 100, 0), (40, 1028, 256, 4), (40, 20, 257, 0), (9, 130, 1000, 2),
    (5000, 256, 4096, 0), (5000, 333, 4097, 0), (3, 64, 9000, 0), (700, 1540, 20000, 4)])
@pytest.mark.parametrize("accumulate", [False, True])
def test_gradient(stream, vocab, dim, n, extra, accumulate):
    rng = np.random.default_rng(vocab + dim + n)
    tok = tokens_of(rng, vocab, n)
    dout = rng.normal(0, 1, (n, dim)).astype(np.float32)
    dout[(tok < 0) | (tok >= vocab)] = np.nan  # padding's rows are not read
    start = rng.normal(0, 1, (vocab, dim)).astype(np.float32) if accumulate else None
    got = gradient(stream, vocab, dim, tok, dout, 2.5, start, extra)
    want, size, count = exact_gradient(vocab, dim, tok, dout, 2.5)
    bound = 2 * (count[:, None] + 1) * U * size
    if accumulate:
        assert_bit_equal(got[count == 0], start[count == 0], "rows without a token")
        want = want + start
        bound = bound + 2 * U * (np.abs(want) + np.abs(start)) * (count[:, None] > 0)
    within(got, want, bound, "gradient")
    again = gradient(stream, vocab, dim, tok, dout, 2.5, start, extra)
    assert_bit_equal(again, got, "a second run")


@pytest.mark.parametrize("n", [0, 5, 300, 5000])
def test_gradient_of_padding_only(stream, n):
    tok = np.full(n, -1, np.int32)
    got = gradient(stream, 70, 65, tok, np.full((n, 65), np.nan, np.float32), 1.0)
    assert_bit_equal(got, np.zeros((70, 65), np.float32), "zeros")
    start = np.arange(70 * 65, dtype=np.float32).reshape(70, 65)
    assert_bit_equal(gradient(stream, 70, 65, tok, np.full((n, 65), np.nan, np.float32), 1.0, start), start, "kept")


@pytest.mark.parametrize("n", [200, 4096, 9999])
def test_gradient_of_one_token(stream, n):
    """All rows one token: the partial sums of every block."""
    rng = np.random.default_rng(n)
    dout = rng.normal(0, 1, (n, 40)).astype(np.float32)
    tok = np.full(n, 11, np.int32)
    want, size, count = exact_gradient(30, 40, tok, dout, 1.0)
    within(gradient(stream, 30, 40, tok, dout, 1.0), want, 2 * (count[:, None] + 1) * U * size, "one token")


def test_gradient_keeps_order_and_specials(stream):
    """Infinities and NaN of a token's rows stay in that token's row."""
    dout = np.zeros((6, 8), np.float32)
    dout[0], dout[1], dout[2], dout[3] = np.inf, 1, np.nan, -np.inf
    tok = np.array([3, 3, 4, 5, 1, 1], np.int32)
    got = gradient(stream, 7, 8, tok, dout, 1.0)
    assert np.isposinf(got[3]).all() and np.isnan(got[4]).all() and np.isneginf(got[5]).all()
    assert (got[[0, 1, 2, 6]] == 0).all()


def test_gradient_is_the_forward_s(stream):
    """<dout, lookup(E + d) - lookup(E)> = <dE, d>: the lookup is linear, so
    the difference is exact up to rounding (the sum over n * dim products of
    f32 roundings stays below 1e-5 of the products' absolute sum)."""
    rng = np.random.default_rng(9)
    vocab, dim, n, scale = 60, 48, 500, 4.0
    tok = tokens_of(rng, vocab, n)
    table, step = rng.normal(0, 1, (vocab, dim)), rng.normal(0, 1, (vocab, dim))
    dout = rng.normal(0, 1, (n, dim)).astype(np.float32)
    outs = []
    for E in (table, table + step):
        d_t, d_k, out = Dev(E.astype(np.float32)), Dev(tok), Dev(np.zeros((n, dim), np.float32))
        pywelvet.embedding_forward(1, vocab, dim, d_t.ptr, d_k.ptr, n, out.ptr, scale=scale, stream=stream)
        outs.append(out.get().astype(np.float64))
    prod = dout * (outs[1] - outs[0])
    grad = gradient(stream, vocab, dim, tok, dout, scale).astype(np.float64)
    moved = (table + step).astype(np.float32).astype(np.float64) - table.astype(np.float32)
    assert abs(prod.sum() - (grad * moved).sum()) <= 1e-5 * np.abs(prod).sum()


def test_refusals(stream):
    a, b, t = Dev(np.zeros(64, np.float32)), Dev(np.zeros(64, np.float32)), Dev(np.zeros(4, np.int32))
    fwd = lambda *args, **kw: pywelvet.embedding_forward(*args, stream=stream, status=True, **kw).code  # noqa: E731
    assert fwd(1, 4, 8, a.ptr, t.ptr, 4, b.ptr) == 0
    assert fwd(4, 4, 8, a.ptr, t.ptr, 4, a.ptr) == 2
    assert fwd(1, 0, 8, a.ptr, t.ptr, 4, a.ptr) == 1
    assert fwd(1, 4, 0, a.ptr, t.ptr, 4, a.ptr) == 1
    assert fwd(1, 4, 8, a.ptr, t.ptr, -1, a.ptr) == 1
    assert fwd(1, 4, 8, None, t.ptr, 4, a.ptr) == 1
    assert fwd(1, 4, 8, a.ptr, None, 4, a.ptr) == 1
    assert fwd(1, 4, 8, a.ptr, t.ptr, 4, None) == 1
    assert fwd(1, 4, 8, a.ptr + 2, t.ptr, 4, a.ptr) == 1
    assert fwd(1, 4, 8, a.ptr, t.ptr, 4, a.ptr, table_stride=7) == 1
    assert fwd(1, 4, 8, a.ptr, None, 0, None) == 0
    bwd = lambda n, need, **kw: pywelvet.embedding_backward(  # noqa: E731
        8, 8, t.ptr, n, a.ptr, a.ptr, ws=a.ptr, ws_bytes=need, stream=stream, status=True, **kw).code
    assert bwd(300, pywelvet.embedding_backward_bytes(8, 8, 300) - 1) == 1
    assert bwd(4, 0, dout_stride=7) == 1
    with pywelvet.Session(np.zeros((4, 8), np.float32), 1) as s:
        assert pywelvet.embedding_store_forward(s, t.ptr, 4, a.ptr, out_stride=7, stream=stream, status=True).code == 1
        assert pywelvet.embedding_store_forward(s, None, 4, a.ptr, stream=stream, status=True).code == 1


def sums_in_order(vocab, tok, dout):
    """The gradient as f32 adds in the documented order: rows by (token, row),
    in runs of 32 whose sums a token's later runs are added to."""
    order = np.argsort(np.where((tok >= 0) & (tok < vocab), tok, vocab), kind="stable")
    out, key = np.zeros((vocab, dout.shape[1]), np.float32), tok[order]
    total = None
    for i, t in enumerate(order):
        if i == 0 or key[i] != key[i - 1] or i % 32 == 0:
            part = np.zeros(dout.shape[1], np.float32)
        part = part + dout[t]
        last = i + 1 == len(order) or key[i + 1] != key[i]
        if last or i % 32 == 31:
            total = part if total is None else total + part
            if last:
                if 0 <= key[i] < vocab:
                    out[key[i]] = total
                total = None
    return out


# one chunk of 2048 sorted rows, joined chunks to 65536 rows, joined spans above
# (twice from 2^19 on)
@pytest.mark.parametrize("skewed", [False, True])
@pytest.mark.parametrize("n", [2047, 2048, 2049, 4095, 16385, 65536, 65537, 100003, 540001])
def test_gradient_sums_in_row_order(stream, n, skewed):
    rng = np.random.default_rng([n, skewed])
    vocab = 3001
    tok = (np.exp(rng.random(n) * np.log(vocab + 40)) if skewed else rng.integers(-20, vocab + 20, n)).astype(np.int32)
    dout = rng.normal(0, 1, (n, 2)).astype(np.float32)
    got = gradient(stream, vocab, 2, tok, dout, 2.0)
    assert_bit_equal(got, sums_in_order(vocab, tok, dout) * np.float32(2.0), "gradient")


# one column less and more than a block's 1024, several blocks, one column
@pytest.mark.parametrize("dim", [1, 1023, 1025, 2051])
@pytest.mark.parametrize("dtype", ["float32", "bfloat16", "fp8e4m3", "int8", "int4", "nf4", "fp4", "uint8", "binary",
                                   "ternary", "int64", "complex64"])
def test_store_lookup_of_wide_rows(stream, dtype, dim):
    rng = np.random.default_rng(dim)
    W = rng.normal(0, 1, (33, dim)).astype(np.float32)
    tok = rng.integers(-2, 36, 300).astype(np.int32)
    tok[:2] = 32, 0
    with pywelvet.Session(W, 1, dtype=pywelvet.DTYPE[dtype]) as s:
        values = s.export_f32()
        d_k, out = Dev(tok), Dev(np.full((300, dim + 1), 9.0, np.float32))
        pywelvet.embedding_store_forward(s, d_k.ptr, 300, out.ptr, scale=-0.5, out_stride=dim + 1, stream=stream)
        got = out.get()
    there = (tok >= 0) & (tok < 33)
    want = np.where(there[:, None], values[np.where(there, tok, 0)] * np.float32(-0.5), np.float32(0))
    assert_bit_equal(got[:, :dim], want.astype(np.float32), dtype)
    assert (got[:, dim] == 9.0).all()


def test_store_lookup_of_a_zero_scale(stream):
    """A store whose scale is 0 decodes as 1, as in the layer's own products."""
    raw = np.random.default_rng(1).integers(-128, 128, (5, 30)).astype(np.int8)
    with pywelvet.Session((5, 30), 1, dtype=pywelvet.DTYPE["int8"], native=(raw.view(np.uint8).reshape(-1), 0.0)) as s:
        d_k, out = Dev(np.arange(5, dtype=np.int32)), Dev(np.full((5, 30), 9.0, np.float32))
        pywelvet.embedding_store_forward(s, d_k.ptr, 5, out.ptr, stream=stream)
        assert_bit_equal(out.get(), raw.astype(np.float32), "rows")
