"""welvet_hip_logits_rules against the rules in f64: rounded once, so the bits
have to be equal, and logits that no rule names keep theirs."""
import numpy as np
import pytest

import pywelvet
from devmem import Stream
from parity import assert_bit_equal
from tokmem import DT, Big, Dev, strided, to_bits, to_f64

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


def rounded(z, dtype):
    """f64 to a type's bits, to nearest even, once."""
    if dtype == "float32":
        return z.astype(np.float32)
    if dtype == "float16":
        return z.astype(np.float16)
    f = z.astype(np.float32)  # the nearest f32, its last bit set where it is not exact: rounds on as the f64 would
    u = f.view(np.uint32).copy()
    off = (f.astype(np.float64) != z) & ~np.isnan(z)
    u = np.where(off & (np.abs(f.astype(np.float64)) > np.abs(z)), u - np.uint32(1), u)
    return to_bits(np.where(off, u | np.uint32(1), u).astype(np.uint32).view(np.float32), dtype)


SHUT = {"float32": np.float32(-np.inf), "float16": np.float16(-np.inf), "bfloat16": np.uint16(0xFF80)}


def make(rng, n, vocab, history=0, biases=0, masks=0, share=0.5):
    """Rules as host arrays; tokens and entries repeat, and lie outside the vocabulary here and there."""
    r = {}
    if history:
        t = rng.integers(0, vocab, (n, history))
        t[:, ::3] = rng.integers(0, max(1, vocab // 50), t[:, ::3].shape)
        t = np.where(rng.random(t.shape) < 0.05, rng.choice([-1, vocab, -2 ** 31, 2 ** 31 - 1], t.shape), t)
        r.update(history=t.astype(np.int32), length=rng.integers(0, history + 1, n).astype(np.int32))
        r["prompt"] = (r["length"] * rng.random(n)).astype(np.int32)
    for k, lo, hi in (("repetition", 0.7, 1.6), ("frequency", -0.3, 0.5), ("presence", -0.5, 1)):
        r[k] = rng.uniform(lo, hi, n).astype(np.float32)
    if biases:
        at = rng.integers(0, vocab, (n, biases))
        at = np.where(rng.random(at.shape) < 0.2, rng.integers(0, max(1, vocab // 100), at.shape), at)
        at = np.where(rng.random(at.shape) < 0.05, rng.choice([-1, vocab, 2 ** 31 - 1], at.shape), at)
        r.update(index=at.astype(np.int32), bias=rng.normal(0, 3, (n, biases)).astype(np.float32))
        if history:  # some of them on tokens that were said
            some = min(biases, history) // 2
            r["index"][:, :some] = r["history"][:, :some]
    if masks:
        words = (vocab + 31) // 32
        bits = rng.random((masks, words * 32)) < share
        r["masks"] = np.packbits(bits, axis=1, bitorder="little").view(np.uint32)
        r["mask"] = rng.integers(-1, masks + 1, n).astype(np.int32)
    return r


def expected(z, dtype, r):
    out = z.copy()
    vocab = z.shape[1]
    for t in range(z.shape[0]):
        v64, touched = to_f64(z[t], dtype), np.zeros(vocab, bool)
        if "history" in r:
            length = int(np.clip(r["length"][t], 0, r["history"].shape[1])) if "length" in r else r["history"].shape[1]
            prompt = int(np.clip(r["prompt"][t], 0, length)) if "prompt" in r else 0
            said = r["history"][t][:length].astype(np.int64)
            ok = (said >= 0) & (said < vocab)
            seen = np.unique(said[ok])
            after = said[prompt:][ok[prompt:]]
            if "repetition" in r:
                rep = np.float64(r["repetition"][t])
                v64[seen] = np.where(v64[seen] > 0, v64[seen] / rep, v64[seen] * rep)
            count = np.bincount(after, minlength=vocab)
            at = np.nonzero(count)[0]
            f = np.float64(r["frequency"][t]) if "frequency" in r else 0.0
            p = np.float64(r["presence"][t]) if "presence" in r else 0.0
            v64[at] = v64[at] - count[at] * f - p
            touched[seen] = True
        if "index" in r:
            sums = {}
            for i, b in zip(r["index"][t].tolist(), r["bias"][t].astype(np.float64)):
                if 0 <= i < vocab:
                    v64[i] = v64[i] + b
                    touched[i] = True
        out[t][touched] = rounded(v64[touched], dtype)
        if "masks" in r:
            m = int(r["mask"][t]) if "mask" in r else t
            if 0 <= m < r["masks"].shape[0]:
                open_ = np.unpackbits(r["masks"][m].view(np.uint8), bitorder="little")[:vocab].astype(bool)
                out[t][~open_] = SHUT[dtype]
    return out


def apply(stream, z, dtype, r, extra=0, shift=0, in_place=False, mask_extra=0):
    n, vocab = z.shape
    d_z = Dev(np.concatenate([np.zeros(shift, z.dtype), strided(z, extra).reshape(-1)]))
    kw, keep = {}, []

    def put(name, a):
        keep.append(Dev(a))
        kw[name] = keep[-1].ptr
    if "history" in r:
        h = r["history"]
        put("d_history", strided(h, extra, fill=0))
        kw.update(history=h.shape[1], history_stride=h.shape[1] + extra)
        for k, name in (("length", "d_history_len"), ("prompt", "d_prompt_len")):
            if k in r:
                put(name, r[k])
    for k in ("repetition", "frequency", "presence"):
        if k in r:
            put("d_" + k, r[k])
    if "index" in r:
        put("d_bias_index", r["index"])
        put("d_bias", r["bias"])
        kw["biases"] = r["index"].shape[1]
    if "masks" in r:
        m = r["masks"]
        put("d_masks", np.concatenate([m, np.full((m.shape[0], mask_extra), 0x55, np.uint32)], 1))
        kw.update(masks=m.shape[0], mask_stride=m.shape[1] + mask_extra)
        if "mask" in r:
            put("d_mask_id", r["mask"])
    rules = pywelvet.LogitRules(**kw)
    ptr = d_z.ptr + shift * z.dtype.itemsize
    other = 0 if in_place else (extra + 1) % 3
    out = d_z if in_place else Dev(np.full((n, vocab + other), 5, z.dtype))
    before = d_z.get()
    rules.apply(DT[dtype], n, vocab, ptr, ptr if in_place else out.ptr, stride=vocab + extra,
                out_stride=vocab + (extra if in_place else other), stream=stream)
    got = out.get()
    if in_place:
        got = got[shift:].reshape(n, vocab + extra)
        rest = before[shift:].reshape(n, vocab + extra)[:, vocab:]
        assert got[:, vocab:].tobytes() == rest.tobytes()
    else:
        assert (got[:, vocab:] == 5).all()
        assert d_z.get().tobytes() == before.tobytes()
    return got[:, :vocab]


SHAPES = [(1, 1, 1, 1, 1), (2, 31, 5, 3, 1), (3, 33, 40, 0, 2), (1, 1001, 500, 8, 0), (4, 32000, 300, 8, 3),
          (3, 50257, 2000, 100, 2), (2, 131072, 5000, 1024, 1), (600, 777, 64, 5, 4), (300, 2049, 1, 1, 0),
          (1, 16384, 0, 20, 1), (2, 16385, 100, 0, 0), (5, 40000, 0, 0, 2), (64, 8192, 3000, 300, 64),
          (520, 8192, 60, 5, 3), (513, 8193, 60, 5, 3)]


@pytest.mark.parametrize("dtype", DT)
@pytest.mark.parametrize("n,vocab,history,biases,masks", SHAPES)
def test_rules(stream, dtype, n, vocab, history, biases, masks):
    rng = np.random.default_rng([n, vocab, history])
    z = to_bits(rng.normal(0, 4, (n, vocab)), dtype)
    r = make(rng, n, vocab, history, biases, masks, (0.5, 0.001, 0.999)[vocab % 3])
    want = expected(z, dtype, r)
    for in_place in (False, True):
        got = apply(stream, z, dtype, r, n % 2, vocab % 4, in_place, n % 3)
        assert got.tobytes() == want.tobytes(), (in_place, np.argwhere(got != want)[:5])


@pytest.mark.parametrize("dtype", DT)
@pytest.mark.parametrize("drop", ["length", "prompt", "repetition", "frequency", "presence", "mask"])
def test_what_is_not_given(stream, dtype, drop):
    rng = np.random.default_rng(len(drop))
    z = to_bits(rng.normal(0, 4, (5, 3000)), dtype)
    r = make(rng, 5, 3000, 200, 9, 4)
    del r[drop]
    want = expected(z, dtype, r)
    for in_place in (False, True):
        assert apply(stream, z, dtype, r, in_place=in_place).tobytes() == want.tobytes()


@pytest.mark.parametrize("dtype", DT)
def test_one_token_over_and_over(stream, dtype):
    """The same token through a whole history, in every entry of the list, and alone under a mask."""
    z = to_bits(np.random.default_rng(1).normal(0, 4, (2, 5000)), dtype)
    r = dict(history=np.full((2, 70000), 4321, np.int32), length=np.array([70000, 2 ** 31 - 1], np.int32),
             prompt=np.array([0, 69999], np.int32), repetition=np.array([1.25, 0.5], np.float32),
             frequency=np.array([1e-4, 0.125], np.float32), presence=np.array([0.5, 0.25], np.float32),
             index=np.full((2, 1024), 4321, np.int32),
             bias=np.random.default_rng(2).normal(0, 1, (2, 1024)).astype(np.float32))
    want = expected(z, dtype, r)
    for in_place in (False, True):
        assert apply(stream, z, dtype, r, in_place=in_place).tobytes() == want.tobytes()
    r["masks"] = np.zeros((1, 157), np.uint32)
    r["masks"][0, 4321 // 32] = 1 << (4321 % 32)
    r["mask"] = np.zeros(2, np.int32)
    want = expected(z, dtype, r)
    assert np.isinf(to_f64(want, dtype)).sum() == 2 * 4999
    for in_place in (False, True):
        assert apply(stream, z, dtype, r, in_place=in_place).tobytes() == want.tobytes()


@pytest.mark.parametrize("dtype", DT)
def test_values_that_are_not_finite(stream, dtype):
    """Infinite logits and biases pass the rules as the formulas have it, a mask
    shuts whatever lies there, and a mask may leave nothing."""
    rng = np.random.default_rng(3)
    z = to_bits(rng.normal(0, 4, (3, 400)), dtype)
    for at, v in ((5, -np.inf), (6, np.inf), (7, 0.0), (8, -0.0), (9, 60000.0), (10, -60000.0)):
        z[:, at] = to_bits(np.array([v]), dtype)[0]
    lowest = {"float32": -3.4028235e38, "float16": -65504.0, "bfloat16": -3.3895314e38}[dtype]
    z[:, 11] = to_bits(np.array([lowest]), dtype)[0]
    r = make(rng, 3, 400, 30, 6, 2)
    r["history"][:, :7] = np.arange(5, 12)
    r["length"][:], r["prompt"][:] = 30, 3
    r["index"][:, 0], r["bias"][:, 0] = 20, -np.inf
    r["index"][:, 1], r["bias"][:, 1] = 5, np.inf  # -inf + inf: NaN
    r["index"][:, 2], r["bias"][:, 2] = 21, 3e38
    r["masks"][0] = 0
    r["mask"][:] = [0, 1, -1]
    with np.errstate(invalid="ignore", over="ignore"):
        want = expected(z, dtype, r)
    for in_place in (False, True):
        got = apply(stream, z, dtype, r, in_place=in_place)
        g, w = to_f64(got, dtype), to_f64(want, dtype)
        assert np.array_equal(np.isnan(g), np.isnan(w)) and np.isnan(w[2, 5])
        some = ~np.isnan(w)
        assert got[some].tobytes() == want[some].tobytes()
    assert np.isneginf(to_f64(got, dtype)[0]).all()


def test_no_rules_copy(stream):
    z = np.random.default_rng(4).normal(0, 1, (3, 1000)).astype(np.float32)
    for in_place in (False, True):
        assert_bit_equal(apply(stream, z, "float32", {}, 1, 1, in_place), z, "a copy")


def test_logits_past_32_bits(stream):
    """Rows that begin past 2^32 bytes."""
    from tokmem import Big
    vocab, stride, n = 1000, (1 << 30) + 1, 3
    big = Big(4 * (stride * (n - 1) + vocab))
    rng = np.random.default_rng(5)
    z = rng.normal(0, 1, (n, vocab)).astype(np.float32)
    for t in range(n):
        big.put(4 * stride * t, z[t])
    r = make(rng, n, vocab, 50, 4)
    keep = [Dev(r[k]) for k in ("history", "length", "prompt", "repetition", "frequency", "presence", "index", "bias")]
    rules = pywelvet.LogitRules(50, keep[0].ptr, None, *(d.ptr for d in keep[1:6]), 4, keep[6].ptr, keep[7].ptr)
    rules.apply(1, n, vocab, big.ptr, big.ptr, stride=stride, out_stride=stride, stream=stream)
    want = expected(z, "float32", r)
    for t in range(n):
        assert_bit_equal(big.get(4 * stride * t, vocab, np.float32), want[t], f"row {t}")
    big.free()


@pytest.mark.parametrize("in_place", [False, True])
def test_rows_past_32_bits(stream, in_place):
    """The last row of the logits and of the history begins past 2^32 values."""
    rng, n, vocab, stride = np.random.default_rng(6), 3, 9000, 2 ** 31 + 24
    z = to_bits(rng.normal(0, 4, (n, vocab)), "bfloat16")
    r = make(rng, n, vocab, 300, 0, 2)
    want = apply(stream, z, "bfloat16", r)
    logits, out, said = (Big(size * (stride * (n - 1) + w)) for size, w in ((2, vocab), (2, vocab), (4, 300)))
    for t in range(n):
        logits.put(2 * stride * t, z[t])
        said.put(4 * stride * t, r["history"][t])
    keep = {k: Dev(r[k]) for k in ("length", "prompt", "repetition", "frequency", "presence", "masks", "mask")}
    rules = pywelvet.LogitRules(
        history=300, d_history=said.ptr, history_stride=stride, d_history_len=keep["length"].ptr,
        d_prompt_len=keep["prompt"].ptr, d_repetition=keep["repetition"].ptr, d_frequency=keep["frequency"].ptr,
        d_presence=keep["presence"].ptr, masks=2, d_masks=keep["masks"].ptr, mask_stride=r["masks"].shape[1],
        d_mask_id=keep["mask"].ptr)
    to = logits if in_place else out
    rules.apply(3, n, vocab, logits.ptr, to.ptr, stride=stride, out_stride=stride, stream=stream)
    keep["mask"].get()
    for t in range(n):
        assert to.get(2 * stride * t, vocab, np.uint16).tobytes() == want[t].tobytes()
    for b in (logits, out, said):
        b.free()
