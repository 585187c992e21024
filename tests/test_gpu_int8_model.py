"""The 8-bit activation operators and the logits' rules together: the example
that trains and answers with them, captured into HIP graphs, and on two streams."""
import os
import sys

import numpy as np
import pytest

import pywelvet
from devmem import Stream
from parity import assert_bit_equal
from rows8ref import Rows, act, act_prime, codes_of
from test_gpu_tokens import Graph
from tokmem import U, Dev

sys.path.insert(0, os.path.join(os.path.dirname(os.path.abspath(__file__)), "..", "examples"))
pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module", autouse=True)
def device():
    pywelvet.init()


@pytest.fixture
def stream():
    s = Stream()
    yield s
    s.sync()
    s.close()


def test_example_runs():
    import int8_mlp as ex
    losses, prompts, answers = ex.run(3, say=lambda s: None)
    assert np.isfinite(losses).all()
    for p, a in zip(prompts, answers):
        assert len(a) == 6 and all(0 <= t < ex.VOCAB for t in a)
        assert not set(p) & set(a)  # the mask shuts the prompt's own tokens


def test_example_gradients():
    """A step's loss and every gradient against f64 at the values that the rows
    and the layers hold.  The forward's values are within 2e-6 of the largest of
    their row (an f32 chain of a few roundings, sums of 8-bit products exact); a
    code of h or y may differ where a quotient lies next to a half, so the
    backward starts from the codes read back.  Each product's bound is its terms'
    magnitudes times 2^-22 and its sum's K U, with what its own input is off."""
    import int8_mlp as ex
    model, n = ex.Model(), ex.ROWS
    tokens, index, teacher = ex.batch(np.random.default_rng(3))
    W = {}
    for name in ("gate", "up", "down", "head"):
        codes, scales = getattr(model, name).mounted.weights()
        W[name] = codes.astype(np.float64) * scales.astype(np.float64)[:, None]
        want, ws = codes_of(getattr(model, name).W.get())
        assert np.array_equal(codes, want) and np.array_equal(scales, ws)
    table = model.table.get().astype(np.float64)
    for to, a in ((model.tokens, tokens), (model.index, index), (model.teacher, teacher)):
        to.put(a)
    model.forward(n)

    def close(got, want, bound, what):
        off = np.abs(got.astype(np.float64) - want)
        assert (off <= bound).all(), (what, (off / bound).max())
    x8, h8, y8 = model.x8.values(), model.h8.values(), model.y8.values()
    codes, scales = codes_of(table[tokens])
    assert np.array_equal(model.x8.codes.get()[:, :ex.DIM], codes)
    g, u = model.g.get(), model.u.get()
    close(g, x8 @ W["gate"].T, 8 * U * np.abs(x8) @ np.abs(W["gate"].T), "gate")
    close(u, x8 @ W["up"].T, 8 * U * np.abs(x8) @ np.abs(W["up"].T), "up")
    g8, u8 = model.gate8.values(), model.up8.values()
    h = act(g.astype(np.float64), "silu") * u
    close(h8, h, 0.501 * model.h8.scales.get()[:, None].astype(np.float64) + 1e-6 * np.abs(h), "h")
    close(model.y.get(), h8 @ W["down"].T, 8 * U * np.abs(h8) @ np.abs(W["down"].T), "y")
    logits = model.logits.get().astype(np.float64)
    close(logits, y8 @ W["head"].T, 8 * U * np.abs(y8) @ np.abs(W["head"].T), "logits")
    pywelvet.distill(1, n, ex.VOCAB, model.logits.ptr, ex.TOP, model.index.ptr, model.teacher.ptr, model.loss.ptr,
                     model.logits.ptr, 1.0, model.weight.ptr, **model.on)
    z = logits - logits.max(1, keepdims=True)
    p = np.exp(z) / np.exp(z).sum(1, keepdims=True)
    q = np.exp(teacher.astype(np.float64))
    q /= q.sum(1, keepdims=True)
    dlogits = p.copy()
    np.add.at(dlogits, (np.arange(n)[:, None], index), -q)
    close(model.logits.get(), dlogits / n, 3000 * U / n, "dlogits")  # the loss's own tests bound it
    dl = model.logits.get().astype(np.float64)
    model.backward(n)

    def product(a, b, da):
        """a . b and its bound where a is off by da."""
        return a @ b, da @ np.abs(b) + (2.0 ** -21 + (2 * a.shape[1] + 12) * U) * np.abs(a) @ np.abs(b)
    none = np.zeros_like(dl)
    dy, e_dy = product(dl, W["head"], none)
    close(model.dy.get(), dy, e_dy, "dy")
    close(model.head.dw.get(), *product(dl.T, y8, none.T), "head's dw")
    dy = model.dy.get().astype(np.float64)
    dh, e_dh = product(dy, W["down"], 0 * dy)
    close(model.dh.get(), dh, e_dh, "dh")
    close(model.down.dw.get(), *product(dy.T, h8, 0 * dy.T), "down's dw")
    dh = model.dh.get().astype(np.float64)
    dg, du = model.g.get(), model.u.get()
    close(dg, dh * u8 * act_prime(g8, "silu"), np.abs(dh * u8) * (70 + np.abs(g8)) * U + 1e-37, "dgate")
    close(du, dh * act(g8, "silu"), np.abs(dh * g8) * (16 + np.abs(g8)) * U + 1e-37, "dup")
    for name, d, to in (("gate", dg, model.dx), ("up", du, model.dx2)):
        d = d.astype(np.float64)
        close(to.get(), *product(d, W[name], 0 * d), name + "'s dx")
        close(getattr(model, name).dw.get(), *product(d.T, x8, 0 * d.T), name + "'s dw")
    model.close()


@pytest.mark.parametrize("n", [70, 5])
def test_graph_of_a_step(stream, n):
    """A layer's step and an answer's rules in one graph: every replay, with other
    inputs and work between them, has the bits of the calls themselves."""
    rng = np.random.default_rng(4)
    inn, inter, vocab = 130, 300, 1000
    x, dy = Dev(np.zeros((n, inn), np.float32)), Dev(np.zeros((n, vocab), np.float32))
    gate, up, head = (pywelvet.Int8Layer(rng.normal(0, 0.1, s), a) for s, a in (((inter, inn), -1), ((inter, inn), -1),
                                                                             ((vocab, inter), 2)))
    x8, g8, u8, h8, p8 = (Rows(n, w) for w in (inn, inter, inter, inter, vocab))
    out = {k: Dev(np.zeros(s, np.float32)) for k, s in dict(
        g=(n, inter), u=(n, inter), h=(n, inter), pre=(n, vocab), post=(n, vocab), dpre=(n, vocab), dh=(n, inter),
        dg=(n, inter), du=(n, inter), dx=(n, inn), dw=(vocab, inter), dwg=(inter, inn), z=(n, vocab), one=(2, vocab)).items()}
    need = max([layer.workspace_bytes(n) for layer in (gate, up, head)] +
               [pywelvet.rows8_backward_bytes(1, n, inter, vocab), pywelvet.rows8_backward_bytes(1, n, inn, inter)])
    ws = Dev(np.zeros(need, np.uint8))
    on = dict(ws=ws.ptr, ws_bytes=need, stream=stream.h)
    history = Dev(rng.integers(0, vocab, (n, 90)).astype(np.int32))
    rep, index, bias = Dev(rng.uniform(1, 2, n).astype(np.float32)), Dev(rng.integers(0, vocab, (n, 5)).astype(np.int32)), \
        Dev(rng.normal(0, 1, (n, 5)).astype(np.float32))
    masks = Dev(rng.integers(0, 2 ** 32, (n, 32), dtype=np.uint64).astype(np.uint32))
    rules = pywelvet.LogitRules(history=90, d_history=history.ptr, d_repetition=rep.ptr, d_frequency=rep.ptr, biases=5,
                                d_bias_index=index.ptr, d_bias=bias.ptr, masks=n, d_masks=masks.ptr)

    def calls():
        gate.forward(1, n, x.ptr, rows=x8.desc, d_post=out["g"].ptr, **on)
        up.product(1, n, x8.desc, d_post=out["u"].ptr, **on)
        pywelvet.rows8_swiglu(1, n, inter, out["g"].ptr, out["u"].ptr, g8.desc, u8.desc, h8.desc, out["h"].ptr,
                              stream=stream.h)
        head.product(1, n, h8.desc, out["pre"].ptr, out["post"].ptr, **on)
        pywelvet.rows8_store(1, n, vocab, out["pre"].ptr, p8.desc, stream=stream.h)
        pywelvet.rows8_load(1, n, vocab, p8.desc, out["z"].ptr, stream=stream.h)
        pywelvet.rows8_backward(2, 1, n, inter, vocab, dy.ptr, p8.desc, h8.desc, head, out["dpre"].ptr, out["dh"].ptr,
                                out["dw"].ptr, **on)
        pywelvet.rows8_swiglu_backward(1, n, inter, g8.desc, u8.desc, out["dh"].ptr, out["dg"].ptr, out["du"].ptr,
                                       stream=stream.h)
        pywelvet.rows8_backward(-1, 1, n, inn, inter, out["dg"].ptr, x=x8.desc, layer=gate, d_dx=out["dx"].ptr,
                                d_dw=out["dwg"].ptr, **on)
        rules.apply(1, n, vocab, out["post"].ptr, out["z"].ptr, stream=stream.h)
        rules.apply(1, n, vocab, out["post"].ptr, out["post"].ptr, stream=stream.h)
        head.forward(1, 2, out["h"].ptr, d_post=out["one"].ptr, **on)  # few rows, by themselves
    from devmem import _ok, hip

    def put(dev, a):
        _ok(hip().hipMemcpy(dev.ptr, np.ascontiguousarray(a).ctypes.data, a.nbytes, 1), "hipMemcpy")
    graph = Graph(stream, calls)
    for i in range(4):
        put(x, rng.normal(0, 1 + i, (n, inn)).astype(np.float32))
        put(dy, rng.normal(0, 1, (n, vocab)).astype(np.float32))
        stream.sync()
        calls()
        stream.sync()
        want = {k: d.get() for k, d in out.items()}
        for d in out.values():
            put(d, np.full(d.shape, 9, np.float32))
        stream.sync()
        graph.launch()
        stream.sync()
        for k, d in out.items():
            assert np.array_equal(d.get(), want[k], equal_nan=True), (i, k)
    graph.close()
    for layer in (gate, up, head):
        layer.close()


def test_backwards_on_two_streams(stream):
    """Two backward calls at once, a workspace each, over one layer."""
    rng = np.random.default_rng(6)
    other = Stream()
    n, inn, out = 200, 700, 520
    layer = pywelvet.Int8Layer(rng.normal(0, 1, (out, inn)))
    sides = []
    for s in (stream, other):
        xc, xs = codes_of(rng.normal(0, 1, (n, inn)).astype(np.float32))
        sides.append(dict(s=s, x8=Rows(n, inn, 0, xc, xs), dy=Dev(rng.normal(0, 1, (n, out)).astype(np.float32)),
                          dx=Dev(np.zeros((n, inn), np.float32)), dw=Dev(np.zeros((out, inn), np.float32)),
                          ws=Dev(np.zeros(pywelvet.rows8_backward_bytes(1, n, inn, out), np.uint8))))

    def go(d):
        pywelvet.rows8_backward(-1, 1, n, inn, out, d["dy"].ptr, x=d["x8"].desc, layer=layer, d_dx=d["dx"].ptr,
                                d_dw=d["dw"].ptr, ws=d["ws"].ptr, ws_bytes=d["ws"].nbytes, stream=d["s"].h)
    want = []
    for d in sides:
        go(d)
        d["s"].sync()
        want.append((d["dx"].get(), d["dw"].get()))
    for _ in range(8):
        for d in sides:
            go(d)
    for d, (dx, dw) in zip(sides, want):
        assert_bit_equal(d["dx"].get(), dx, "dx")
        assert_bit_equal(d["dw"].get(), dw, "dw")
    other.close()
    layer.close()


@pytest.mark.parametrize("inn,out", [(50, 70), (4096, 300), (11008, 64)])
def test_forward_workspace_serves_smaller_batches(inn, out):
    with pywelvet.Int8Layer(np.ones((out, inn), np.float32)) as layer:
        sizes = [layer.workspace_bytes(n) for n in (*range(0, 300), 2047, 2048, 5000)]
        assert sizes == sorted(sizes)
