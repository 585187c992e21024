"""A token model whose layers multiply in 8-bit integers, trained and answering.

tokens -> embedding -> SwiGLU (gate, up, down) -> output layer -> logits, every
layer an Int8Layer with a scale a token and a scale a channel.  A training step
keeps nothing of the forward but rows in 8 bits (the layers' inputs as their
products took them, gate and up):

    embedding_forward -> gate.forward(rows) -> up.product(rows)
    -> rows8_swiglu (gate8, up8, h8) -> down.product(h8) -> head.forward(rows)
    -> distill (loss and gradient)
    -> rows8_backward (head, down) -> rows8_swiglu_backward
    -> rows8_backward (gate, up) -> embedding_backward

and applies SGD to master weights in float32, from which the layers are mounted
again.  Afterwards prompts are continued token by token, each answer the largest
logit that LogitRules leaves: no token of the prompt's own, fewer repetitions.

    python examples/int8_mlp.py [steps]
"""
import os
import sys

import numpy as np

sys.path.insert(0, os.path.join(os.path.dirname(os.path.abspath(__file__)), "..", "welvet.metal_amd"))
sys.path.insert(0, os.path.dirname(os.path.abspath(__file__)))
import pywelvet  # noqa: E402
from distill_adapters import Array, zeros  # noqa: E402

F32 = pywelvet.DTYPE["float32"]
LINEAR = pywelvet.ACT["linear"]
VOCAB, DIM, INTER, TOP = 300, 72, 200, 8
ROWS, RATE = 130, 0.5


class Rows:
    """Rows in 8 bits on the device."""

    def __init__(self, n, width):
        self.width, stride = width, pywelvet.rows8_stride(width)
        self.codes, self.scales = zeros(n, stride, dtype=np.int8), zeros(n)
        self.desc = pywelvet.rows8(self.codes.ptr, stride, self.scales.ptr)

    def values(self):
        return self.codes.get()[:, :self.width].astype(np.float64) * self.scales.get().astype(np.float64)[:, None]


class Layer:
    """Master weights in float32, their int8 layer and their gradient."""

    def __init__(self, W):
        self.W, self.dw = Array(W), zeros(*W.shape)
        self.out, self.inn = W.shape
        self.mounted = None
        self.mount()

    def mount(self):
        if self.mounted is not None:
            self.mounted.close()
        self.mounted = pywelvet.Int8Layer.from_device(self.W.ptr, self.inn, self.out)

    def step(self, rate):
        self.W.put(self.W.get() - np.float32(rate) * self.dw.get())
        self.mount()


class Model:
    def __init__(self, seed=5):
        rng = np.random.default_rng(seed)
        weights = lambda out, inn: rng.normal(0, inn ** -0.5, (out, inn)).astype(np.float32)  # noqa: E731
        self.table = Array(rng.normal(0, 1, (VOCAB, DIM)).astype(np.float32))
        self.gate, self.up = Layer(weights(INTER, DIM)), Layer(weights(INTER, DIM))
        self.down, self.head = Layer(weights(DIM, INTER)), Layer(weights(VOCAB, DIM))
        self.layers = (self.gate, self.up, self.down, self.head)
        n = ROWS
        self.x, self.g, self.u, self.y, self.logits = (zeros(n, w) for w in (DIM, INTER, INTER, DIM, VOCAB))
        self.x8, self.gate8, self.up8, self.h8, self.y8 = (Rows(n, w) for w in (DIM, INTER, INTER, INTER, DIM))
        self.dy, self.dh, self.dx, self.dx2 = (zeros(n, w) for w in (DIM, INTER, DIM, DIM))
        self.tokens, self.index, self.teacher = zeros(n, dtype=np.int32), zeros(n, TOP, dtype=np.int32), zeros(n, TOP)
        self.loss, self.weight = zeros(n), Array(np.full(n, 1.0 / n, np.float32))
        self.bytes = max([layer.mounted.workspace_bytes(n) for layer in self.layers] +
                         [pywelvet.rows8_backward_bytes(F32, n, layer.inn, layer.out) for layer in self.layers] +
                         [pywelvet.embedding_backward_bytes(VOCAB, DIM, n), pywelvet.distill_bytes(F32, n, VOCAB, TOP)])
        self.ws = zeros(self.bytes, dtype=np.uint8)
        self.on = dict(ws=self.ws.ptr, ws_bytes=self.bytes)

    def forward(self, n):
        """Logits of the n tokens in self.tokens; the rows that a backward reads."""
        pywelvet.embedding_forward(F32, VOCAB, DIM, self.table.ptr, self.tokens.ptr, n, self.x.ptr)
        self.gate.mounted.forward(F32, n, self.x.ptr, rows=self.x8.desc, d_post=self.g.ptr, **self.on)
        self.up.mounted.product(F32, n, self.x8.desc, d_post=self.u.ptr, **self.on)
        pywelvet.rows8_swiglu(F32, n, INTER, self.g.ptr, self.u.ptr, self.gate8.desc, self.up8.desc, self.h8.desc)
        self.down.mounted.product(F32, n, self.h8.desc, d_post=self.y.ptr, **self.on)
        self.head.mounted.forward(F32, n, self.y.ptr, rows=self.y8.desc, d_post=self.logits.ptr, **self.on)

    def backward(self, n):
        """Gradients of the n rows' loss, from dlogits in the logits' place."""
        def layer(which, d_out, rows, d_in):
            pywelvet.rows8_backward(LINEAR, F32, n, which.inn, which.out, d_out.ptr, x=rows.desc, layer=which.mounted,
                                    d_dx=d_in.ptr, d_dw=which.dw.ptr, **self.on)
        layer(self.head, self.logits, self.y8, self.dy)
        layer(self.down, self.dy, self.h8, self.dh)
        # gate's and up's gradients take the places of their projections
        pywelvet.rows8_swiglu_backward(F32, n, INTER, self.gate8.desc, self.up8.desc, self.dh.ptr, self.g.ptr, self.u.ptr)
        layer(self.gate, self.g, self.x8, self.dx)
        layer(self.up, self.u, self.x8, self.dx2)

    def step(self, tokens, index, teacher, rate=RATE):
        """One SGD step; the mean loss before it."""
        for to, a in ((self.tokens, tokens), (self.index, index), (self.teacher, teacher)):
            to.put(a)
        self.forward(ROWS)
        pywelvet.distill(F32, ROWS, VOCAB, self.logits.ptr, TOP, self.index.ptr, self.teacher.ptr, self.loss.ptr,
                         self.logits.ptr, 1.0, self.weight.ptr, **self.on)
        self.backward(ROWS)
        for dx in (self.dx, self.dx2):  # the table's own SGD step, in place
            pywelvet.embedding_backward(VOCAB, DIM, self.tokens.ptr, ROWS, dx.ptr, self.table.ptr, -rate, True, **self.on)
        for layer in self.layers:
            layer.step(rate)
        return float(self.loss.get().sum())

    def answer(self, prompts, length):
        """Each prompt continued by `length` tokens."""
        n = len(prompts)
        history = np.full((n, max(map(len, prompts)) + length), -1, np.int32)
        at = np.array([len(p) for p in prompts], np.int32)
        for t, p in enumerate(prompts):
            history[t, :len(p)] = p
        words = (VOCAB + 31) // 32
        allowed = np.ones((n, words * 32), bool)
        for t, p in enumerate(prompts):
            allowed[t, list(p)] = False  # a grammar of a kind: none of the prompt's own tokens
        masks = Array(np.packbits(allowed, axis=1, bitorder="little").view(np.uint32))
        d_history, d_len, d_prompt = Array(history), Array(at), Array(at)
        repetition, presence = Array(np.full(n, 1.2, np.float32)), Array(np.full(n, 0.5, np.float32))
        rules = pywelvet.LogitRules(history=history.shape[1], d_history=d_history.ptr, d_history_len=d_len.ptr,
                                    d_prompt_len=d_prompt.ptr, d_repetition=repetition.ptr, d_presence=presence.ptr,
                                    masks=n, d_masks=masks.ptr)
        tokens = np.zeros(ROWS, np.int32)
        for _ in range(length):
            tokens[:n] = history[np.arange(n), at - 1]
            self.tokens.put(tokens)
            self.forward(n)
            rules.apply(F32, n, VOCAB, self.logits.ptr, self.logits.ptr)  # in place
            history[np.arange(n), at] = self.logits.get()[:n].argmax(1)
            at += 1
            d_history.put(history)
            d_len.put(at)
        return [history[t, len(p):at[t]].tolist() for t, p in enumerate(prompts)]

    def close(self):
        for layer in self.layers:
            layer.mounted.close()


def batch(rng):
    """Tokens, and a teacher that follows each with one of a few others."""
    tokens = rng.integers(0, VOCAB, ROWS).astype(np.int32)
    index = ((tokens[:, None] * 7 + np.arange(TOP) * 11 + 1) % VOCAB).astype(np.int32)
    teacher = np.tile(np.linspace(8, 1, TOP), (ROWS, 1)).astype(np.float32)
    return tokens, index, teacher


def run(steps=20, say=print):
    """The steps' losses, and the prompts' answers after them."""
    rng, model = np.random.default_rng(11), Model()
    losses = []
    for i in range(steps):
        losses.append(model.step(*batch(rng)))
        if i % 5 == 0 or i == steps - 1:
            say(f"step {i:3d}  loss {losses[-1]:.4f}")
    prompts = [[1, 2, 3], [40], [7, 7, 250, 9, 8]]
    answers = model.answer(prompts, 6)
    for p, a in zip(prompts, answers):
        say(f"{p} -> {a}")
    model.close()
    return losses, prompts, answers


if __name__ == "__main__":
    run(int(sys.argv[1]) if len(sys.argv) > 1 else 20)
