"""Two tenants' adapters on one frozen FP8 layer, distilled and then served.

A small language model of one projection: tokens -> embedding (trained) ->
output layer (a packed FP8 E4M3 store, frozen) + the tenant's low-rank adapter
(trained) -> logits.  Each tenant has a teacher of its own, of which only the
top logits of every position are kept.  A training step is

    embedding_forward -> Session.forward_device -> Adapters.forward
    -> distill (loss and gradient)
    -> the frozen layer's dX -> Adapters.backward -> embedding_backward

on one stream, the activations on the device throughout; the embedding takes
its SGD step in place (a gradient added with scale -rate).  Afterwards the
trained table is mounted as a BFloat16 store and one batch of single tokens
from both tenants is answered through embedding_store_forward.

    python examples/distill_adapters.py [steps]
"""
import ctypes as C
import os
import sys

import numpy as np

sys.path.insert(0, os.path.join(os.path.dirname(os.path.abspath(__file__)), "..", "welvet.metal_amd"))
import pywelvet  # noqa: E402

F32, BF16, FP8 = (pywelvet.DTYPE[name] for name in ("float32", "bfloat16", "fp8e4m3"))
LINEAR = pywelvet.ACT["linear"]
VOCAB, DIM, RANK, TOP, TENANTS = 512, 96, 8, 16, 2
ROWS, TEMPERATURE, RATE = 192, 2.0, 3.0


class Array:
    """A numpy array's copy in device memory."""
    hip = None

    def __init__(self, a):
        if Array.hip is None:
            pywelvet.init()
            Array.hip = C.CDLL("libamdhip64.so.7")  # the runtime the library runs on
            Array.hip.hipMemcpy.argtypes = [C.c_void_p, C.c_void_p, C.c_size_t, C.c_int]
            Array.hip.hipFree.argtypes = [C.c_void_p]
        a = np.ascontiguousarray(a)
        self.shape, self.dtype, self.nbytes = a.shape, a.dtype, a.nbytes
        p = C.c_void_p()
        self._ok(Array.hip.hipMalloc(C.byref(p), C.c_size_t(max(a.nbytes, 16))))
        self.ptr = p.value
        self.put(a)

    @staticmethod
    def _ok(rc):
        if rc:
            raise RuntimeError(f"HIP error {rc}")

    def put(self, a):
        a = np.ascontiguousarray(a, self.dtype)
        assert a.shape == self.shape
        self._ok(Array.hip.hipMemcpy(self.ptr, a.ctypes.data, self.nbytes, 1))

    def get(self):  # waits for the null stream, which this example runs on
        out = np.empty(self.shape, self.dtype)
        self._ok(Array.hip.hipMemcpy(out.ctypes.data, self.ptr, self.nbytes, 2))
        return out

    def __del__(self):
        if getattr(self, "ptr", None):
            Array.hip.hipFree(self.ptr)
            self.ptr = None


def zeros(*shape, dtype=np.float32):
    return Array(np.zeros(shape, dtype))


def make(seed=7):
    """The frozen layer's weights, the starting table and the teachers' rows."""
    rng = np.random.default_rng(seed)
    W = rng.normal(0, DIM ** -0.5, (VOCAB, DIM)).astype(np.float32)
    table = rng.normal(0, 1, (VOCAB, DIM)).astype(np.float32)
    bend = 0.5 * rng.normal(0, 1, (TENANTS, VOCAB, 4)) @ rng.normal(0, DIM ** -0.5, (TENANTS, 4, DIM))
    teacher = 2 * (table[None].astype(np.float64) @ (W + bend).swapaxes(1, 2))  # [tenant][token][vocab]
    return rng, W, table, teacher


def top(teacher, tokens, ids):
    """The teachers' largest logits at the rows: indices and values."""
    z = teacher[ids, tokens]
    index = np.argsort(-z, axis=1)[:, :TOP].astype(np.int32)
    return index, np.take_along_axis(z, index, axis=1).astype(np.float32)


class Student:
    def __init__(self, W, table, rng):
        self.layer = pywelvet.Session(W, ROWS, LINEAR, FP8)
        # the frozen store's transpose gives the layer's dX on the device
        self.back = pywelvet.Session(np.ascontiguousarray(self.layer.export_f32().T), ROWS, LINEAR, FP8)
        self.table = Array(table)
        self.down = Array(rng.normal(0, DIM ** -0.5, (TENANTS, RANK, DIM)).astype(np.float32))
        self.up = zeros(TENANTS, RANK, VOCAB)  # at first the adapters add nothing
        self.adapters = pywelvet.Adapters(F32, TENANTS, RANK, DIM, VOCAB, self.down.ptr, self.up.ptr)
        self.bytes = max(self.adapters.workspace_bytes(ROWS),
                         pywelvet.embedding_backward_bytes(VOCAB, DIM, ROWS),
                         pywelvet.distill_bytes(F32, ROWS, VOCAB, TOP))
        self.ws = zeros(self.bytes, dtype=np.uint8)
        self.x, self.h = zeros(ROWS, DIM), zeros(ROWS, RANK)
        self.pre, self.base, self.logits = zeros(ROWS, VOCAB), zeros(ROWS, VOCAB), zeros(ROWS, VOCAB)
        self.loss = zeros(ROWS)
        self.dpre, self.dx = zeros(ROWS, DIM), zeros(ROWS, DIM)
        self.ddown, self.dup = zeros(TENANTS, RANK, DIM), zeros(TENANTS, RANK, VOCAB)
        self.tokens, self.ids = zeros(ROWS, dtype=np.int32), zeros(ROWS, dtype=np.int32)
        self.index, self.values = zeros(ROWS, TOP, dtype=np.int32), zeros(ROWS, TOP)
        self.weight = Array(np.full(ROWS, 1.0 / ROWS, np.float32))  # the mean over the rows

    def step(self, tokens, ids, index, values):
        """One SGD step; the rows' mean loss before it."""
        for to, a in ((self.tokens, tokens), (self.ids, ids), (self.index, index), (self.values, values)):
            to.put(a)
        ws = dict(ws=self.ws.ptr, ws_bytes=self.bytes)
        pywelvet.embedding_forward(F32, VOCAB, DIM, self.table.ptr, self.tokens.ptr, ROWS, self.x.ptr)
        self.layer.forward_device(self.x.ptr, self.pre.ptr, self.base.ptr)
        self.adapters.forward(self.x.ptr, self.ids.ptr, ROWS, self.base.ptr, self.logits.ptr, self.h.ptr, **ws)
        # the gradient takes the logits' place
        pywelvet.distill(F32, ROWS, VOCAB, self.logits.ptr, TOP, self.index.ptr, self.values.ptr, self.loss.ptr,
                         self.logits.ptr, TEMPERATURE, self.weight.ptr, **ws)
        self.back.forward_device(self.logits.ptr, self.dpre.ptr, self.dx.ptr)
        self.adapters.backward(self.x.ptr, self.ids.ptr, ROWS, self.h.ptr, self.logits.ptr, self.dx.ptr, self.dx.ptr,
                               self.ddown.ptr, self.dup.ptr, **ws)
        pywelvet.embedding_backward(VOCAB, DIM, self.tokens.ptr, ROWS, self.dx.ptr, self.table.ptr, -RATE, True, **ws)
        self.down.put(self.down.get() - RATE * self.ddown.get())
        self.up.put(self.up.get() - RATE * self.dup.get())
        return float(self.loss.get().sum())

    def serve(self, tokens, ids):
        """Logits of one token a request, from the table mounted as a store."""
        n = len(tokens)
        with pywelvet.Session(self.table.get(), 1, LINEAR, BF16) as store:
            d_tokens, d_ids, x = Array(np.asarray(tokens, np.int32)), Array(np.asarray(ids, np.int32)), zeros(n, DIM)
            pre, y = zeros(n, VOCAB), zeros(n, VOCAB)
            pywelvet.embedding_store_forward(store, d_tokens.ptr, n, x.ptr)
            self.layer.forward_noalloc(n, x.ptr, pre.ptr, y.ptr)
            self.adapters.forward(x.ptr, d_ids.ptr, n, y.ptr, y.ptr, ws=self.ws.ptr, ws_bytes=self.bytes)
            return y.get()

    def close(self):
        self.layer.close()
        self.back.close()


def run(steps=60, say=print):
    """Losses of the steps, and how often the served answer is the teacher's
    before and after them."""
    rng, W, table, teacher = make()
    student = Student(W, table, rng)
    asked, who = np.repeat(rng.integers(0, VOCAB, 32), TENANTS), np.tile(np.arange(TENANTS), 32)
    agree = lambda: float((student.serve(asked, who).argmax(1) == teacher[who, asked].argmax(1)).mean())  # noqa: E731
    before, losses = agree(), []
    for i in range(steps):
        tokens, ids = rng.integers(0, VOCAB, ROWS), rng.integers(0, TENANTS, ROWS)
        losses.append(student.step(tokens, ids, *top(teacher, tokens, ids)))
        if i % 10 == 0 or i == steps - 1:
            say(f"step {i:3d}  loss {losses[-1]:.4f}")
    after = agree()
    say(f"answers as the teachers': {before:.0%} -> {after:.0%} of {len(asked)}")
    student.close()
    return losses, before, after


if __name__ == "__main__":
    run(int(sys.argv[1]) if len(sys.argv) > 1 else 60)
