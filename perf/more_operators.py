"""Performance cases of the 8-bit activation operators and of the logits' rules.

A case is one call, or the calls of one layer's step, that a program makes
around this library's Dense layers when activations are held in 8 bits, or
when it answers from logits:

  int8_forward    a layer whose product runs in 8-bit integers, a scale for
                  each token and each output channel
                  (welvet_hip_int8_mount_device, welvet_hip_int8_forward)
  checkpoint      a Dense layer's input and pre-activations kept in 8 bits and
                  its backward pass from them: dpre, dx, dw
                  (welvet_hip_rows8_store, welvet_hip_rows8_backward)
  swiglu          SwiGLU's product with its two inputs kept in 8 bits, and its
                  backward pass from them (welvet_hip_rows8_swiglu,
                  welvet_hip_rows8_swiglu_backward)
  logits          repetition, frequency and presence penalties, biases and
                  grammar masks on logits (welvet_hip_logits_rules)

Activations, gradients and logits are float32, float16 or bfloat16; weights'
gradients float32.
"""
import math
import os
import sys

import torch

own = False

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
DEV = "cuda:0"
TYPES = {"float32": torch.float32, "float16": torch.float16, "bfloat16": torch.bfloat16}
IDS = {"float32": 1, "float16": 2, "bfloat16": 3}
ACTS = {"linear": -1, "relu": 0, "silu": 1, "gelu": 2, "tanh": 3}
OPEN = (0.0005, 0.02, 0.5, 0.97)  # shares of the vocabulary that grammar masks leave, in turn


def listed():
    return [
        # one token's up projection: a call's latency and the weights' bytes
        {"name": "int8_forward_bf16_4096x11008_n1", "op": "int8_forward", "dtype": "bfloat16", "inn": 4096,
         "out": 11008, "n": 1, "act": "linear", "bias": False},
        # three rows through a small layer whose sizes are nothing's multiple
        {"name": "int8_forward_f32_1001x777_n3", "op": "int8_forward", "dtype": "float32", "inn": 1001, "out": 777,
         "n": 3, "act": "tanh", "bias": True},
        # one decode step of 64 requests: the down projection
        {"name": "int8_forward_bf16_11008x4096_n64", "op": "int8_forward", "dtype": "bfloat16", "inn": 11008,
         "out": 4096, "n": 64, "act": "linear", "bias": False},
        # prefill of a batch of prompts: the up projection
        {"name": "int8_forward_f16_4096x11008_n8192", "op": "int8_forward", "dtype": "float16", "inn": 4096,
         "out": 11008, "n": 8192, "act": "silu", "bias": True},
        # a step of a small ragged layer, the first one of its network: no dx
        {"name": "checkpoint_f16_1001x777_n100", "op": "checkpoint", "dtype": "float16", "inn": 1001, "out": 777,
         "n": 100, "act": "gelu", "dx": False},
        # the two-layer MLP's first layer in float32
        {"name": "checkpoint_f32_2048x8192_n256", "op": "checkpoint", "dtype": "float32", "inn": 2048, "out": 8192,
         "n": 256, "act": "tanh", "dx": True},
        # a training batch of a large layer
        {"name": "checkpoint_bf16_4096x11008_n8192", "op": "checkpoint", "dtype": "bfloat16", "inn": 4096,
         "out": 11008, "n": 8192, "act": "silu", "dx": True},
        # a few rows of a ragged width
        {"name": "swiglu_f32_1001_n100", "op": "swiglu", "dtype": "float32", "width": 1001, "n": 100},
        # a training batch of the large MLP
        {"name": "swiglu_bf16_11008_n8192", "op": "swiglu", "dtype": "bfloat16", "width": 11008, "n": 8192},
        # the next token of 4 requests: penalties for what was said, a few biases
        {"name": "logits_f32_32000_n4", "op": "logits", "dtype": "float32", "vocab": 32000, "n": 4, "history": 500,
         "biases": 8, "masks": 0},
        # 64 requests with long histories, most of them under a grammar
        {"name": "logits_bf16_131072_n64", "op": "logits", "dtype": "bfloat16", "vocab": 131072, "n": 64,
         "history": 8192, "biases": 0, "masks": 12},
        # every position of a batch of drafts, rows on every alignment
        {"name": "logits_f16_50257_n1000", "op": "logits", "dtype": "float16", "vocab": 50257, "n": 1000,
         "history": 1024, "biases": 100, "masks": 40},
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def _size(rng, lo, hi):
    """A width: half of them multiples of 64, a quarter of 4, a quarter any."""
    n = _log(rng, lo, hi)
    r = rng.random()
    return max(lo, n // 64 * 64) if r < 0.5 else max(lo, n // 4 * 4) if r < 0.75 else n


def draw(rng):
    op = rng.choice(("int8_forward", "int8_forward", "checkpoint", "checkpoint", "swiglu", "logits"))
    most = [work(c) for c in listed() if c["op"] == op]
    while True:
        c = {"op": op, "dtype": rng.choice(tuple(TYPES))}
        if op == "swiglu":
            c.update(width=_size(rng, 256, 16384), n=_log(rng, 1, 8192))
        elif op == "logits":
            c.update(vocab=_size(rng, 1000, 152064), n=_log(rng, 1, 1000), history=_log(rng, 1, 16384),
                     biases=rng.choice((0, 1, 8, 100, 300)), masks=rng.choice((0, 0, 1, 12, 40)))
        else:
            c.update(inn=_size(rng, 256, 11008), out=_size(rng, 256, 11008), n=_log(rng, 1, 8192),
                     act=rng.choice(tuple(ACTS)))
            c.update(bias=rng.random() < 0.5) if op == "int8_forward" else c.update(dx=rng.random() < 0.7)
        w = work(c)
        if all(w[k] <= max(m[k] for m in most) for k in w):
            return c


def _rand(g, *shape):
    return torch.randn(*shape, device=DEV, generator=g)


def _wild(g, n, width):
    """Activations of a layer: some columns ten times the others, rows of their own size."""
    col = torch.where(torch.rand(width, device=DEV, generator=g) < 0.01, 10.0, 1.0)
    return _rand(g, n, width) * col * torch.exp(_rand(g, n, 1) * 0.5)


def _package():
    package = os.path.join(ROOT, "welvet.metal_amd")
    if package not in sys.path:
        sys.path.insert(0, package)
    import pywelvet

    return pywelvet


def _layer(s, g, inn, out, act, bias):
    """A layer's weights in 8 bits, a scale a channel: what a mounted one holds."""
    w = _rand(g, out, inn) / math.sqrt(inn)
    bias = _rand(g, out) * 0.1 if bias else None
    s["w8"], s["bias"] = _codes(w), bias
    if own:
        pw = _package()
        s["layer"] = pw.Int8Layer.from_device(w.data_ptr(), inn, out, ACTS[act],
                                              None if bias is None else bias.double().cpu().numpy())


def _stride(width):
    return (width + 15) // 16 * 16


def _rows8(n, width):
    """Room for n rows in 8 bits."""
    return torch.empty(n, _stride(width), dtype=torch.int8, device=DEV), torch.empty(n, device=DEV)


def prepare(case, seed):
    g = torch.Generator(device=DEV)
    g.manual_seed(seed)
    s = {"case": dict(case)}
    op, n, t = case["op"], case["n"], TYPES[case["dtype"]]
    if op == "int8_forward":
        inn, out = case["inn"], case["out"]
        _layer(s, g, inn, out, case["act"], case["bias"])
        s.update(x=_wild(g, n, inn).to(t), y=torch.empty(n, out, dtype=t, device=DEV))
    elif op == "checkpoint":
        inn, out = case["inn"], case["out"]
        if case["dx"]:
            _layer(s, g, inn, out, case["act"], False)
            s["dx"] = torch.empty(n, inn, dtype=t, device=DEV)
        s.update(x=_wild(g, n, inn).to(t), pre=_wild(g, n, out).to(t), dy=(_rand(g, n, out) * 1e-2).to(t),
                 x8=_rows8(n, inn), pre8=_rows8(n, out), dpre=torch.empty(n, out, dtype=t, device=DEV),
                 dw=torch.empty(out, inn, device=DEV))
    elif op == "swiglu":
        w = case["width"]
        s.update(gate=_wild(g, n, w).to(t), up=_wild(g, n, w).to(t), dh=(_rand(g, n, w) * 1e-2).to(t),
                 gate8=_rows8(n, w), up8=_rows8(n, w))
        s.update({k: torch.empty(n, w, dtype=t, device=DEV) for k in ("h", "dgate", "dup")})
    else:
        vocab, most = case["vocab"], case["history"]
        rank = torch.exp(torch.rand(n, most, device=DEV, generator=g) * math.log(vocab)).long().clamp_(max=vocab) - 1
        said = torch.randperm(vocab, device=DEV, generator=g)[rank].to(torch.int32)  # as skewed as text
        length = (torch.rand(n, device=DEV, generator=g) * (most + 1)).to(torch.int32).clamp_(max=most)
        s.update(logits=(_rand(g, n, vocab) * 3).to(t), history=said, length=length,
                 prompt=(length * torch.rand(n, device=DEV, generator=g)).to(torch.int32),
                 repetition=1 + torch.rand(n, device=DEV, generator=g) * 0.3,
                 frequency=torch.rand(n, device=DEV, generator=g) * 0.2,
                 presence=torch.rand(n, device=DEV, generator=g) * 0.5, out=torch.empty(n, vocab, dtype=t, device=DEV))
        k = min(case["biases"], vocab)
        if k:  # one index a stretch of the vocabulary; some rows have fewer
            at = (torch.rand(n, k, device=DEV, generator=g) * (vocab // k)).long().clamp_(max=vocab // k - 1)
            at += torch.arange(k, device=DEV) * vocab // k
            at = torch.where(torch.rand(n, k, device=DEV, generator=g) < 0.1, torch.full_like(at, -1), at)
            s.update(bias_index=at.to(torch.int32), bias=_rand(g, n, k) * 4)
        if case["masks"]:
            m, words = case["masks"], (vocab + 31) // 32
            share = torch.tensor(OPEN, device=DEV)[torch.arange(m, device=DEV) % len(OPEN)]
            bits = torch.rand(m, words * 32, device=DEV, generator=g) < share[:, None]
            value = (bits.view(m, words, 32).long() << torch.arange(32, device=DEV)).sum(2)
            s["masks"] = torch.where(value >= 2 ** 31, value - 2 ** 32, value).to(torch.int32)
            at = torch.arange(n, device=DEV, dtype=torch.int32) % (m + m // 4 + 1)  # some rows are under none
            s["mask"] = torch.where(at < m, at, torch.full_like(at, -1))
    return s


# ---- the operators in elementary operations, in 32 bits (codes next to a border in 64)

def _codes(x):
    """A row's values in 8 bits: codes, as floats, and the row's scale, its largest magnitude over 127."""
    x = x.float()
    scale = (x.abs().amax(1).double() / 127).float()
    code = (x.double() / scale.double()[:, None]).round_().nan_to_num_(0.0, 0.0, 0.0).clamp_(-127, 127)
    return code.float(), scale


def _values(codes):
    return codes[0] * codes[1][:, None]


def _act(x, act):
    if act == "relu":
        return x.clamp(min=0)
    if act == "silu":
        return x * torch.sigmoid(x)
    if act == "gelu":
        return 0.5 * x * (1 + torch.tanh(0.7978845608028654 * (x + 0.044715 * x * x * x)))
    return torch.tanh(x) if act == "tanh" else x


def _act_prime(x, act):
    if act == "relu":
        return (x > 0).to(x.dtype)
    if act == "silu":
        z = torch.sigmoid(x)
        return z * (1 + x * (1 - z))
    if act == "gelu":
        t = torch.tanh(0.7978845608028654 * (x + 0.044715 * x * x * x))
        return 0.5 * (1 + t) + 0.5 * x * (1 - t * t) * (0.7978845608028654 * (1 + 3 * 0.044715 * x * x))
    return 1 - torch.tanh(x) ** 2 if act == "tanh" else torch.ones_like(x)


def _plain(s):
    case, op, n = s["case"], s["case"]["op"], s["case"]["n"]
    t = TYPES[case["dtype"]]
    if op == "int8_forward":
        codes, scale = _codes(s["x"])
        y = (codes @ s["w8"][0].t()) * scale[:, None] * s["w8"][1]
        if s["bias"] is not None:
            y = y + s["bias"]
        return _act(y, case["act"]).to(t)
    if op == "checkpoint":
        x, pre = _values(_codes(s["x"])), _values(_codes(s["pre"]))
        dpre = s["dy"].float() * _act_prime(pre, case["act"])
        r = {"dpre": dpre.to(t), "dw": dpre.t() @ x}
        if case["dx"]:
            r["dx"] = ((dpre * s["w8"][1]) @ s["w8"][0]).to(t)
        return r
    if op == "swiglu":
        gate, up, dh = s["gate"].float(), s["up"].float(), s["dh"].float()
        h = gate * torch.sigmoid(gate) * up
        gate, up = _values(_codes(gate)), _values(_codes(up))
        z = torch.sigmoid(gate)
        return {"h": h.to(t), "dgate": (dh * up * (z * (1 + gate * (1 - z)))).to(t), "dup": (dh * (gate * z)).to(t)}
    vocab, z = case["vocab"], s["logits"].float()
    place = torch.arange(case["history"], device=DEV)
    live = place < s["length"][:, None]
    said = live & (place >= s["prompt"][:, None])
    at = s["history"].long()
    seen = torch.zeros(n, vocab, device=DEV).scatter_add_(1, at, live.float()) > 0
    count = torch.zeros(n, vocab, device=DEV).scatter_add_(1, at, said.float())
    r = s["repetition"][:, None]
    z = torch.where(seen, torch.where(z > 0, z / r, z * r), z)
    z = z - s["frequency"][:, None] * count - s["presence"][:, None] * (count > 0)
    if "bias" in s:
        none = s["bias_index"] < 0
        z.scatter_add_(1, s["bias_index"].long().masked_fill(none, 0), s["bias"].masked_fill(none, 0.0))
    if "masks" in s:
        v = torch.arange(vocab, device=DEV)
        allowed = (s["masks"][:, v // 32] >> (v % 32)) & 1
        shut = (allowed[s["mask"].clamp(min=0).long()] == 0) & (s["mask"] >= 0)[:, None]
        z = z.masked_fill(shut, -math.inf)
    return z.to(t)


# ---- the framework's operators

def _kernels(s):
    pw = _package()
    case, op, n = s["case"], s["case"]["op"], s["case"]["n"]
    t, stream = IDS[case["dtype"]], torch.cuda.current_stream().cuda_stream

    def rows(name):
        codes, scales = s[name]
        return pw.rows8(codes.data_ptr(), codes.stride(0), scales.data_ptr())

    if op == "int8_forward":
        if "ws" not in s:  # a program keeps its workspace
            s["ws"] = torch.empty(max(s["layer"].workspace_bytes(n), 16), dtype=torch.uint8, device=DEV)
        s["layer"].forward(t, n, s["x"].data_ptr(), d_post=s["y"].data_ptr(), ws=s["ws"].data_ptr(),
                           ws_bytes=s["ws"].numel(), stream=stream)
        return s["y"]
    if op == "checkpoint":
        inn, out = case["inn"], case["out"]
        if "ws" not in s:
            s["ws"] = torch.empty(max(pw.rows8_backward_bytes(t, n, inn, out), 16), dtype=torch.uint8, device=DEV)
        pw.rows8_store(t, n, inn, s["x"].data_ptr(), rows("x8"), stream=stream)
        pw.rows8_store(t, n, out, s["pre"].data_ptr(), rows("pre8"), stream=stream)
        pw.rows8_backward(ACTS[case["act"]], t, n, inn, out, s["dy"].data_ptr(), pre=rows("pre8"), x=rows("x8"),
                          layer=s["layer"] if case["dx"] else None, d_dpre=s["dpre"].data_ptr(),
                          d_dx=s["dx"].data_ptr() if case["dx"] else None, d_dw=s["dw"].data_ptr(),
                          ws=s["ws"].data_ptr(), ws_bytes=s["ws"].numel(), stream=stream)
        return {k: s[k] for k in (("dpre", "dw", "dx") if case["dx"] else ("dpre", "dw"))}
    if op == "swiglu":
        w = case["width"]
        pw.rows8_swiglu(t, n, w, s["gate"].data_ptr(), s["up"].data_ptr(), gate=rows("gate8"), up=rows("up8"),
                        d_h=s["h"].data_ptr(), stream=stream)
        pw.rows8_swiglu_backward(t, n, w, rows("gate8"), rows("up8"), s["dh"].data_ptr(), s["dgate"].data_ptr(),
                                 s["dup"].data_ptr(), stream=stream)
        return {"h": s["h"], "dgate": s["dgate"], "dup": s["dup"]}
    if "rules" not in s:
        k = s["bias"].shape[1] if "bias" in s else 0
        s["rules"] = pw.LogitRules(
            history=s["history"].shape[1], d_history=s["history"].data_ptr(), d_history_len=s["length"].data_ptr(),
            d_prompt_len=s["prompt"].data_ptr(), d_repetition=s["repetition"].data_ptr(),
            d_frequency=s["frequency"].data_ptr(), d_presence=s["presence"].data_ptr(), biases=k,
            d_bias_index=s["bias_index"].data_ptr() if k else None, d_bias=s["bias"].data_ptr() if k else None,
            masks=case["masks"], d_masks=s["masks"].data_ptr() if "masks" in s else None,
            d_mask_id=s["mask"].data_ptr() if "masks" in s else None)
    s["rules"].apply(t, n, case["vocab"], s["logits"].data_ptr(), s["out"].data_ptr(), stream=stream)
    return s["out"]


def run(state):
    return _kernels(state) if own else _plain(state)


# ---- the definitions in 64 bits

def _exact_codes(x):
    """Codes and scales of rows: the scale is kept in 32 bits, the code is the whole number nearest to the quotient."""
    x = x.double()
    scale = (x.abs().max(1).values / 127).float().double()
    code = torch.zeros_like(x)
    some = scale > 0
    code[some] = torch.clamp(torch.round(x[some] / scale[some][:, None]), -127, 127)
    return code, scale


def _exact_sigmoid(x):
    e = torch.exp(-x.abs())
    return torch.where(x >= 0, 1 / (1 + e), e / (1 + e))


def _exact_act(x, act, prime):
    if act == "linear":
        return torch.ones_like(x) if prime else x
    if act == "relu":
        return torch.heaviside(x, torch.zeros_like(x)) if prime else torch.maximum(x, torch.zeros_like(x))
    if act == "silu":
        z = _exact_sigmoid(x)
        return z + x * z * (1 - z) if prime else x * z
    if act == "tanh":
        return 1 / torch.cosh(x.clamp(-300, 300)) ** 2 if prime else torch.tanh(x)
    a = math.sqrt(2 / math.pi)  # gelu by its tanh form: x sigmoid(2 u)
    z = _exact_sigmoid(2 * a * (x + 0.044715 * x ** 3))
    return z + x * z * (1 - z) * 2 * a * (1 + 0.134145 * x ** 2) if prime else x * z


def exact(case, seed):
    s = prepare(case, seed)
    op, n = case["op"], case["n"]
    if op == "int8_forward":
        xc, xs = _exact_codes(s["x"])
        y = xc @ s["w8"][0].double().t().contiguous()
        y = y * torch.outer(xs, s["w8"][1].double())
        if s["bias"] is not None:
            y += s["bias"].double()
        return _exact_act(y, case["act"], False)
    if op == "checkpoint":
        xc, xs = _exact_codes(s["x"])
        pc, ps = _exact_codes(s["pre"])
        dpre = s["dy"].double() * _exact_act(pc * ps[:, None], case["act"], True)
        r = {"dpre": dpre, "dw": dpre.t().contiguous() @ (xc * xs[:, None])}
        if case["dx"]:
            r["dx"] = dpre @ (s["w8"][0].double() * s["w8"][1].double()[:, None])
        return r
    if op == "swiglu":
        gate, up, dh = s["gate"].double(), s["up"].double(), s["dh"].double()
        h = _exact_act(gate, "silu", False) * up
        (gc, gs), (uc, us) = _exact_codes(gate), _exact_codes(up)
        gate, up = gc * gs[:, None], uc * us[:, None]
        return {"h": h, "dgate": dh * up * _exact_act(gate, "silu", True), "dup": dh * _exact_act(gate, "silu", False)}
    vocab, out = case["vocab"], s["logits"].double()
    length, prompt = s["length"].tolist(), s["prompt"].tolist()
    mask = s["mask"].tolist() if "mask" in s else [-1] * n
    for r in range(n):
        z = out[r]
        said = s["history"][r, :length[r]].long()
        tokens = torch.unique(said)
        rep = s["repetition"][r].double()
        old = z[tokens]
        z[tokens] = torch.where(old > 0, old / rep, old * rep)
        tokens, count = torch.unique(said[prompt[r]:], return_counts=True)
        z[tokens] -= count.double() * s["frequency"][r].double() + s["presence"][r].double()
        if "bias" in s:
            there = s["bias_index"][r] >= 0
            z[s["bias_index"][r][there].long()] += s["bias"][r][there].double()
        if mask[r] >= 0:
            words = s["masks"][mask[r]].long() & 0xffffffff
            bits = torch.stack([(words >> b) & 1 for b in range(32)], 1).reshape(-1)[:vocab]
            z[bits == 0] = -math.inf
    return out


def work(case):
    n, op, size = case["n"], case["op"], TYPES[case["dtype"]].itemsize
    if op == "int8_forward":
        inn, out = case["inn"], case["out"]
        return {"bytes": size * n * (inn + out) + inn * out + (12 if case["bias"] else 4) * out, "flops": 2 * n * inn * out}
    if op == "checkpoint":
        inn, out = case["inn"], case["out"]
        b = size * n * (inn + 3 * out) + n * (inn + out + 8) + 4 * inn * out
        if case["dx"]:
            b += size * n * inn + inn * out + 4 * out
        return {"bytes": b, "flops": (4 if case["dx"] else 2) * n * inn * out}
    if op == "swiglu":
        return {"bytes": n * (case["width"] * (6 * size + 2) + 8), "flops": 40 * n * case["width"]}
    vocab, m = case["vocab"], case["masks"]
    read = 1.0  # of the logits: what a mask shuts is not read
    if m:
        ids = [OPEN[i % len(OPEN)] for i in range(m)] + [1.0] * (m // 4 + 1)
        read = sum(ids[r % len(ids)] for r in range(n)) / n
    b = n * (vocab * size * (1 + read) + 2 * case["history"] + 20 + 8 * case["biases"]) + m * ((vocab + 31) // 32) * 4
    return {"bytes": b, "flops": n * vocab}
