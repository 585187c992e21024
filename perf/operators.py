"""Performance cases of the token-side operators: embedding, adapters, distillation.

A case is one call, or the forward or backward call of a step, that a program
with a token model around this library's Dense layers makes:

  embed_fwd     rows of an embedding table for a batch of tokens, scaled
                (welvet_hip_embedding_forward)
  embed_bwd     the table's gradient of a batch, or of two batches that follow
                one another, the second added to the first's
                (welvet_hip_embedding_backward)
  adapters_fwd  low-rank adapters added to a Dense layer's output, each row
                with its own adapter (welvet_hip_adapters_forward)
  adapters_bwd  their gradients (welvet_hip_adapters_backward)
  distill       the loss against a teacher's top logits and the gradient of
                the logits (welvet_hip_distill)

Activations, gradients and the teacher's logits are float32; tables, adapter
factors and the student's logits float32, float16 or bfloat16.
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


def listed():
    return [
        # the input of one decode step of 8 sequences: a call's latency
        {"name": "embed_fwd_bf16_32000x4096_n8", "op": "embed_fwd", "dtype": "bfloat16", "vocab": 32000, "dim": 4096,
         "n": 8, "pad": 0.0},
        # the input of a training batch of padded sequences
        {"name": "embed_fwd_f32_50257x1024_n16384", "op": "embed_fwd", "dtype": "float32", "vocab": 50257,
         "dim": 1024, "n": 16384, "pad": 0.1},
        # a small network whose sizes are nothing's multiple, its gradient over two batches
        {"name": "embed_bwd_1001x777_n100", "op": "embed_bwd", "vocab": 1001, "dim": 777, "n": 100, "pad": 0.0,
         "batches": 2},
        # the table's gradient of a training batch, tokens as skewed as text
        {"name": "embed_bwd_32000x4096_n16384", "op": "embed_bwd", "vocab": 32000, "dim": 4096, "n": 16384,
         "pad": 0.05, "batches": 1},
        # three requests on a small ragged layer
        {"name": "adapters_fwd_f32_1001x777_r5_n3", "op": "adapters_fwd", "dtype": "float32", "inn": 1001, "out": 777,
         "rank": 5, "count": 4, "n": 3, "mixed": True},
        # one decode step of 64 requests over 48 adapters beside the up projection
        {"name": "adapters_fwd_bf16_4096x11008_r16_n64", "op": "adapters_fwd", "dtype": "bfloat16", "inn": 4096,
         "out": 11008, "rank": 16, "count": 48, "n": 64, "mixed": True},
        # prefill of a few prompts, an adapter each
        {"name": "adapters_fwd_f16_4096x4096_r64_n2048", "op": "adapters_fwd", "dtype": "float16", "inn": 4096,
         "out": 4096, "rank": 64, "count": 4, "n": 2048, "mixed": False},
        # fine-tuning the two-layer MLP's first layer with one adapter in float32
        {"name": "adapters_bwd_f32_2048x8192_r8_n256", "op": "adapters_bwd", "dtype": "float32", "inn": 2048,
         "out": 8192, "rank": 8, "count": 1, "n": 256, "mixed": False},
        # a training step of eight tenants' adapters at once
        {"name": "adapters_bwd_bf16_4096x11008_r32_n8192", "op": "adapters_bwd", "dtype": "bfloat16", "inn": 4096,
         "out": 11008, "rank": 32, "count": 8, "n": 8192, "mixed": False},
        # a few tokens with loss and gradient, as in online distillation while decoding
        {"name": "distill_f32_32000_n4_k20", "op": "distill", "dtype": "float32", "vocab": 32000, "n": 4, "k": 20,
         "temp": 1.0, "rest": False, "grad": True},
        # a validation pass: the loss alone, prompts masked out
        {"name": "distill_f16_50257_n1000_k100", "op": "distill", "dtype": "float16", "vocab": 50257, "n": 1000,
         "k": 100, "temp": 1.0, "rest": True, "grad": False},
        # a training step over a large vocabulary: the largest
        {"name": "distill_bf16_131072_n4096_k64", "op": "distill", "dtype": "bfloat16", "vocab": 131072, "n": 4096,
         "k": 64, "temp": 2.0, "rest": False, "grad": True},
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def _size(rng, lo, hi):
    """A width: half of them multiples of 64, a quarter of 4, a quarter any."""
    while True:
        n = _log(rng, lo, hi)
        r = rng.random()
        n = max(lo, n // 64 * 64) if r < 0.5 else max(lo, n // 4 * 4) if r < 0.75 else n
        if n != 3072:
            return n


def draw(rng):
    op = rng.choice(("embed_fwd", "embed_bwd", "adapters_fwd", "adapters_bwd", "distill"))
    top = max(work(c)["bytes"] for c in listed())
    while True:
        c = {"op": op}
        if op != "embed_bwd":
            c["dtype"] = rng.choice(tuple(TYPES))
        if op.startswith("embed"):
            c.update(vocab=_size(rng, 1000, 131072), dim=_size(rng, 256, 8192), n=_log(rng, 1, 32768),
                     pad=rng.choice((0.0, 0.0, 0.1)))
            if op == "embed_bwd":
                c["batches"] = rng.choice((1, 2))
        elif op.startswith("adapters"):
            c.update(inn=_size(rng, 256, 11008), out=_size(rng, 256, 11008), rank=rng.choice((4, 8, 16, 16, 32, 64, 7, 20)),
                     count=_log(rng, 1, 64), n=_log(rng, 1, 8192), mixed=rng.random() < 0.5)
            if c["n"] * c["count"] * c["rank"] * (c["inn"] + c["out"]) > 2 ** 40:  # what the plain form multiplies
                continue
        else:
            c.update(vocab=_size(rng, 1000, 131072), n=_log(rng, 1, 4096), k=_log(rng, 1, 256),
                     temp=rng.choice((1.0, 2.0, 0.7)), rest=rng.random() < 0.5, grad=rng.random() < 0.6)
        if work(c)["bytes"] <= top:
            return c


def _rand(g, *shape):
    return torch.randn(*shape, device=DEV, generator=g)


def _tokens(case, g):
    """Tokens as skewed as text: rank k of a shuffled vocabulary with a frequency near 1/k, and padding (-1)."""
    n, vocab = case["n"], case["vocab"]
    u = torch.rand(n, device=DEV, generator=g)
    rank = torch.exp(u * math.log(vocab)).long().clamp_(max=vocab) - 1
    tok = torch.randperm(vocab, device=DEV, generator=g)[rank].to(torch.int32)
    return torch.where(torch.rand(n, device=DEV, generator=g) < case["pad"], torch.full_like(tok, -1), tok)


def prepare(case, seed):
    g = torch.Generator(device=DEV)
    g.manual_seed(seed)
    s = {"case": dict(case)}
    op, n = case["op"], case["n"]
    if op == "embed_fwd":
        s.update(table=(_rand(g, case["vocab"], case["dim"]) * 0.02).to(TYPES[case["dtype"]]),
                 tokens=_tokens(case, g), scale=math.sqrt(case["dim"]), out=torch.empty(n, case["dim"], device=DEV))
    elif op == "embed_bwd":
        s.update(tokens=[_tokens(case, g) for _ in range(case["batches"])], scale=math.sqrt(case["dim"]),
                 dout=[_rand(g, n, case["dim"]) * 1e-2 for _ in range(case["batches"])],
                 dtable=torch.empty(case["vocab"], case["dim"], device=DEV))
    elif op.startswith("adapters"):
        inn, out, rank, count = case["inn"], case["out"], case["rank"], case["count"]
        t = TYPES[case["dtype"]]
        s["down"] = (_rand(g, count, rank, inn) / math.sqrt(inn)).to(t)
        s["up"] = (_rand(g, count, rank, out) * 0.02).to(t)
        ranks = torch.full((count,), rank, dtype=torch.int32, device=DEV)
        few = torch.rand(count, device=DEV, generator=g) < 0.25  # a quarter of the adapters are of half the rank
        s["ranks"] = torch.where(few, ranks // 2, ranks)
        s["scales"] = torch.rand(count, device=DEV, generator=g) + 0.5
        ids = torch.randint(0, count, (n,), device=DEV, generator=g, dtype=torch.int32)
        if case["mixed"]:  # requests in any order, one in eight without an adapter
            ids = torch.where(torch.rand(n, device=DEV, generator=g) < 0.125, torch.full_like(ids, -1), ids)
        else:  # prompts one after the other
            ids = torch.sort(ids).values
        s.update(ids=ids, x=_rand(g, n, inn))
        if op == "adapters_fwd":
            s.update(base=_rand(g, n, out), y=torch.empty(n, out, device=DEV), h=torch.empty(n, rank, device=DEV))
        else:
            s.update(dy=_rand(g, n, out) * 1e-2, dxb=_rand(g, n, inn) * 1e-2)
            s["h"] = _down_rows(s, s["x"], s["down"])  # the forward's
            s.update(dx=torch.empty(n, inn, device=DEV), ddown=torch.empty(count, rank, inn, device=DEV),
                     dup=torch.empty(count, rank, out, device=DEV))
    else:
        vocab, k, temp = case["vocab"], min(case["k"], case["vocab"]), case["temp"]
        at = (torch.rand(n, k, device=DEV, generator=g) * (vocab // k)).long().clamp_(max=vocab // k - 1)
        at += torch.arange(k, device=DEV) * vocab // k  # one index a stretch of the vocabulary: all differ
        at = at.gather(1, torch.argsort(torch.rand(n, k, device=DEV, generator=g), 1))
        teacher = torch.sort(_rand(g, n, k) * 2 + 9, 1, descending=True).values
        z = _rand(g, n, vocab) * 1.5
        z.scatter_add_(1, at, teacher * 0.8 + _rand(g, n, k))  # a student that has learnt some of it
        weight = torch.rand(n, device=DEV, generator=g) + 0.5
        weight = torch.where(torch.rand(n, device=DEV, generator=g) < 0.15, torch.zeros_like(weight), weight)
        last = torch.randint(1, k + 1, (n, 1), device=DEV, generator=g)
        few = torch.rand(n, 1, device=DEV, generator=g) < 0.1  # some rows have fewer entries: the rest are absent
        at = torch.where(few & (torch.arange(k, device=DEV) >= last), torch.full_like(at, -1), at)
        s.update(logits=z.to(TYPES[case["dtype"]]), index=at.to(torch.int32), teacher=teacher, weight=weight)
        del z
        if case["rest"]:  # the teacher's own log-sum over its whole vocabulary
            s["lse"] = torch.logsumexp(teacher / temp, 1) + torch.rand(n, device=DEV, generator=g) * 0.5
        s["loss"] = torch.empty(n, device=DEV)
        if case["grad"]:
            s["dlogits"] = torch.empty_like(s["logits"])
    return s


# ---- the operators in elementary operations, in 32 bits

def _pick(s):
    """For each row: its adapter (0 where it has none), and which of the rank's rows count."""
    count, rank = s["down"].shape[0], s["down"].shape[1]
    none = (s["ids"] < 0) | (s["ids"] >= count)
    a = s["ids"].long().masked_fill(none, 0)
    return a, (torch.arange(rank, device=a.device) < s["ranks"][a][:, None]) & ~none[:, None]


def _down_rows(s, x, factor):
    """[n][rank]: each row's product with its own adapter's [rank][width] factor (all adapters' products, its own taken)."""
    a, live = _pick(s)
    count, rank, width = factor.shape
    all_h = (x @ factor.float().reshape(count * rank, width).t()).view(-1, count, rank)
    return all_h[torch.arange(x.shape[0], device=x.device), a] * live


def _spread(s, h):
    """[n][count * rank]: each row's values at its own adapter's place, zeros elsewhere."""
    a, live = _pick(s)
    wide = torch.zeros(h.shape[0], s["down"].shape[0], h.shape[1], device=h.device)
    wide[torch.arange(h.shape[0], device=h.device), a] = h * live
    return wide.view(h.shape[0], -1)


def _plain(s):
    case, op = s["case"], s["case"]["op"]
    if op == "embed_fwd":
        none = (s["tokens"] < 0) | (s["tokens"] >= case["vocab"])
        rows = s["table"][s["tokens"].long().masked_fill(none, 0)].float() * s["scale"]
        return rows.masked_fill(none[:, None], 0.0)
    if op == "embed_bwd":
        table = s["dtable"].zero_()
        for tokens, dout in zip(s["tokens"], s["dout"]):
            none = (tokens < 0) | (tokens >= case["vocab"])
            table.index_add_(0, tokens.long().masked_fill(none, 0), (dout * s["scale"]).masked_fill(none[:, None], 0.0))
        return table
    if op == "adapters_fwd":
        h = _down_rows(s, s["x"], s["down"])
        scale = s["scales"][_pick(s)[0]][:, None]
        y = s["base"] + _spread(s, h * scale) @ s["up"].float().reshape(-1, case["out"])
        return {"y": y, "h": h}
    if op == "adapters_bwd":
        scale = s["scales"][_pick(s)[0]][:, None]
        g = _down_rows(s, s["dy"], s["up"]) * scale
        wide = _spread(s, g)
        dx = s["dxb"] + wide @ s["down"].float().reshape(-1, case["inn"])
        return {"dx": dx, "ddown": (wide.t() @ s["x"]).view(s["ddown"].shape),
                "dup": (_spread(s, s["h"] * scale).t() @ s["dy"]).view(s["dup"].shape)}
    z, temp = s["logits"].float() / case["temp"], case["temp"]
    live = (s["index"] >= 0) & (s["index"] < case["vocab"])
    at = s["index"].long().masked_fill(~live, 0)
    top = (s["teacher"] / temp).masked_fill(~live, -math.inf)
    some = live.any(1, keepdim=True)
    if case["rest"]:
        logq = top - s["lse"][:, None]
    else:
        most = top.max(1, keepdim=True).values.masked_fill(~some, 0.0)
        logq = top - most - (top - most).exp().sum(1, keepdim=True).log()
    q = logq.exp().masked_fill(~live, 0.0)
    z = z - z.max(1, keepdim=True).values
    e = z.exp()
    total = e.sum(1, keepdim=True)
    logp = z.gather(1, at) - total.log()
    weight = s["weight"]
    loss = (q * (logq - logp)).masked_fill(~live, 0.0).sum(1) * (temp * temp) * weight
    if not case["grad"]:
        return {"loss": loss}
    d = e * (q.sum(1, keepdim=True) / total)
    d.scatter_add_(1, at, -q)
    d = d * (weight * temp)[:, None]
    return {"loss": loss, "dlogits": d.to(s["logits"].dtype)}


# ---- the framework's operators

def _workspace(s, nbytes):
    """A program keeps its workspace: made at the first call."""
    if "ws" not in s:
        s["ws"] = torch.empty(max(nbytes(), 16), dtype=torch.uint8, device=DEV)
    return s["ws"].data_ptr(), s["ws"].numel()


def _kernels(s):
    package = os.path.join(ROOT, "welvet.metal_amd")
    if package not in sys.path:
        sys.path.insert(0, package)
    import pywelvet as pw

    case, op = s["case"], s["case"]["op"]
    n, stream = case["n"], torch.cuda.current_stream().cuda_stream
    if op == "embed_fwd":
        pw.embedding_forward(IDS[case["dtype"]], case["vocab"], case["dim"], s["table"].data_ptr(),
                             s["tokens"].data_ptr(), n, s["out"].data_ptr(), scale=s["scale"], stream=stream)
        return s["out"]
    if op == "embed_bwd":
        vocab, dim = case["vocab"], case["dim"]
        ws = _workspace(s, lambda: pw.embedding_backward_bytes(vocab, dim, n))
        for i in range(case["batches"]):
            pw.embedding_backward(vocab, dim, s["tokens"][i].data_ptr(), n, s["dout"][i].data_ptr(),
                                  s["dtable"].data_ptr(), scale=s["scale"], accumulate=i > 0, ws=ws[0], ws_bytes=ws[1],
                                  stream=stream)
        return s["dtable"]
    if op.startswith("adapters"):
        if "adapters" not in s:
            s["adapters"] = pw.Adapters(IDS[case["dtype"]], case["count"], case["rank"], case["inn"], case["out"],
                                        s["down"].data_ptr(), s["up"].data_ptr(), d_ranks=s["ranks"].data_ptr(),
                                        d_scales=s["scales"].data_ptr())
        ad = s["adapters"]
        ws = _workspace(s, lambda: ad.workspace_bytes(n))
        if op == "adapters_fwd":
            ad.forward(s["x"].data_ptr(), s["ids"].data_ptr(), n, s["base"].data_ptr(), s["y"].data_ptr(),
                       d_h=s["h"].data_ptr(), ws=ws[0], ws_bytes=ws[1], stream=stream)
            return {"y": s["y"], "h": s["h"]}
        ad.backward(s["x"].data_ptr(), s["ids"].data_ptr(), n, s["h"].data_ptr(), s["dy"].data_ptr(),
                    d_dx_base=s["dxb"].data_ptr(), d_dx=s["dx"].data_ptr(), d_ddown=s["ddown"].data_ptr(),
                    d_dup=s["dup"].data_ptr(), ws=ws[0], ws_bytes=ws[1], stream=stream)
        return {"dx": s["dx"], "ddown": s["ddown"], "dup": s["dup"]}
    vocab, k = case["vocab"], s["index"].shape[1]
    ws = _workspace(s, lambda: pw.distill_bytes(IDS[case["dtype"]], n, vocab, k))
    pw.distill(IDS[case["dtype"]], n, vocab, s["logits"].data_ptr(), k, s["index"].data_ptr(), s["teacher"].data_ptr(),
               d_loss=s["loss"].data_ptr(), d_dlogits=s["dlogits"].data_ptr() if case["grad"] else None,
               temperature=case["temp"], d_weight=s["weight"].data_ptr(),
               d_teacher_lse=s["lse"].data_ptr() if case["rest"] else None, ws=ws[0], ws_bytes=ws[1], stream=stream)
    return {"loss": s["loss"], "dlogits": s["dlogits"]} if case["grad"] else {"loss": s["loss"]}


def run(state):
    return _kernels(state) if own else _plain(state)


# ---- the definitions in 64 bits, an adapter or a stretch of rows at a time

def exact(case, seed):
    s = prepare(case, seed)
    op, n = case["op"], case["n"]
    if op == "embed_fwd":
        out = torch.zeros(n, case["dim"], dtype=torch.float64, device=DEV)
        at = ((s["tokens"] >= 0) & (s["tokens"] < case["vocab"])).nonzero()[:, 0]
        out[at] = s["table"].index_select(0, s["tokens"][at].long()).double() * s["scale"]
        return out
    if op == "embed_bwd":
        out = torch.zeros(case["vocab"], case["dim"], dtype=torch.float64, device=DEV)
        for tokens, dout in zip(s["tokens"], s["dout"]):
            at = ((tokens >= 0) & (tokens < case["vocab"])).nonzero()[:, 0]
            tok = tokens[at].long()
            out.scatter_add_(0, tok[:, None].expand(-1, case["dim"]), dout[at].double() * s["scale"])
        return out
    if op.startswith("adapters"):
        fwd = op == "adapters_fwd"
        y = (s["base"] if fwd else s["dxb"]).double()
        h = torch.zeros(n, case["rank"], dtype=torch.float64, device=DEV)
        ddown, dup = torch.zeros(s["down"].shape, dtype=torch.float64, device=DEV), torch.zeros(
            s["up"].shape, dtype=torch.float64, device=DEV)
        for a, (rank, scale) in enumerate(zip(s["ranks"].tolist(), s["scales"].double().tolist())):
            rows = (s["ids"] == a).nonzero()[:, 0]
            if not rank or not len(rows):
                continue
            down, up, x = s["down"][a, :rank].double(), s["up"][a, :rank].double(), s["x"][rows].double()
            if fwd:
                part = x @ down.t().contiguous()
                h[rows, :rank] = part
                y[rows] += scale * (part @ up)
            else:
                dy = s["dy"][rows].double()
                part = scale * (dy @ up.t().contiguous())
                y[rows] += part @ down
                ddown[a, :rank] = part.t().contiguous() @ x
                dup[a, :rank] = scale * (s["h"][rows, :rank].double().t().contiguous() @ dy)
        return {"y": y, "h": h} if fwd else {"dx": y, "ddown": ddown, "dup": dup}
    losses, grads = [], []
    temp = case["temp"]
    for r in range(0, n, 256):
        z = s["logits"][r:r + 256].double() / temp
        logp = torch.log_softmax(z, 1)
        at, teacher = s["index"][r:r + 256].long(), s["teacher"][r:r + 256].double() / temp
        teacher = torch.where(at >= 0, teacher, torch.full_like(teacher, -math.inf))
        norm = s["lse"][r:r + 256].double() if case["rest"] else torch.logsumexp(teacher, 1)
        q = torch.exp(teacher - norm[:, None])
        w = s["weight"][r:r + 256].double()
        term = torch.xlogy(q, q) - q * logp.gather(1, at.clamp(min=0))
        losses.append(w * temp ** 2 * term.sum(1))
        if case["grad"]:
            d = logp.exp() * q.sum(1, keepdim=True)
            d.scatter_add_(1, at.clamp(min=0), -q)
            grads.append(d * (w * temp)[:, None])
    loss = torch.cat(losses)
    return {"loss": loss, "dlogits": torch.cat(grads)} if case["grad"] else {"loss": loss}


def work(case):
    n, op = case["n"], case["op"]
    size = TYPES[case["dtype"]].itemsize if "dtype" in case else 4
    if op.startswith("embed"):
        vocab, dim = case["vocab"], case["dim"]
        # rows of a table that n tokens of this skew name: sum over its ranks of the chance to be drawn at all
        step = max(1, vocab // 2048)
        rows = sum(step * -math.expm1(-n * math.log1p(1.0 / (k + step / 2)) / math.log(vocab))
                   for k in range(0, vocab, step)) if vocab > 1 else 1
        rows = min(n, vocab, rows) * (1 - case["pad"])
        if op == "embed_fwd":
            return {"bytes": 4 * n + rows * dim * size + 4 * n * dim, "flops": n * dim}
        b = case["batches"]
        return {"bytes": b * (4 * n + 4 * n * dim) + 4 * vocab * dim + (b - 1) * 8 * rows * dim, "flops": b * n * dim}
    if op.startswith("adapters"):
        used = case["count"] * -math.expm1(n * math.log1p(-1.0 / case["count"])) if case["count"] > 1 else 1
        factors = used * case["rank"] * (case["inn"] + case["out"])
        if op == "adapters_fwd":
            return {"bytes": 4 * n * (case["inn"] + 2 * case["out"] + case["rank"] + 1) + factors * size,
                    "flops": 2 * n * case["rank"] * (case["inn"] + case["out"])}
        grads = 4 * case["count"] * case["rank"] * (case["inn"] + case["out"])
        return {"bytes": 4 * n * (3 * case["inn"] + case["out"] + case["rank"] + 1) + factors * size + grads,
                "flops": 4 * n * case["rank"] * (case["inn"] + case["out"])}
    return {"bytes": n * case["vocab"] * size * (2 if case["grad"] else 1) + n * (case["k"] * 8 + 8),
            "flops": n * case["vocab"] * (6 if case["grad"] else 4)}
