"""What the operators on a checkpoint's tensors are timed on: rows of an embedding table and their gradient,
projections through a shared weight with low-rank adapters of many requests beside it and their gradients, and the
merge of an adapter into a weight.

With `own` false every case is computed in its plain form, elementary torch operations in 32 bits rounded once at the
end; with `own` true by the calls that a user of this package makes.  Weights are as checkpoints hold them
(N(0, 0.02)), adapters as training leaves them (A like a fresh projection, B small, alpha / rank between a half and
two), tokens as text has them (a few ids make up most of it), activations N(0, 1).
"""
from __future__ import annotations

import math

import numpy as np
import torch

own = False

DTYPES = {"bf16": torch.bfloat16, "f16": torch.float16, "f32": torch.float32}
BYTES = {"bf16": 2, "f16": 2, "f32": 4}
ZIPF_SHIFT = 2.7                          # ranks of words in text: p(v) ~ 1 / (v + 2.7)


def listed():
    return [
        # the embedding of one new token while a model answers: latency alone
        dict(name="rows: 1 of 128256x4096", op="rows", tokens=1, rows=128256, dim=4096, dtype="bf16", scaled=False, grad=False),
        # the embeddings of a batch of prompts, a scaled FP32 table of an encoder with a large vocabulary
        dict(name="rows: 16384 of 250002x1024 f32", op="rows", tokens=16384, rows=250002, dim=1024, dtype="f32", scaled=True, grad=False),
        # a training step's embeddings and the table's dense gradient
        dict(name="rows + grad: 8192 of 128256x4096", op="rows", tokens=8192, rows=128256, dim=4096, dtype="bf16", scaled=False, grad=True),
        # the same for a small table of odd sizes in half precision, rows used many times over
        dict(name="rows + grad: 3001 of 997x250 f16", op="rows", tokens=3001, rows=997, dim=250, dtype="f16", scaled=True, grad=True),
        # one request of one token: a shared projection read once, one adapter beside it
        dict(name="project: 1 token, 4096x4096 r16", op="project", tokens=1, inp=4096, out=4096, rank=16, adapters=64, index="requests", dtype="bf16", grad=False),
        # a step of a server: 64 requests of a token each, most with an adapter of their own
        dict(name="project: 64 tokens, 4096x14336 r16, 48 adapters", op="project", tokens=64, inp=4096, out=14336, rank=16, adapters=48, index="mixed", dtype="bf16", grad=False),
        # a batch of prompts of several requests, ragged lengths, some of them without an adapter
        dict(name="project: 4096 tokens, 4096x4096 r32, 8 adapters", op="project", tokens=4096, inp=4096, out=4096, rank=32, adapters=8, index="requests", dtype="bf16", grad=False),
        # odd sizes in half precision, where no row starts on a boundary
        dict(name="project: 333 tokens, 777x1001 r5 f16, 5 adapters", op="project", tokens=333, inp=777, out=1001, rank=5, adapters=5, index="requests", dtype="f16", grad=False),
        # training several small adapters at once over one batch
        dict(name="project + grad: 2047 tokens, 1024x1024 r8, 4 adapters", op="project", tokens=2047, inp=1024, out=1024, rank=8, adapters=4, index="requests", dtype="bf16", grad=True),
        # training one adapter beside the widest projection of an 8B model
        dict(name="project + grad: 8192 tokens, 4096x14336 r64", op="project", tokens=8192, inp=4096, out=14336, rank=64, adapters=1, index="one", dtype="bf16", grad=True),
        # restoring a fine-tuned weight from its base and its adapter
        dict(name="merge: 14336x4096 r64", op="merge", inp=4096, out=14336, rank=64, dtype="bf16"),
        # the same for a small odd weight in half precision
        dict(name="merge: 1000x771 r5 f16", op="merge", inp=771, out=1000, rank=5, dtype="f16"),
    ]


def _log(rng, lo, hi):
    return max(lo, min(hi, round(math.exp(rng.uniform(math.log(lo), math.log(hi))))))


def _size(rng, lo, hi):
    """A size of the range: mostly what models have (multiples of 64), some odd ones."""
    n = _log(rng, lo, hi)
    return n if rng.random() < 0.3 or n < 64 else n // 64 * 64


def draw(rng):
    op = rng.choice(("rows", "project", "project", "merge"))
    if op == "rows":
        grad = rng.random() < 0.5
        return dict(op="rows", tokens=_log(rng, 1, 16384), rows=_log(rng, 100, 131072), dim=_size(rng, 8, 4096),
                    dtype=rng.choice(("bf16", "bf16", "f16", "f32")), scaled=rng.random() < 0.5, grad=grad)
    rank = rng.choice((1, 4, 5, 8, 16, 16, 32, 64, 100, 128))
    dtype = rng.choice(("bf16", "bf16", "f16"))
    if op == "merge":
        return dict(op="merge", inp=_size(rng, 64, 4096), out=_size(rng, 64, 14336), rank=rank, dtype=dtype)
    adapters = _log(rng, 1, 64)
    return dict(op="project", tokens=_log(rng, 1, 8192), inp=_size(rng, 64, 4096), out=_size(rng, 64, 8192), rank=rank, adapters=adapters,
                index=rng.choice(("requests", "requests", "mixed")), dtype=dtype, grad=rng.random() < 0.4)


def _generator(seed):
    g = torch.Generator(device="cuda")
    g.manual_seed(seed)
    return g


def _normal(g, shape, std, dtype):
    return (torch.randn(shape, generator=g, device="cuda", dtype=torch.float32) * std).to(dtype)


def _index(case, g, seed):
    """Which adapter each token's request has (-1: none)."""
    tokens, n, kind = case["tokens"], case["adapters"], case["index"]
    if kind == "one":
        return torch.zeros(tokens, dtype=torch.int32, device="cuda")
    if kind == "mixed":
        return torch.randint(-1 if n > 1 else 0, n, (tokens,), generator=g, device="cuda", dtype=torch.int32)
    rng = np.random.default_rng(seed)
    requests = max(1, min(tokens, n + n // 4))
    cuts = np.sort(rng.integers(0, tokens, requests - 1)) if requests > 1 else np.zeros(0, dtype=np.int64)
    whose = rng.integers(0, n, requests)
    whose[1::5] = -1
    runs = np.diff(np.concatenate(([0], cuts, [tokens])))
    return torch.from_numpy(np.repeat(whose, runs).astype(np.int32)).cuda()


def prepare(case, seed):
    g = _generator(seed)
    dtype = DTYPES[case["dtype"]]
    if case["op"] == "rows":
        rows, dim, tokens = case["rows"], case["dim"], case["tokens"]
        u = torch.rand(tokens, generator=g, device="cuda", dtype=torch.float64)
        ids = (ZIPF_SHIFT * (((rows + ZIPF_SHIFT) / ZIPF_SHIFT) ** u - 1)).to(torch.int64).clamp_(0, rows - 1)
        s = dict(op="rows", table=_normal(g, (rows, dim), 0.02, dtype), tokens=ids, scale=math.sqrt(dim) if case["scaled"] else 1.0, grad=case["grad"])
        if case["grad"]:
            s["table"].requires_grad_(True)
            s["dy"] = _normal(g, (tokens, dim), 1.0, dtype)
        return s
    inp, out, rank = case["inp"], case["out"], case["rank"]
    w = _normal(g, (out, inp), 0.02, dtype)
    if case["op"] == "merge":
        return dict(op="merge", w=w, a=_normal(g, (rank, inp), inp ** -0.5, dtype), b=_normal(g, (out, rank), 0.02, dtype), scale=0.5 + 1.5 * (seed % 4) / 3)
    n = case["adapters"]
    s = dict(op="project", w=w, x=_normal(g, (case["tokens"], inp), 1.0, dtype), a=_normal(g, (n, rank, inp), inp ** -0.5, dtype),
             b=_normal(g, (n, out, rank), 0.02, dtype), scale=0.5 + 1.5 * torch.rand(n, generator=g, device="cuda"), index=_index(case, g, seed), grad=case["grad"])
    if case["grad"]:
        for k in ("x", "a", "b"):
            s[k].requires_grad_(True)
        s["dy"] = _normal(g, (case["tokens"], out), 1.0, dtype)
    return s


def run(s):
    if own:
        return _own(s)
    with torch.no_grad():
        return {"rows": _plain_rows, "project": _plain_project, "merge": _plain_merge}[s["op"]](s)


def _own(s):
    from lmz_b200 import adapters, embed
    if s["op"] == "rows":
        y = embed.lookup(s["table"], s["tokens"], scale=s["scale"])
        if not s["grad"]:
            return {"y": y}
        return {"y": y, "dtable": torch.autograd.grad(y, s["table"], s["dy"])[0]}
    if s["op"] == "merge":
        return {"w": adapters.merge(s["w"], s["a"], s["b"], scale=s["scale"])}
    y = adapters.project(s["x"], s["w"], s["a"], s["b"], s["index"], scale=s["scale"])
    if not s["grad"]:
        return {"y": y}
    dx, da, db = torch.autograd.grad(y, (s["x"], s["a"], s["b"]), s["dy"])
    return {"y": y, "dx": dx, "da": da, "db": db}


def _plain_rows(s):
    table, tokens, scale = s["table"], s["tokens"], s["scale"]
    y = {"y": (table[tokens].float() * scale).to(table.dtype)}
    if s["grad"]:
        total = torch.zeros(table.shape, dtype=torch.float32, device="cuda")
        total.index_add_(0, tokens, s["dy"].float() * scale)
        y["dtable"] = total.to(table.dtype)
    return y


def _plain_project(s):
    x, w, a, b = s["x"].float(), s["w"].float(), s["a"].float(), s["b"].float()
    (n, rank, inp), out, dtype = a.shape, b.shape[1], s["x"].dtype
    every = torch.arange(n, device="cuda")
    factor = torch.where(s["index"].long()[:, None] == every, s["scale"], torch.zeros((), device="cuda"))    # [tokens, n]
    factor = factor.repeat_interleave(rank, 1)                                                             # [tokens, n * rank]
    down, up = a.reshape(n * rank, inp), b.permute(0, 2, 1).reshape(n * rank, out)
    h = (x @ down.t()) * factor
    y = {"y": (x @ w.t() + h @ up).to(dtype)}
    if s["grad"]:
        dy = s["dy"].float()
        dh = (dy @ up.t()) * factor
        y["dx"] = (dy @ w + dh @ down).to(dtype)
        y["da"] = (dh.t() @ x).reshape(n, rank, inp).to(dtype)
        y["db"] = (h.t() @ dy).reshape(n, rank, out).permute(0, 2, 1).contiguous().to(dtype)
    return y


def _plain_merge(s):
    return {"w": (s["w"].float() + s["scale"] * (s["b"].float() @ s["a"].float())).to(s["w"].dtype)}


def _distinct(rows, tokens):
    """How many different rows that many tokens name, on average."""
    v = np.arange(rows, dtype=np.float64)
    p = np.log((v + 1 + ZIPF_SHIFT) / (v + ZIPF_SHIFT)) / math.log((rows + ZIPF_SHIFT) / ZIPF_SHIFT)
    return float(np.sum(-np.expm1(tokens * np.log1p(-np.minimum(p, 1 - 1e-12)))))


def work(case):
    e = BYTES[case["dtype"]]
    if case["op"] == "rows":
        t, d = case["tokens"], case["dim"]
        moved = t * 8 + (_distinct(case["rows"], t) + t) * d * e
        if not case["grad"]:
            return {"bytes": moved, "flops": t * d}
        return {"bytes": moved + (t + case["rows"]) * d * e, "flops": 3 * t * d}
    i, o, r = case["inp"], case["out"], case["rank"]
    if case["op"] == "merge":
        return {"bytes": (2 * i * o + r * (i + o)) * e, "flops": 2 * i * o * r}
    t, used = case["tokens"], min(case["adapters"], case["tokens"])
    forward = {"bytes": (t * i + o * i + used * r * (i + o) + t * o) * e + t * 4, "flops": 2 * t * (i * o + r * (i + o))}
    if not case["grad"]:
        return forward
    # forwards as above; backwards dy, x, w and the factors again, dx and the gradients of all factors written
    return {"bytes": forward["bytes"] + (t * o + t * i + o * i + used * r * (i + o) + t * i + case["adapters"] * r * (i + o)) * e,
            "flops": 2 * t * (2 * i * o + 4 * r * (i + o))}


def exact(case, seed):
    """The definitions, adapter by adapter and in 64 bits."""
    s = prepare(case, seed)
    with torch.no_grad():
        if case["op"] == "rows":
            y = {"y": torch.index_select(s["table"], 0, s["tokens"]).double().mul_(s["scale"])}
            if case["grad"]:
                dy = s["dy"].double() * s["scale"]
                order = torch.argsort(s["tokens"])
                ids, counts = torch.unique_consecutive(s["tokens"][order], return_counts=True)
                sums = torch.zeros((ids.numel(), case["dim"]), dtype=torch.float64, device="cuda")
                sums.index_add_(0, torch.repeat_interleave(torch.arange(ids.numel(), device="cuda"), counts), dy[order])
                y["dtable"] = torch.zeros(s["table"].shape, dtype=torch.float64, device="cuda")
                y["dtable"][ids] = sums
            return y
        w, a, b = s["w"].double(), s["a"].double(), s["b"].double()
        if case["op"] == "merge":
            return {"w": torch.addmm(w, b, a, alpha=s["scale"])}
        x = s["x"].double()
        y = {"y": torch.mm(x, w.t())}
        if case["grad"]:
            dy = s["dy"].double()
            y |= {"dx": torch.mm(dy, w), "da": torch.zeros_like(a), "db": torch.zeros_like(b)}
        for i, scale in enumerate(s["scale"].double().tolist()):
            mine = torch.nonzero(s["index"] == i).flatten()
            if not mine.numel():
                continue
            h = torch.mm(x[mine], a[i].t())
            y["y"][mine] += scale * torch.mm(h, b[i].t())
            if case["grad"]:
                dh = torch.mm(dy[mine], b[i])
                y["dx"][mine] += scale * torch.mm(dh, a[i])
                y["da"][i] = scale * torch.mm(dh.t(), x[mine])
                y["db"][i] = scale * torch.mm(dy[mine].t(), h)
        return y
