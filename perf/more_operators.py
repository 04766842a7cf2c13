"""What the operators of a layer around a checkpoint's weights are timed on: root-mean-square norms with the residual's
addition and their gradients, the same with an output in 8 bits, products with bias, activation, factor and residual in
their epilogue and their gradients, products of 8-bit rows and weights, and products of rows with their experts' weights
and their gradients.

With `own` false every case is computed in its plain form, elementary torch operations in 32 bits rounded once at the
end; with `own` true by the calls that a user of this package makes.  Weights are as checkpoints hold them
(N(0, 0.02), norms' around one), activations N(0, 1), the residual stream wider and with a few large channels, as trained
models have them; experts get unequal shares of the rows, and some get none.
"""
from __future__ import annotations

import math

import numpy as np
import torch

own = False

DTYPES = {"bf16": torch.bfloat16, "f16": torch.float16, "f32": torch.float32}
BYTES = {"bf16": 2, "f16": 2, "f32": 4}
E4M3_MOST = 448.0                         # the largest number of 8 bits with 4 of exponent and 3 of mantissa
EPS = 1e-5


def listed():
    return [
        # one new token while a model answers: the residual's addition and the norm in front of a block, latency alone
        dict(name="norm: 1x4096", op="norm", tokens=1, dim=4096, dtype="bf16", residual=True, grad=False),
        # a training step's norms over a batch, the residual stream in and out
        dict(name="norm + grad: 16384x4096", op="norm", tokens=16384, dim=4096, dtype="bf16", residual=True, grad=True),
        # an encoder in FP32, rows of an odd size
        dict(name="norm + grad: 3001x997 f32", op="norm", tokens=3001, dim=997, dtype="f32", residual=False, grad=True),
        # a batch of prompts in front of products in 8 bits
        dict(name="norm to 8 bits: 8192x8192", op="norm8", tokens=8192, dim=8192, dtype="bf16", residual=True),
        # the same for a few requests of a token each, in half precision
        dict(name="norm to 8 bits: 16x4096 f16", op="norm8", tokens=16, dim=4096, dtype="f16", residual=True),
        # one token through the gated half of a feed-forward block: the weight read once
        dict(name="linear: 1 token 4096x14336", op="linear", tokens=1, inp=4096, out=14336, dtype="bf16", bias=False, activation="silu", times=True,
             residual=False, grad=False),
        # training with biases in half precision, odd sizes, where no row starts on a boundary
        dict(name="linear + grad: 333 tokens 777x1001 f16", op="linear", tokens=333, inp=777, out=1001, dtype="f16", bias=True, activation="gelu", times=False,
             residual=True, grad=True),
        # training the widest projection of an 8B model, gated
        dict(name="linear + grad: 8192 tokens 4096x14336", op="linear", tokens=8192, inp=4096, out=14336, dtype="bf16", bias=False, activation="silu", times=True,
             residual=False, grad=True),
        # requests of a token each through a block's last projection in 8 bits, back into the residual stream
        dict(name="linear of 8 bits: 16 tokens 14336x4096", op="linear8", tokens=16, inp=14336, out=4096, bias=False, activation="none", residual=True),
        # a batch of prompts through the widest projection in 8 bits
        dict(name="linear of 8 bits: 8192 tokens 4096x14336", op="linear8", tokens=8192, inp=4096, out=14336, bias=True, activation="silu", residual=False),
        # a server's step with experts: a few rows each, their weights read once
        dict(name="experts: 128 rows of 64, 2048x1408", op="experts", rows=128, experts=64, spare=0, inp=2048, out=1408, dtype="bf16", activation="silu", times=True,
             grad=False),
        # training experts over a batch, ragged shares, a padded end
        dict(name="experts + grad: 16384 rows of 16, 2048x4096", op="experts", rows=16384, experts=16, spare=100, inp=2048, out=4096, dtype="bf16", activation="none",
             times=False, grad=True),
    ]


def _log(rng, lo, hi):
    return max(lo, min(hi, round(math.exp(rng.uniform(math.log(lo), math.log(hi))))))


def _size(rng, lo, hi):
    """A size of the range: mostly what models have (multiples of 64), some odd ones."""
    n = _log(rng, lo, hi)
    return n if rng.random() < 0.3 or n < 64 else n // 64 * 64


def draw(rng):
    op = rng.choice(("norm", "norm8", "linear", "linear", "linear8", "experts", "experts"))
    dtype = rng.choice(("bf16", "bf16", "f16"))
    if op in ("norm", "norm8"):
        c = dict(op=op, tokens=_log(rng, 1, 16384), dim=_size(rng, 8, 8192), dtype=rng.choice((dtype, dtype, dtype, "f32")), residual=rng.random() < 0.7)
        return c if op == "norm8" else c | dict(grad=rng.random() < 0.5)
    activation = rng.choice(("none", "relu", "silu", "gelu", "gelu_tanh"))
    inp, out = _size(rng, 64, 4096), _size(rng, 64, 14336)
    if op == "linear":
        return dict(op=op, tokens=_log(rng, 1, 8192), inp=inp, out=out, dtype=dtype, bias=rng.random() < 0.5, activation=activation, times=rng.random() < 0.4,
                    residual=rng.random() < 0.4, grad=rng.random() < 0.4)
    if op == "linear8":
        return dict(op=op, tokens=_log(rng, 1, 8192), inp=inp, out=out, bias=rng.random() < 0.5, activation=activation, residual=rng.random() < 0.4)
    return dict(op=op, rows=_log(rng, 1, 8192), experts=_log(rng, 2, 64), spare=rng.choice((0, 0, 50)), inp=_size(rng, 64, 2048), out=_size(rng, 64, 4096), dtype=dtype,
                activation=activation, times=rng.random() < 0.4, grad=rng.random() < 0.4)


def _generator(seed):
    g = torch.Generator(device="cuda")
    g.manual_seed(seed)
    return g


def _normal(g, shape, std, dtype):
    return (torch.randn(shape, generator=g, device="cuda", dtype=torch.float32) * std).to(dtype)


def _stream(g, tokens, dim, dtype):
    """A residual stream: every hundredth channel ten times as wide."""
    wide = torch.where(torch.rand(dim, generator=g, device="cuda") < 0.01, 20.0, 2.0)
    return (torch.randn((tokens, dim), generator=g, device="cuda", dtype=torch.float32) * wide).to(dtype)


def _in_8_bits(v):
    """Rows as numbers of 8 bits and a scale each."""
    scale = (v.abs().amax(1) / E4M3_MOST).clamp_min(2.0 ** -126)
    return (v / scale[:, None]).to(torch.float8_e4m3fn), scale


def _counts(case, seed):
    """How many rows each expert has: shares that differ by a factor of e more or less."""
    rng = np.random.default_rng(seed)
    p = np.exp(0.8 * rng.standard_normal(case["experts"]))
    p[3::7] = 0                           # (nobody's favourite)
    return rng.multinomial(case["rows"], p / p.sum())


def prepare(case, seed):
    g = _generator(seed)
    if case["op"] in ("norm", "norm8"):
        dtype, shape = DTYPES[case["dtype"]], (case["tokens"], case["dim"])
        s = dict(op=case["op"], x=_normal(g, shape, 1.0, dtype) if case["residual"] else _stream(g, *shape, dtype),
                 residual=_stream(g, *shape, dtype) if case["residual"] else None, weight=(1 + 0.2 * _normal(g, case["dim"], 1.0, torch.float32)).to(dtype),
                 grad=case.get("grad", False))
        if s["grad"]:
            s["dy"] = _normal(g, shape, 1.0, dtype)
            s["ds"] = _normal(g, shape, 1.0, dtype) if case["residual"] else None
        trained = ("x", "residual", "weight")
    elif case["op"] == "experts":
        dtype, rows, inp, out = DTYPES[case["dtype"]], case["rows"] + case["spare"], case["inp"], case["out"]
        counts = _counts(case, seed)
        s = dict(op="experts", x=_normal(g, (rows, inp), 1.0, dtype), weight=_normal(g, (case["experts"], out, inp), 0.02, dtype),
                 offsets=torch.from_numpy(np.concatenate(([0], np.cumsum(counts))).astype(np.int32)).cuda(), most=int(counts.max()),
                 activation=case["activation"], times=_normal(g, (rows, out), 1.0, dtype) if case["times"] else None, grad=case["grad"])
        if s["grad"]:
            s["dy"] = _normal(g, (rows, out), 1.0, dtype)
        trained = ("x", "weight", "times")
    else:
        tokens, inp, out = case["tokens"], case["inp"], case["out"]
        dtype = DTYPES[case.get("dtype", "bf16")]
        s = dict(op=case["op"], x=_normal(g, (tokens, inp), 1.0, dtype), weight=_normal(g, (out, inp), 0.02, dtype),
                 bias=_normal(g, out, 0.1, dtype) if case["bias"] else None, activation=case["activation"],
                 times=_normal(g, (tokens, out), 1.0, dtype) if case.get("times") else None,
                 residual=_stream(g, tokens, out, dtype) if case["residual"] else None, grad=case.get("grad", False))
        if case["op"] == "linear8":
            for k in ("x", "weight"):
                s[k], s[k + "_scale"] = _in_8_bits(s[k].float())
        if s["grad"]:
            s["dy"] = _normal(g, (tokens, out), 1.0, dtype)
        trained = ("x", "weight", "bias", "times", "residual")
    if s["grad"]:
        s["trained"] = [k for k in trained if s[k] is not None]
        for k in s["trained"]:
            s[k].requires_grad_(True)
    return s


def run(s):
    if own:
        return _own(s)
    with torch.no_grad():
        return {"norm": _plain_norm, "norm8": _plain_norm8, "linear": _plain_linear, "linear8": _plain_linear8, "experts": _plain_experts}[s["op"]](s)


def _own(s):
    from lmz_b200 import experts, linear, norms
    activation = None if s.get("activation") == "none" else s.get("activation")
    if s["op"] == "norm8":
        if s["residual"] is None:
            q, scale = norms.rms_norm_8bit(s["x"], s["weight"], eps=EPS)
            return {"q": q, "scale": scale}
        q, scale, stream = norms.rms_norm_8bit(s["x"], s["weight"], s["residual"], eps=EPS)
        return {"q": q, "scale": scale, "stream": stream}
    if s["op"] == "linear8":
        return {"y": linear.project_8bit(s["x"], s["x_scale"], s["weight"], s["weight_scale"], bias=s["bias"], activation=activation, residual=s["residual"],
                                         dtype=torch.bfloat16)}
    if s["op"] == "norm":
        if s["residual"] is None:
            y = {"y": norms.rms_norm(s["x"], s["weight"], eps=EPS)}
        else:
            y = dict(zip(("y", "stream"), norms.rms_norm(s["x"], s["weight"], s["residual"], eps=EPS)))
    elif s["op"] == "linear":
        y = {"y": linear.project(s["x"], s["weight"], bias=s["bias"], activation=activation, times=s["times"], residual=s["residual"])}
    else:
        y = {"y": experts.project(s["x"], s["weight"], s["offsets"], activation=activation, times=s["times"])}
    if s["grad"]:
        given = [s["dy"]] + ([s["ds"]] if "stream" in y else [])
        y |= zip(("d" + k for k in s["trained"]), torch.autograd.grad(list(y.values()), [s[k] for k in s["trained"]], given))
    return y


def _plain_norm(s):
    x, w, dtype = s["x"].float(), s["weight"].float(), s["x"].dtype
    y = {}
    if s["residual"] is not None:
        y["stream"] = (x + s["residual"].float()).to(dtype)
        x = y["stream"].float()
    r = torch.rsqrt((x * x).mean(1, keepdim=True) + EPS)
    y["y"] = (x * r * w).to(dtype)
    if s["grad"]:
        dy, n = s["dy"].float(), x * r
        d = dy * w
        dx = r * (d - n * (d * n).mean(1, keepdim=True))
        if "stream" in y:
            dx = dx + s["ds"].float()
            y["dresidual"] = dx.to(dtype)
        y["dx"] = dx.to(dtype)
        y["dweight"] = (dy * n).sum(0).to(dtype)
    return y


def _plain_norm8(s):
    x, y = s["x"].float(), {}
    if s["residual"] is not None:
        y["stream"] = (x + s["residual"].float()).to(s["x"].dtype)
        x = y["stream"].float()
    v = x * torch.rsqrt((x * x).mean(1, keepdim=True) + EPS) * s["weight"].float()
    y["q"], y["scale"] = _in_8_bits(v)
    return y


def _act(kind, z):
    """The activation and its derivative."""
    if kind == "none":
        return z, torch.ones((), device="cuda")
    if kind == "relu":
        return z * (z > 0), (z > 0).float()
    if kind == "silu":
        e = 1 / (1 + torch.exp(-z))
        return z * e, e * (1 + z * (1 - e))
    if kind == "gelu":
        c = 0.5 * (1 + torch.erf(z * math.sqrt(0.5)))
        return z * c, c + z * torch.exp(-0.5 * z * z) / math.sqrt(2 * math.pi)
    k = math.sqrt(2 / math.pi)
    t = torch.tanh(k * (z + 0.044715 * z * z * z))
    return 0.5 * z * (1 + t), 0.5 * (1 + t) + 0.5 * z * (1 - t * t) * k * (1 + 3 * 0.044715 * z * z)


def _epilogue(s, z, dtype):
    """The result of the sums z; with gradients also the gradient of z, and those of what stands in the epilogue."""
    a, da = _act(s["activation"], z)
    v = a
    times, residual = s.get("times"), s.get("residual")
    if times is not None:
        v = v * times.float()
    if residual is not None:
        v = v + residual.float()
    y, dz = {"y": v.to(dtype)}, None
    if s.get("grad"):
        dy = s["dy"].float()
        if residual is not None:
            y["dresidual"] = s["dy"].clone()
        dz = dy * da
        if times is not None:
            y["dtimes"] = (dy * a).to(dtype)
            dz = dz * times.float()
        if s.get("bias") is not None:
            y["dbias"] = dz.sum(0).to(dtype)
    return y, dz


def _plain_linear(s):
    x, w, dtype = s["x"].float(), s["weight"].float(), s["x"].dtype
    z = x @ w.t()
    if s["bias"] is not None:
        z = z + s["bias"].float()
    y, dz = _epilogue(s, z, dtype)
    if s["grad"]:
        y["dx"], y["dweight"] = (dz @ w).to(dtype), (dz.t() @ x).to(dtype)
    return y


def _plain_linear8(s):
    z = (s["x"].float() @ s["weight"].float().t()) * s["x_scale"][:, None] * s["weight_scale"]
    if s["bias"] is not None:
        z = z + s["bias"].float()
    return _epilogue(s, z, torch.bfloat16)[0]


def _plain_experts(s):
    """Every expert's rows beside the others', padded with zeros to the longest, and batched products of them."""
    x, w, offsets, dtype = s["x"].float(), s["weight"].float(), s["offsets"].long(), s["x"].dtype
    rows = torch.arange(x.shape[0], device="cuda")
    whose = torch.bucketize(rows, offsets[1:], right=True).clamp_max_(w.shape[0] - 1)
    has = (rows < offsets[-1])[:, None]
    places = offsets[:-1, None] + torch.arange(s["most"], device="cuda")               # [experts, most]
    live = (places < offsets[1:, None])[..., None]
    places = places.clamp_max(x.shape[0] - 1)
    zero = torch.zeros((), device="cuda")
    apart = lambda v: torch.where(live, v[places], zero)                              # noqa: E731
    back = lambda v: torch.where(has, v[whose, (rows - offsets[whose]).clamp_max(s["most"] - 1)], zero)   # noqa: E731
    xs = apart(x)
    y, dz = _epilogue(s, back(xs @ w.transpose(1, 2)), dtype)
    y["y"] = torch.where(has, y["y"], torch.zeros((), dtype=dtype, device="cuda"))
    if s["grad"]:
        if "dtimes" in y:
            y["dtimes"] = torch.where(has, y["dtimes"], torch.zeros((), dtype=dtype, device="cuda"))
        ds = apart(dz)
        y["dx"], y["dweight"] = back(ds @ w).to(dtype), (ds.transpose(1, 2) @ xs).to(dtype)
    return y


def work(case):
    if case["op"] in ("norm", "norm8"):
        e, n = BYTES[case["dtype"]], case["tokens"] * case["dim"]
        read = n * e * (2 if case["residual"] else 1) + case["dim"] * e
        written = n * e * (1 if case["residual"] else 0) + (n + 4 * case["tokens"] if case["op"] == "norm8" else n * e)
        if not case.get("grad"):
            return {"bytes": read + written, "flops": 6 * n}
        # backwards dy, the normed tensor and the stream's gradient read, one gradient written (the residual's is the same tensor)
        return {"bytes": read + written + n * e * (4 if case["residual"] else 3) + 2 * case["dim"] * e, "flops": 16 * n}
    inp, out = case["inp"], case["out"]
    if case["op"] == "experts":
        t, n = case["rows"], case["experts"]
        used = n * -math.expm1(t * math.log1p(-1 / n))
    else:
        t, n, used = case["tokens"], 1, 1
    if case["op"] == "linear8":
        return {"bytes": t * inp + out * inp + 4 * (t + out) + t * out * (4 if case["residual"] else 2) + (2 * out if case["bias"] else 0), "flops": 2 * t * inp * out}
    beside = (1 if case.get("times") else 0) + (1 if case.get("residual") else 0)
    moved = t * inp + used * out * inp + t * out * (1 + beside) + (out if case.get("bias") else 0)
    if not case["grad"]:
        return {"bytes": 2 * moved, "flops": 2 * t * inp * out}
    # backwards dy, x, the weights and what stood in the epilogue again, all their gradients written
    again = t * out + t * inp + used * out * inp + (t * out if case.get("times") else 0) + t * inp + n * out * inp + t * out * (1 if case.get("times") else 0)
    return {"bytes": 2 * (moved + again), "flops": 6 * t * inp * out}


def exact(case, seed):
    """The definitions in 64 bits, gradients by their own formulas, expert by expert."""
    s = prepare(case, seed)
    with torch.no_grad():
        return {"norm": _exact_norm, "norm8": _exact_norm}.get(case["op"], _exact_products)(s)


def _exact_norm(s):
    x, w = s["x"].double(), s["weight"].double()
    y = {}
    if s["residual"] is not None:
        y["stream"] = x.add(s["residual"].double())
        x = y["stream"].to(s["x"].dtype).double()
    square = torch.einsum("td,td->t", x, x).div(x.shape[1]).add(EPS)
    normed = torch.einsum("td,t->td", x, square.pow(-0.5))
    v = normed.mul(w)
    if s["op"] == "norm8":
        most = v.abs().max(dim=1).values
        return y | {"q": v.mul(E4M3_MOST).div(most[:, None]), "scale": most.div(E4M3_MOST)}
    y["y"] = v
    if s["grad"]:
        dy = s["dy"].double()
        along = torch.einsum("td,td,d->t", dy, normed, w).div(x.shape[1])
        dx = torch.addcmul(dy.mul(w), normed, along[:, None], value=-1).mul(square.pow(-0.5)[:, None])
        if "stream" in y:
            dx += s["ds"].double()
            y["dresidual"] = dx
        y |= {"dx": dx, "dweight": torch.einsum("td,td->d", dy, normed)}
    return y


def _exact_act(kind, z):
    if kind == "none":
        return z, torch.ones_like(z)
    if kind == "relu":
        return z.clamp_min(0), (z > 0).double()
    if kind == "silu":
        e = torch.sigmoid(z)
        return z * e, e + z * e * torch.sigmoid(-z)
    if kind == "gelu":
        below = 0.5 * torch.special.erfc(-z / math.sqrt(2))
        return z * below, below + z * torch.exp(-z.square() / 2) * (2 * math.pi) ** -0.5
    u = math.sqrt(2 / math.pi) * (z + 0.044715 * z ** 3)
    below = torch.sigmoid(2 * u)          # (1 + tanh u) / 2
    return z * below, below + 2 * z * below * torch.sigmoid(-2 * u) * math.sqrt(2 / math.pi) * (1 + 0.134145 * z ** 2)


def _exact_products(s):
    rows, out = s["x"].shape[0], s["weight"].shape[-2]
    weights = s["weight"] if s["weight"].dim() == 3 else s["weight"][None]
    ends = s["offsets"].tolist() if "offsets" in s else [0, rows]
    y = {"y": torch.zeros((rows, out), dtype=torch.float64, device="cuda")}
    if s["grad"]:
        y |= {"d" + k: torch.zeros(s[k].shape, dtype=torch.float64, device="cuda") for k in s["trained"]}
    for e, (lo, hi) in enumerate(zip(ends, ends[1:])):
        if lo == hi:
            continue
        x, w = s["x"][lo:hi].double(), weights[e].double()
        if "x_scale" in s:
            x, w = x * s["x_scale"][lo:hi].double()[:, None], w * s["weight_scale"].double()[:, None]
        z = torch.mm(x, w.t())
        if s.get("bias") is not None:
            z += s["bias"].double()
        a, da = _exact_act(s["activation"], z)
        v = a
        if s["times"] is not None:
            v = v * s["times"][lo:hi].double()
        if s.get("residual") is not None:
            v = v + s["residual"][lo:hi].double()
        y["y"][lo:hi] = v
        if not s["grad"]:
            continue
        dy = s["dy"][lo:hi].double()
        dz = dy * da
        if s["times"] is not None:
            y["dtimes"][lo:hi] = dy * a
            dz = dz * s["times"][lo:hi].double()
        if s.get("residual") is not None:
            y["dresidual"][lo:hi] = dy
        if s.get("bias") is not None:
            y["dbias"] += dz.sum(0)
        y["dx"][lo:hi] = torch.mm(dz, w)
        (y["dweight"][e] if weights is s["weight"] else y["dweight"]).add_(torch.mm(dz.t(), x))
    return y
