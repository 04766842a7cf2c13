"""The operators of a layer by their definitions in 64 bits, and how far 32-bit sums and the roundings they make may be from those.

A sum of n terms in 32 bits is off by at most n * 2^-23 times the sum of the terms' magnitudes (tensor cores cut where an addition would
round); a rounding to a type by half a step of it.  Errors are carried through what follows by the magnitudes of its factors.
"""
import math

import torch

STEP = 2.0 ** -23
SLOPE, BEND = 1.13, 1.0                  # no activation is steeper, or bends more, than that


def half_step(dtype):
    return torch.finfo(dtype).eps / 2


def least(dtype):
    """Half the step between the smallest numbers."""
    return torch.finfo(dtype).smallest_normal * torch.finfo(dtype).eps / 2


def act(kind, z):
    if kind is None:
        return z, torch.ones_like(z)
    if kind == "relu":
        return z.clamp_min(0), (z > 0).to(z.dtype)
    if kind == "silu":
        e = torch.sigmoid(z)
        return z * e, e * (1 + z * torch.sigmoid(-z))
    if kind == "gelu":
        below = 0.5 * torch.special.erfc(-z * math.sqrt(0.5))
        return z * below, below + z * torch.exp(-0.5 * z * z) / math.sqrt(2 * math.pi)
    u = math.sqrt(2 / math.pi) * (z + 0.044715 * z ** 3)
    below = torch.sigmoid(2 * u)
    return z * below, below + 2 * z * below * torch.sigmoid(-2 * u) * math.sqrt(2 / math.pi) * (1 + 3 * 0.044715 * z ** 2)


def products(x, weight, bias=None, kind=None, times=None, residual=None, dy=None, starts=None, x_scale=None, weight_scale=None, dtype=None):
    """{name: (exact, tolerance)} of y and, with dy, of the gradients.  `starts`: where the experts' rows begin (host numbers), for a
    weight [experts, out, in]."""
    dtype = dtype or x.dtype
    u, tiny = half_step(dtype), least(dtype)
    weights = weight if weight.dim() == 3 else weight[None]
    starts = [0, x.shape[0]] if starts is None else starts
    rows, (experts, out, inp) = x.shape[0], weights.shape
    new = lambda *s: torch.zeros(s, dtype=torch.float64, device=x.device)          # noqa: E731
    got = {"y": [new(rows, out), new(rows, out)]}
    if dy is not None:
        got |= {"dx": [new(rows, inp), new(rows, inp)], "dweight": [new(*weights.shape), new(*weights.shape)], "dbias": [new(experts, out), new(experts, out)],
                "dtimes": [new(rows, out), new(rows, out)]}
    for e in range(experts):
        lo, hi = starts[e], starts[e + 1]
        if hi <= lo:
            continue
        xs, w = x[lo:hi].double(), weights[e].double()
        z, size = xs @ w.t(), xs.abs() @ w.abs().t()
        if x_scale is not None:
            scale = x_scale[lo:hi].double()[:, None] * weight_scale.double()
            z, size = z * scale, size * scale
        if bias is not None:
            b = (bias[e] if bias.dim() == 2 else bias).double()
            z, size = z + b, size + b.abs()
        off = (inp + 6) * STEP * size                       # of z
        a, slope = act(kind, z)
        a_off = SLOPE * off + 8 * STEP * (z.abs() + 1) * (kind is not None)
        m = torch.ones_like(z) if times is None else times[lo:hi].double()
        y, y_off = a * m, a_off * m.abs() + 2 * STEP * (a * m).abs()
        if residual is not None:
            r = residual[lo:hi].double()
            y, y_off = y + r, y_off + 2 * STEP * (y.abs() + r.abs())
        got["y"][0][lo:hi], got["y"][1][lo:hi] = y, y_off + u * (y.abs() + y_off) + tiny
        if dy is None:
            continue
        d = dy[lo:hi].double()
        kept = off + (2 ** -15 * z.abs() if kind is not None or times is not None else 0)           # z as the gradients have it: 16 bits of mantissa, cut
        s_off = BEND * kept + 8 * STEP * (z.abs() + 1) * (kind is not None)
        if kind == "relu":
            s_off = s_off + (z.abs() <= kept)              # (either side of the corner)
        if kind is None:
            s_off = 0 * off
        dz, dz_off = d * slope * m, (d * m).abs() * s_off + 3 * STEP * (d * slope * m).abs()
        db, db_off = dz.sum(0), dz_off.sum(0) + (hi - lo + 2) * STEP * (dz.abs() + dz_off).sum(0)
        if kind is not None or times is not None:          # (else dz is dy itself)
            dz_off = dz_off + u * (dz.abs() + dz_off) + tiny
        most = dz.abs() + dz_off
        dx, dx_off = dz @ w, dz_off @ w.abs() + (out + 2) * STEP * (most @ w.abs())
        dw, dw_off = dz.t() @ xs, dz_off.t() @ xs.abs() + (hi - lo + 2) * STEP * (most.t() @ xs.abs())
        dm, dm_off = d * a, d.abs() * (SLOPE * kept + 8 * STEP * (z.abs() + 1)) + 2 * STEP * (d * a).abs()
        for name, place, v, v_off in (("dx", slice(lo, hi), dx, dx_off), ("dweight", e, dw, dw_off), ("dbias", e, db, db_off), ("dtimes", slice(lo, hi), dm, dm_off)):
            got[name][0][place], got[name][1][place] = v, v_off + u * (v.abs() + v_off) + tiny
    if weight.dim() == 2 and dy is not None:
        for name in ("dweight", "dbias"):
            got[name] = [t[0] for t in got[name]]
    return got


def norm_steps(dim):
    """Additions that a square goes through on its way into a row's sum, and what else touches the result."""
    return 16 * math.ceil(dim / 16384) + 48


def norms(x, weight, residual=None, eps=1e-6, dy=None, ds=None):
    """{name: (exact, tolerance)} of y, what was normed, and with dy of dx and dweight."""
    dtype = x.dtype
    u, tiny = half_step(dtype), least(dtype)
    s = (x if residual is None else (x.float() + residual.float()).to(dtype)).double()
    w, dim = weight.double(), x.shape[-1]
    rstd = (s.square().mean(-1, keepdim=True) + eps).rsqrt()
    n, few = s * rstd, norm_steps(dim) * STEP
    y = n * w
    got = {"s": (s, 0 * s), "y": (y, (u + few) * y.abs() + tiny), "wide": (y, few * y.abs())}
    if dy is None:
        return got
    g = dy.double()
    d, size = g * w, (g * w * n).abs().mean(-1, keepdim=True)
    dx = rstd * (d - n * (d * n).mean(-1, keepdim=True))
    off = few * 3 * rstd * (d.abs() + n.abs() * size)
    if ds is not None:
        dx, off = dx + ds.double(), off + 2 * STEP * ds.double().abs()
    got["dx"] = dx, off + u * (dx.abs() + off) + tiny
    dw, dw_size = (g * n).sum(0), (g * n).abs().sum(0)
    dw_off = (x.shape[0] * STEP + few) * dw_size
    got["dweight"] = dw, dw_off + half_step(weight.dtype) * (dw.abs() + dw_off) + least(weight.dtype)
    return got


def close(got, want):
    exact, off = want
    assert got.shape == exact.shape, (got.shape, exact.shape)
    bad = ~((got.double() - exact).abs() <= off)
    if bad.any():
        i = tuple(int(v) for v in torch.nonzero(bad)[0])
        raise AssertionError(f"{int(bad.sum())} of {bad.numel()} are off, the first at {i}: {float(got[i])} for {float(exact[i])} within {float(off[i])}")
