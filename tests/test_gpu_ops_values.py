"""Operators with adapters on values at the ends of their types' ranges."""
import math

import pytest
import torch

from test_gpu_ops import DTYPES, _check, _index, _randn, _rows_of

pytestmark = pytest.mark.gpu


@pytest.fixture(autouse=True)
def _library(gpu):
    return gpu


def _whole(seed, shape, dtype, most=1):
    g = torch.Generator(device="cuda").manual_seed(seed)
    return torch.randint(-most, most + 1, shape, generator=g, device="cuda").to(dtype)


def _same_class(got, want, what):
    """Whole numbers small enough to be exact, or the same infinity, or NaN both."""
    got = got.double()
    same = (got == want) | (torch.isnan(got) & torch.isnan(want))
    assert same.all(), f"{what}: {int((~same).sum())} of {same.numel()}, the first {got[~same][0].item()} for {want[~same][0].item()}"


# tokens, in, out, rank, adapters, index: one adapter's runs, sixteens of several, a pair's tiles, a cluster's, tokens by adapter
LAYOUTS = [(1, 64, 64, 8, 1, "none"), (40, 128, 96, 16, 3, "mixed"), (64, 128, 264, 16, 2, "none"), (300, 64, 520, 24, 4, "runs"), (700, 128, 1288, 8, 3, "mixed"),
           (600, 64, 2056, 72, 2, "runs"), (2500, 64, 4104, 72, 5, "mixed"), (333, 77, 131, 5, 4, "runs"), (256, 64, 128, 136, 2, "short")]


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("tokens, inp, out, rank, n, kind", LAYOUTS)
@pytest.mark.parametrize("where", ["b", "a", "x", "dy"])
def test_infinities_are_the_definitions(dtype, tokens, inp, out, rank, n, kind, where):
    """An infinity times a thin product is an infinity of its sign, and NaN where that is zero, however tokens lie: whole numbers,
    so that the products are exact, many of them zero, and the 16-bit type holds them."""
    from lmz_b200 import adapters
    x, w, a, b, dy = (_whole(i, s, dtype) for i, s in enumerate(((tokens, inp), (out, inp), (n, rank, inp), (n, out, rank), (tokens, out))))
    x[:, inp // 2:] = 0                                    # (thin products stay small)
    dy[:, 16:] = 0
    g = torch.Generator(device="cuda").manual_seed(9)
    for t in ([b], [a], [x], [dy])[("b", "a", "x", "dy").index(where)]:
        flat = t.view(-1)
        at = torch.randint(0, flat.numel(), (1 + flat.numel() // 200,), generator=g, device="cuda")
        flat[at] = torch.where(_whole(8, at.shape, torch.float32) >= 0, math.inf, -math.inf).to(dtype)
    index = _index(kind, tokens, n)
    leaves = [t.requires_grad_(True) for t in (x, a, b)]
    y = adapters.project(x, w, a, b, index, scale=2.0)
    got = (y.detach(), *torch.autograd.grad(y, leaves, dy))
    # The definition, term by term.
    xd, wd, ad, bd, dyd = (t.detach().double() for t in (x, w, a, b, dy))
    want_y, want_x = _product(xd, wd.t()), _product(dyd, wd)
    want_a, want_b = torch.zeros_like(ad), torch.zeros_like(bd)
    own = torch.zeros(tokens, dtype=torch.int64, device="cuda") if index is None else index
    for i in range(n):
        at = torch.nonzero(own == i).flatten()
        if not at.numel():
            continue
        h, gr = 2 * _product(xd[at], ad[i].t()), 2 * _product(dyd[at], bd[i])
        want_y[at] += _product(h, bd[i].t())
        want_x[at] += _product(gr, ad[i])
        want_a[i], want_b[i] = _product(gr.t(), xd[at]), _product(dyd[at].t(), h)
    for g_, w_, what in zip(got, (want_y, want_x, want_a, want_b), ("y", "dx", "da", "db")):
        big = w_.abs() > 2 ** (8 if dtype == torch.bfloat16 else 11)      # (whole numbers that T does not hold)
        assert (big & w_.isfinite()).double().mean() < 0.5
        _same_class(torch.where(big & w_.isfinite(), torch.zeros_like(g_), g_), torch.where(big & w_.isfinite(), 0.0, w_), what)


def _product(p, q):
    """p @ q with every term's infinity and NaN as the definition has it (a library's product may skip zeros)."""
    clean = torch.where(p.isfinite(), p, 0.0) @ torch.where(q.isfinite(), q, 0.0)
    pn, qn = p.isnan(), q.isnan()
    f = lambda c: c.double()                               # noqa: E731
    nan = f(pn) @ torch.ones_like(q) + torch.ones_like(p) @ f(qn) + f(p.isinf()) @ f(q == 0) + f(p == 0) @ f(q.isinf())
    up = f(p == math.inf) @ f(q > 0) + f(p == -math.inf) @ f(q < 0) + f(p > 0) @ f(q == math.inf) + f(p < 0) @ f(q == -math.inf)
    down = f(p == math.inf) @ f(q < 0) + f(p == -math.inf) @ f(q > 0) + f(p > 0) @ f(q == -math.inf) + f(p < 0) @ f(q == math.inf)
    out = torch.where(up > 0, math.inf, torch.where(down > 0, -math.inf, clean))
    return torch.where((nan > 0) | ((up > 0) & (down > 0)), math.nan, out)


# F16 whose thin products leave its range, while the results do not: standard deviations of x, W, A, B and dy.
RANGES = {"large h, tiny g": (3000.0, 1e-3, 4.0, 1e-4, 1e-3), "large g, tiny h": (1e-3, 1e-3, 1e-4, 4.0, 3000.0), "tiny dy": (30.0, 0.05, 0.1, 1.0, 1e-6),
          "tiny x": (1e-6, 0.05, 0.1, 1.0, 30.0), "b of zeros": (3000.0, 1e-3, 4.0, 0.0, 1e-3)}


@pytest.mark.parametrize("tokens, inp, out, rank, n, kind", LAYOUTS)
@pytest.mark.parametrize("stds", RANGES.values(), ids=RANGES)
def test_f16_over_its_range(tokens, inp, out, rank, n, kind, stds):
    """The bounds of test_gpu_ops, less their allowance for thin products kept in F16: 2^-16 of their magnitude, wherever that is."""
    from lmz_b200 import adapters
    dtype = torch.float16
    x, w, a, b, dy = (_randn(70 + i, s, dtype, std) for i, (s, std) in enumerate(zip(((tokens, inp), (out, inp), (n, rank, inp), (n, out, rank), (tokens, out)), stds)))
    scales = 0.5 + torch.arange(n, device="cuda").float() / 2
    index = _index(kind, tokens, n)
    leaves = [t.requires_grad_(True) for t in (x, a, b)]
    y = adapters.project(x, w, a, b, index, scale=scales)
    got = (y.detach(), *torch.autograd.grad(y, leaves, dy))
    xd, wd, ad, bd, dyd = (t.detach().double() for t in (x, w, a, b, dy))
    want = [xd @ wd.t(), dyd @ wd, torch.zeros_like(ad), torch.zeros_like(bd)]
    size = [xd.abs() @ wd.abs().t(), dyd.abs() @ wd.abs(), torch.zeros_like(ad), torch.zeros_like(bd)]
    carried = [torch.zeros_like(t) for t in want]
    largest = 0.0
    for i in range(n):
        at, s = _rows_of(index, tokens, i), float(scales[i])
        if not at.numel():
            continue
        h, hs = s * (xd[at] @ ad[i].t()), s * (xd[at].abs() @ ad[i].abs().t())
        g, gs = s * (dyd[at] @ bd[i]), s * (dyd[at].abs() @ bd[i].abs())
        largest = max(largest, float(h.abs().max()), float(g.abs().max()))
        for k, (rows, p, ps, q) in enumerate(((at, h, hs, bd[i].t()), (at, g, gs, ad[i]), (i, g.t(), gs.t(), xd[at]), (i, dyd[at].t(), dyd[at].abs().t(), h))):
            want[k][rows] += p @ q
            size[k][rows] += ps @ (hs if k == 3 else q.abs())
            carried[k][rows] += 2 ** -16 * (p.abs() @ q.abs())
    assert largest > 65504 or "tiny" in [k for k, v in RANGES.items() if v == stds][0] or tokens == 1
    for v, w_, s_, c, terms, what in zip(got, want, size, carried, (inp + rank + 8, out + rank + 8, tokens + out + 8, tokens + inp + 8), ("y", "dx", "da", "db")):
        # (F16 ends at 65504, and what is nearer to 65536 is infinite: from 65520 on, give or take what the sums may be off by)
        slack = (1 + 2 ** -11) * (terms * 2 ** -23 * s_ + c)
        inside, beyond = w_.abs() + slack < 65520, w_.abs() - slack >= 65520
        assert (v[beyond].double() == w_[beyond].sign() * math.inf).all(), what
        assert inside.double().mean() > 0.9
        _check(torch.where(inside, v, torch.zeros_like(v)), torch.where(inside, w_, 0.0), s_, c, terms, what)
