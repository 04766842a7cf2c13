"""Operators with adapters on values at the ends of their types' ranges."""
import math

import pytest
import torch

from test_gpu_ops import DTYPES, _index

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
