"""Norms, products and experts' products where numbers are small, large or next to a border: the far sides of activations, scales and gradients at the ends of
their ranges, sums that round one way in 32 bits and another in fewer, against the definitions in 64 bits."""
import pytest
import torch

from layers import STEP, act, close, half_step, least

pytestmark = pytest.mark.gpu

BF16, F16 = torch.bfloat16, torch.float16


@pytest.fixture(autouse=True)
def _library(gpu):
    yield gpu
    from lmz_b200 import adapters
    adapters.check()


def _numbers(dtype, lo, hi):
    """Every number of a 16-bit type whose magnitude is in [lo, hi], of both signs."""
    every = torch.arange(-2 ** 15, 2 ** 15, device="cuda").to(torch.int16).view(dtype)
    return every[(every.abs() >= lo) & (every.abs() <= hi)]


def _exponent(kind, z):
    """How large the exponential's argument gets that an activation's far side goes by."""
    return {"silu": z.abs(), "gelu": z * z, "gelu_tanh": 1.6 * (z + 0.044715 * z ** 3).abs()}[kind]


@pytest.mark.parametrize("dtype", [BF16, F16])
@pytest.mark.parametrize("kind", ["silu", "gelu", "gelu_tanh"])
def test_far_sides_of_activations(kind, dtype):
    """Relative to the result itself, wherever it can be held: one rounding to the type, and in 32 bits the exponential's error, which grows with its argument
    (an argument of A is off by A 2^-24 a rounding, of which there are up to four, and the function by (2 + 1.2 A) 2^-23), and eight roundings more.  (128 times the
    smallest number of 32 bits beside that, where the exponential itself is among those.)"""
    from lmz_b200 import linear
    z = _numbers(dtype, 2.0 ** -20, 100.0)
    x, w = z[:, None].clone().requires_grad_(True), torch.ones((1, 1), dtype=dtype, device="cuda")
    m = torch.ones_like(x).requires_grad_(True)
    y = linear.project(x, w, activation=kind, times=m)
    dx, dm = torch.autograd.grad(y, (x, m), torch.ones_like(y))
    with torch.no_grad():
        v = z[:, None].double()
        a, slope = act(kind, v)
        off = (10 + 4 * _exponent(kind, v)) * STEP
        u, tiny = half_step(dtype), least(dtype) + 2.0 ** -142
        below = torch.where(v == 0, 0.5, a / v)              # what z is multiplied by
        size = below + (slope - below).abs()                 # the slope's two terms
        for got, want, o in ((y, a, off * a.abs()), (dm, a, off * a.abs()), (dx, slope, off * size)):
            close(got, (want, o + u * (want.abs() + o) + tiny))
