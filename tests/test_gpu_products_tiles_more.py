"""Products in tiles that long sums of few rows take (clusters of two to eight at 32 to 128 columns), for each of the three products, with one weight and with several and in 8
bits; and how far all of a result is off, not only each element: an element's tolerance goes by the worst that its sum can do, beside which a part that is missing could pass.

In the 2-norm: half a step of the type, and four standard deviations of a random walk of as many steps as a sum has, none above 2^-23 of the magnitudes' sum."""
import pytest
import torch

from layers import STEP, close, half_step, products as want_products

pytestmark = pytest.mark.gpu

# rows, in, out, experts
SHAPES = [(4066, 562, 517, 1), (68, 13873, 538, 1), (622, 388, 4273, 1), (390, 260, 9424, 1), (298, 19, 3950, 1), (294, 129, 6145, 1), (72, 275, 12949, 1), (738, 4044, 424, 1), (401, 9257, 279, 1),
          (151, 4304, 140, 1), (290, 6368, 144, 1), (5480, 293, 776, 2), (7951, 390, 295, 2), (4929, 10, 10, 2), (495, 3613, 26, 5), (787, 643, 2829, 2), (858, 267, 4417, 2), (382, 265, 9206, 2),
          (171, 12, 3884, 9), (288, 146, 5418, 2), (1796, 538, 13, 16), (476, 27, 3587, 5), (796, 3029, 732, 2), (747, 3972, 389, 2), (520, 9714, 137, 3), (165, 3845, 10, 9), (537, 5425, 11, 5),
          (6618, 10, 130, 64), (1, 14336, 4096, 1), (200, 4096, 4096, 1), (2304, 4096, 1024, 1)]
SHAPES_8 = [(71, 518, 12966), (878, 5303, 642), (625, 8212, 386), (1, 8, 8), (146, 7792, 132), (623, 3869, 399), (306, 11031, 133), (16, 14336, 4096), (2304, 4096, 1024)]


@pytest.fixture(autouse=True)
def _library(gpu):
    yield gpu
    from lmz_b200 import adapters
    adapters.check()


def _randn(seed, shape, dtype=torch.bfloat16, std=1.0):
    g = torch.Generator(device="cuda")
    g.manual_seed(seed)
    return (torch.randn(shape, generator=g, device="cuda") * std).to(dtype)


def _check(name, got, want, size, terms):
    """`size`: the magnitudes' sums, of `terms` each."""
    try:
        close(got, want)
    except AssertionError as e:
        raise AssertionError(f"{name}: {e}") from None
    exact = want[0]
    off, most = float((got.double() - exact).norm()), half_step(got.dtype) * float(exact.norm()) + 4 * terms ** 0.5 * STEP * float(size.norm())
    assert off <= most, (name, off, most)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("rows, inp, out, experts", SHAPES)
def test_tiles(rows, inp, out, experts, dtype):
    from lmz_b200 import experts as ex, linear
    x, b, dy = _randn(1, (rows, inp), dtype), _randn(3, (experts, out), dtype), _randn(6, (rows, out), dtype)
    w = _randn(2, (experts, out, inp), dtype, inp ** -0.5)
    each = rows // experts
    starts = [min(rows, e * each + min(each, 3) * (e % 2)) for e in range(experts)] + [rows]
    x.requires_grad_(True), w.requires_grad_(True)
    y = linear.project(x, w[0], b[0]) if experts == 1 else ex.project(x, w, torch.tensor(starts, device="cuda"), bias=b)
    dx, dw = torch.autograd.grad(y, (x, w), dy)
    with torch.no_grad():
        want = want_products(x, w, b, dy=dy, starts=starts)
        size = {"y": torch.zeros_like(want["y"][0]), "dx": torch.zeros_like(want["dx"][0]), "dweight": torch.zeros_like(want["dweight"][0])}
        for e, (lo, hi) in enumerate(zip(starts, starts[1:])):
            xs, we, ds = x[lo:hi].abs().double(), w[e].abs().double(), dy[lo:hi].abs().double()
            size["y"][lo:hi], size["dx"][lo:hi], size["dweight"][e] = xs @ we.t() + b[e].abs(), ds @ we, ds.t() @ xs
        for name, got, terms in (("y", y, inp + 1), ("dx", dx, out), ("dweight", dw, max(hi - lo for lo, hi in zip(starts, starts[1:])))):
            _check(name, got, want[name], size[name], terms)
        if experts == 1:
            r = _randn(5, (rows, out), dtype)
            close(linear.project(x, w[0], b[0], "silu", residual=r), want_products(x, w[0], b[0], "silu", residual=r)["y"])


@pytest.mark.parametrize("rows, inp, out", SHAPES_8)
def test_tiles_in_8_bits(rows, inp, out):
    from lmz_b200 import linear, norms
    q, s = norms.to_8bit(_randn(1, (rows, inp), torch.float32, 3.0))
    wq, ws = norms.to_8bit(_randn(2, (out, inp), torch.float32, 0.02))
    b, r = _randn(3, out), _randn(5, (rows, out))
    size = (q.float().abs().double() @ wq.float().abs().double().t()) * s.double()[:, None] * ws.double()
    _check("y", linear.project_8bit(q, s, wq, ws), want_products(q.float(), wq.float(), x_scale=s, weight_scale=ws, dtype=torch.bfloat16)["y"], size, inp)
    close(linear.project_8bit(q, s, wq, ws, bias=b, activation="silu", residual=r),
          want_products(q.float(), wq.float(), b, "silu", residual=r, x_scale=s, weight_scale=ws, dtype=torch.bfloat16)["y"])
