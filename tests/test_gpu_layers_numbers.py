"""Norms, products and experts' products where numbers are small, large or next to a border: the far sides of activations, scales and gradients at the ends of
their ranges, sums that round one way in 32 bits and another in fewer, against the definitions in 64 bits."""
import pytest
import torch

from layers import STEP, act, close, half_step, least, products as want_products

pytestmark = pytest.mark.gpu

BF16, F16, F32 = torch.bfloat16, torch.float16, torch.float32


@pytest.fixture(autouse=True)
def _library(gpu):
    yield gpu
    from lmz_b200 import adapters
    adapters.check()


def _randn(seed, shape, dtype=BF16, std=1.0):
    g = torch.Generator(device="cuda")
    g.manual_seed(seed)
    return (torch.randn(shape, generator=g, device="cuda") * std).to(dtype)


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


@pytest.mark.parametrize("rows, inp, out, residual", [(3, 256, 64, False), (3, 256, 64, True), (2, 256, 33, False), (1, 8192, 64, False), (1, 8192, 64, True), (1, 8192, 33, True), (300, 256, 512, False),
                                                      (300, 256, 512, True)])
@pytest.mark.parametrize("x_power, w_power", [(-90, -62), (-126, 126), (126, -126), (100, 40), (-50, -95), (-140, 10), (0, 0)])
def test_scales_of_8_bits_at_the_ends_of_their_range(rows, inp, out, residual, x_power, w_power):
    """Neither two small nor two large scales, nor one of each, lose what the result can hold; a sum of zero stays zero."""
    from lmz_b200 import linear
    both = x_power + w_power
    small = -both > 100                                      # (the sums are as large as they get, or as small)
    x, w = (_randn(k, s, F32, 120.0 if both < 0 else 0.01).clamp(-448, 448).abs().to(torch.float8_e4m3fn) for k, s in ((1, (rows, inp)), (2, (out, inp))))
    x[-1], w[out // 2] = 0, 0
    xs, ws = ((1 + 0.9 * torch.rand(n, generator=torch.Generator("cuda").manual_seed(n), device="cuda")) * 2.0 ** p for n, p in ((rows, x_power), (out, w_power)))
    r = torch.zeros((rows, out), dtype=BF16, device="cuda") if residual else None
    y = linear.project_8bit(x, xs, w, ws, residual=r)
    exact, off = want_products(x.float(), w.float(), x_scale=xs, weight_scale=ws, dtype=BF16)["y"]
    # (32 bits' own smallest numbers, of which a product may pass through one; what is above 16 bits' largest number is infinite)
    fits = exact.abs() < 2.0 ** 127
    close(torch.where(fits, y, 0), (torch.where(fits, exact, 0), off.clamp_max(2.0 ** 127) + 2.0 ** -148))
    assert not y.isnan().any() and (y[-1] == 0).all() and (y[:, out // 2] == 0).all()
    assert rows == 1 or small or (y[0] != 0).any()


@pytest.mark.parametrize("dtype, far, near", [(F16, 2.0 ** -11, 2.0 ** -20), (BF16, 2.0 ** -8, 2.0 ** -20)])
@pytest.mark.parametrize("rows, out", [(1, 1), (3, 8), (300, 264), (2304, 512)])
def test_a_factors_gradient_is_rounded_once(dtype, far, near, rows, out):
    """z a little above the middle between two numbers: its last bits decide."""
    from lmz_b200 import linear
    x = torch.zeros((rows, 16), dtype=dtype, device="cuda")
    w = torch.zeros((out, 16), dtype=dtype, device="cuda")
    x[:, 0], x[:, 1], x[:, 2] = 1.0, far, 2.0 ** -10
    w[:, 0], w[:, 1], w[:, 2] = 1.0, 1.0, near * 2.0 ** 10
    m = torch.ones((rows, out), dtype=dtype, device="cuda").requires_grad_(True)
    (dm,) = torch.autograd.grad(linear.project(x, w, times=m), m, torch.ones_like(m))
    assert (dm == 1 + 2 * far).all()


@pytest.mark.parametrize("rows, inp, out", [(40, 64, 96), (40, 33, 50), (700, 64, 264), (2304, 512, 2304)])
@pytest.mark.parametrize("kind", [None, "silu"])
@pytest.mark.parametrize("large", [True, False])
def test_gradients_of_sums_outside_half_precisions_range(rows, inp, out, kind, large):
    """dz above F16's largest number, or below its smallest, where what it is made of and what is made of it are inside: an element of dz is as good as F16 holds one of
    ordinary size, or off by 2^-38 of its group's largest."""
    from lmz_b200 import experts, linear
    # dz is dy times the factor, 2^22 or 2^-26 and around; dx and dW some 2^10, or 2^-10 and more
    far, w_std, x_std = (2.0 ** 11, 2.0 ** -12 / out ** 0.5, 2.0 ** -12 / rows ** 0.5) if large else (2.0 ** -13, 2.0 ** 13, 2.0 ** 13)
    x, w = _randn(1, (rows, inp), F16, x_std), _randn(2, (3, out, inp), F16, w_std)
    m, dy = _randn(3, (rows, out), F16, far), _randn(4, (rows, out), F16, far)
    x[1], w[:, 1] = 0, 0
    starts = [0, rows // 2, rows - 20, rows - 3]
    m[starts[2]:] /= far                                     # (an expert with a factor of ordinary size)
    for dense in (True, False):
        v, u = x.clone().requires_grad_(True), (w[0] if dense else w).clone().requires_grad_(True)
        y = linear.project(v, u, activation=kind, times=m) if dense else experts.project(v, u, torch.tensor(starts, device="cuda"), activation=kind, times=m)
        dx, dw = torch.autograd.grad(y, (v, u), dy)
        ends, weights = ([0, rows], w[:1]) if dense else (starts, w)
        for e, (lo, hi) in enumerate(zip(ends, ends[1:])):
            if lo == hi:
                assert (dw[e] == 0).all()
                continue
            xs, we = x[lo:hi].double(), weights[e].double()
            z = xs @ we.t()
            z_off = (inp + 6) * STEP * (xs.abs() @ we.abs().t())
            _, slope = act(kind, z)
            d = dy[lo:hi].double() * m[lo:hi].double()
            dz = d * slope
            # (no slope bends more than one; beyond 40 SiLU's is zero or one)
            bent = 0 if kind is None else torch.where(z.abs() < z_off + 40, z_off.clamp_max(1.1), 0) + 20 * STEP
            off = d.abs() * bent + half_step(F16) * 1.01 * dz.abs() + 2.0 ** -38 * dz.abs().max()
            most = dz.abs() + off
            for got, a, b, n in ((dx[lo:hi], (dz, off, most), we, out), ((dw if dense else dw[e]), (dz.t(), off.t(), most.t()), xs, hi - lo)):
                want = a[0] @ b
                o = a[1] @ b.abs() + (n + 4) * STEP * (a[2] @ b.abs())
                close(got, (want, o + half_step(F16) * (want.abs() + o) + least(F16)))
        assert dx.isfinite().all() and dw.isfinite().all()


@pytest.mark.parametrize("dtype, size, slope", [(BF16, 1e-17, 1e7), (BF16, 1e17, 1e-9), (BF16, 1e17, 1e25), (F32, 1e-17, 1e7), (F32, 1e17, 1e-9), (F32, 1e17, 1e25), (BF16, 1.0, 1.0)])
@pytest.mark.parametrize("rows, dim", [(3, 64), (5, 77), (2, 4096), (2, 17000)])
def test_norms_of_small_and_large_rows(dtype, size, slope, rows, dim):
    """Rows whose squares 32 bits hold, and gradients that they hold: neither becomes infinite nor loses bits on the way."""
    from layers import norms as want_norms

    from lmz_b200 import norms
    x, w, dy = _randn(1, (rows, dim), dtype, size), _randn(2, dim, dtype), _randn(3, (rows, dim), dtype, slope)
    x.requires_grad_(True), w.requires_grad_(True)
    y = norms.rms_norm(x, w, eps=0.0)
    dx, dw = torch.autograd.grad(y, (x, w), dy)
    with torch.no_grad():
        want = want_norms(x, w, None, 0.0, dy)
        close(y, want["y"]), close(dx, want["dx"]), close(dw, want["dweight"])


@pytest.mark.parametrize("low, high", [(-4, 4), (-61, -59), (59, 61), (-100, -99), (-120, 110)])
def test_quotients_next_to_the_middle_between_two_numbers_of_8_bits(low, high):
    """What is divided by its row's scale lies on the middle between two numbers of 8 bits, or up to three steps of 32 bits beside it."""
    from lmz_b200 import norms
    g = torch.Generator("cuda")
    g.manual_seed(1)
    every = torch.arange(0x7F, device="cuda").to(torch.uint8).view(torch.float8_e4m3fn).double()
    middles = (every[1:] + every[:-1]) / 2
    rows, near = 4000, torch.arange(-3, 4, device="cuda")
    most = (448 * 2.0 ** (torch.rand(rows, 1, generator=g, device="cuda") * (high - low) + low)).float()
    # (scales of 1 - 2^-24 and around, and of other round numbers)
    turn = torch.arange(rows // 2, device="cuda").to(torch.int32)
    power = 2.0 ** (low + turn % max(high - low, 1)).float()
    most[:rows // 2, 0] = ((torch.tensor(448.0, device="cuda") * (8 + turn // 11 % 9) / 8).view(torch.int32) + turn % 11 - 5).view(F32) * power
    scale = most / torch.full_like(most, 448)              # (by a number of the host torch would multiply by its reciprocal)
    u = (middles[None] * scale.double()).float()[:, :, None].repeat(1, 1, 7).view(torch.int32)
    u = torch.where(u > 8, u + near.to(torch.int32), u).view(F32).flatten(1)
    x = torch.cat((most, u.clamp_max(most), -u.clamp_max(most)), 1)
    q, s = norms.to_8bit(x)
    assert torch.equal(s, scale[:, 0])
    assert torch.equal(q.view(torch.uint8), (x / scale).to(torch.float8_e4m3fn).view(torch.uint8))


def test_captured_gradients_in_half_precision_follow_their_sizes():
    """A graph finds the power that dz is written by anew at each replay: ordinary, far above F16's range, far below, and back."""
    from lmz_b200 import experts, linear
    rows, inp, out = 90, 72, 104
    x, w, ws = _randn(1, (rows, inp), F16, 2.0 ** -12), _randn(2, (out, inp), F16, 2.0 ** -12), _randn(3, (3, out, inp), F16, 2.0 ** -12)
    m, dy = _randn(4, (rows, out), F16), _randn(5, (rows, out), F16)
    offsets = torch.tensor([2, 40, 40, 87], device="cuda")
    leaves = [t.requires_grad_(True) for t in (x, w, ws)]

    def step():
        y, e = linear.project(x, w, activation="gelu", times=m), experts.project(x, ws, offsets, activation="silu", times=m)
        return *torch.autograd.grad(y, leaves[:2], dy), *torch.autograd.grad(e, (x, ws), dy)

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step()
    torch.cuda.current_stream().wait_stream(side)
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        kept = step()
    ordinary = [t.detach().clone() for t in (x, w, ws, m, dy)]
    for far in (1.0, 2.0 ** 11, 2.0 ** -12, 2.0 ** 10, 1.0):
        with torch.no_grad():
            for t, o in zip((x, w, ws, m, dy), ordinary):
                t.copy_(o if far >= 1 or t is m or t is dy else o * 2.0 ** 24)
            m.mul_(far), dy.mul_(far)
        g.replay()
        torch.cuda.synchronize()
        for a, b in zip([t.clone() for t in kept], step()):
            assert torch.equal(a, b) and a.isfinite().all() and (a != 0).any()


def test_slopes_at_infinity():
    """Where an activation is a straight line in the end its slope is that line's, at infinity, too; what comes from there stays with its own row and feature."""
    from lmz_b200 import linear
    inf = float("inf")
    x = torch.tensor([[inf], [-inf], [2.0]], dtype=BF16, device="cuda").requires_grad_(True)
    w, dy = torch.ones((1, 1), dtype=BF16, device="cuda"), torch.tensor([[3.0], [5.0], [0.0]], dtype=BF16, device="cuda")
    for kind in ("relu", "gelu_tanh"):
        y = linear.project(x, w, activation=kind)
        (dx,) = torch.autograd.grad(y, x, dy)
        assert y[0, 0] == inf and dx[:, 0].tolist() == [3.0, 0.0, 0.0]
