"""Norms with the residual's addition, their output in 8 bits and their gradients, against their definitions in 64 bits (tolerances: layers.py)."""
import pytest
import torch

from layers import STEP, close, norm_steps, norms as want_norms

pytestmark = pytest.mark.gpu

ALL = [torch.bfloat16, torch.float16, torch.float32]
EPS = 1e-5


@pytest.fixture(autouse=True)
def _library(gpu):
    return gpu


def _randn(seed, shape, dtype, std=1.0):
    g = torch.Generator(device="cuda")
    g.manual_seed(seed)
    return (torch.randn(shape, generator=g, device="cuda") * std).to(dtype)


def _inputs(rows, dim, dtype, wdtype=None):
    return _randn(1, (rows, dim), dtype), _randn(2, (rows, dim), dtype, 2.0), (1 + 0.3 * _randn(3, dim, torch.float32)).to(wdtype or dtype)


# one element, fewer than a thread's, a thread's and one more, a warp's, a block's, rows that no vector fits, the first that stay out of registers, long ones
SHAPES = [(1, 1), (3, 2), (5, 7), (2, 8), (7, 16), (9, 17), (33, 64), (300, 250), (64, 511), (65, 512), (17, 513), (3001, 96), (31, 997), (12, 4096), (5, 4104), (3, 8191),
          (4, 16384), (2, 16385), (3, 16392), (2, 40000)]


@pytest.mark.parametrize("dtype", ALL)
@pytest.mark.parametrize("rows, dim", SHAPES)
def test_norm(dtype, rows, dim):
    from lmz_b200 import norms
    x, r, w = _inputs(rows, dim, dtype)
    close(norms.rms_norm(x, w, eps=EPS), want_norms(x, w, eps=EPS)["y"])
    y, s = norms.rms_norm(x, w, r, eps=EPS)
    want = want_norms(x, w, r, EPS)
    close(s, want["s"])
    close(y, want["y"])
    assert y.is_contiguous() and y.dtype == s.dtype == dtype


@pytest.mark.parametrize("dtype", ALL)
@pytest.mark.parametrize("residual", [False, True])
@pytest.mark.parametrize("rows, dim", SHAPES + [(0, 64), (20000, 40), (1500, 4096)])
def test_norm_gradient(dtype, residual, rows, dim):
    from lmz_b200 import norms
    x, r, w = _inputs(rows, dim, dtype)
    dy, ds = _randn(4, (rows, dim), dtype), _randn(5, (rows, dim), dtype)
    leaves = [t.requires_grad_(True) for t in ((x, r, w) if residual else (x, w))]
    for again in range(2):
        out = norms.rms_norm(x, w, r if residual else None, eps=EPS)
        got = torch.autograd.grad(out, leaves, (dy, ds) if residual else dy)
        if again:
            assert all(torch.equal(a, b) for a, b in zip(got, first))
        first = got
    with torch.no_grad():
        want = want_norms(x, w, r if residual else None, EPS, dy, ds if residual else None)
    close(got[0], want["dx"])
    close(got[-1], want["dweight"])
    if residual:
        assert torch.equal(got[1], got[0])


@pytest.mark.parametrize("dtype", ALL[:2])
def test_norm_with_a_weight_in_32_bits(dtype):
    from lmz_b200 import norms
    for rows, dim in ((7, 96), (33, 1000), (5, 250), (3, 77), (2, 17000)):
        x, r, w = _inputs(rows, dim, dtype, torch.float32)
        dy = _randn(4, (rows, dim), dtype)
        x.requires_grad_(True), w.requires_grad_(True)
        y = norms.rms_norm(x, w, eps=EPS)
        dx, dw = torch.autograd.grad(y, (x, w), dy)
        with torch.no_grad():
            want = want_norms(x, w, None, EPS, dy)
            assert dw.dtype == torch.float32
            close(y, want["y"]), close(dx, want["dx"]), close(dw, want["dweight"])


def test_only_the_gradients_that_are_wanted():
    from lmz_b200 import norms
    x, r, w = _inputs(40, 256, torch.bfloat16)
    dy, ds = _randn(4, (40, 256), torch.bfloat16), _randn(5, (40, 256), torch.bfloat16)
    every = [t.clone().requires_grad_(True) for t in (x, r, w)]
    full = torch.autograd.grad(norms.rms_norm(every[0], every[2], every[1]), every, (dy, ds))
    for i, name in enumerate("xrw"):
        leaves = [x, r, w]
        leaves[i] = leaves[i].clone().requires_grad_(True)
        (got,) = torch.autograd.grad(norms.rms_norm(leaves[0], leaves[2], leaves[1]), leaves[i], (dy, ds))
        assert torch.equal(got, full[i]), name
    # the stream alone, and the norm alone
    leaves = [t.clone().requires_grad_(True) for t in (x, r, w)]
    y, s = norms.rms_norm(leaves[0], leaves[2], leaves[1])
    got = torch.autograd.grad(s, leaves, ds, retain_graph=True)
    assert torch.equal(got[0], ds) and torch.equal(got[1], ds) and (got[2] == 0).all()
    got = torch.autograd.grad(y, leaves, dy)
    want = want_norms(x, w, r, 1e-6, dy)
    close(got[0], want["dx"])
    assert torch.equal(got[2], full[2])


@pytest.mark.parametrize("dtype", ALL)
@pytest.mark.parametrize("offset, stride", [(0, 264), (1, 257), (2, 258), (4, 260), (0, 0), (8, 256)])
def test_rows_of_any_stride_and_alignment(dtype, offset, stride):
    from lmz_b200 import norms
    block = _randn(6, (40 * stride + 300,), dtype)
    x = block[offset:].as_strided((40, 256), (stride, 1))
    w = _randn(7, (300,), dtype)[offset:offset + 256]
    r = _randn(8, (40, 300), dtype)[:, offset:offset + 256]
    y, s = norms.rms_norm(x, w, r, eps=EPS)
    want = want_norms(x, w, r, EPS)
    close(s, want["s"]), close(y, want["y"])
    t = _randn(9, (256, 40), dtype).t()                    # columns next to each other
    close(norms.rms_norm(t, w, eps=EPS), want_norms(t, w, eps=EPS)["y"])
    cube = _randn(10, (5, 256, 8), dtype).transpose(1, 2)
    assert torch.equal(norms.rms_norm(cube, w), norms.rms_norm(cube.contiguous().reshape(40, 256), w).reshape(5, 8, 256))
    line = _randn(11, 256, dtype)
    assert norms.rms_norm(line, w).shape == (256,) and norms.rms_norm_8bit(line, w)[1].shape == ()
    # gradients of what does not lie in rows
    x2, dy = x.clone(), _randn(12, (40, 256), dtype).t().contiguous().t()
    lone = t.detach().requires_grad_(True)
    (dx,) = torch.autograd.grad(norms.rms_norm(lone, w, eps=EPS), lone, dy)
    close(dx, want_norms(t, w, None, EPS, dy)["dx"])
    del x2


def _eight_bits_hold(q, scale, want, dtype):
    """q * scale is y rounded to 8 bits; `want`: y in 64 bits and what 32 bits may be off."""
    y, off = want
    most = y.abs().amax(-1)
    lo, hi = (most - off.amax(-1)) / 448, (most + off.amax(-1)) / 448
    assert ((scale.double() >= (lo * (1 - STEP)).clamp_min(2.0 ** -126)) & (scale.double() <= (hi * (1 + STEP)).clamp_min(2.0 ** -126))).all()
    # half a step of 3 bits of mantissa (2^-4), half the smallest number (2^-10)
    bound = off + 2 ** -4 * (y.abs() + off) * (1 + 4 * STEP) + 2 ** -10 * scale.double()[..., None] * (1 + 4 * STEP)
    close(q.double() * scale.double()[..., None], (y, bound))


@pytest.mark.parametrize("dtype", ALL)
@pytest.mark.parametrize("rows, dim", SHAPES + [(0, 64)])
def test_norm_in_8_bits(dtype, rows, dim):
    from lmz_b200 import norms
    x, r, w = _inputs(rows, dim, dtype)
    q, scale = norms.rms_norm_8bit(x, w, eps=EPS)
    assert q.dtype == torch.float8_e4m3fn and q.shape == x.shape and scale.shape == (rows,)
    _eight_bits_hold(q, scale, want_norms(x, w, eps=EPS)["wide"], dtype)
    q, scale, s = norms.rms_norm_8bit(x, w, r, eps=EPS)
    want = want_norms(x, w, r, EPS)
    close(s, want["s"])
    _eight_bits_hold(q, scale, want["wide"], dtype)
    q, scale = norms.to_8bit(x)
    _eight_bits_hold(q, scale, (x.double(), 0 * x.double()), dtype)
    # without a norm there is nothing but one division and one rounding
    # (by a tensor: torch divides by a number as a product with its reciprocal, which is another rounding)
    most = x.float().abs().amax(-1)
    by = (most / torch.full_like(most, 448)).clamp_min(2.0 ** -126)
    assert torch.equal(scale, by) and torch.equal(q.view(torch.uint8), (x.float() / by[:, None]).to(torch.float8_e4m3fn).view(torch.uint8))


def test_rows_that_are_zero_or_not_finite():
    from lmz_b200 import norms
    inf, nan = float("inf"), float("nan")
    x = _randn(13, (6, 300), torch.bfloat16)
    x[0], x[1, 17], x[2, 299], x[3, 5] = 0, inf, nan, -inf
    w = torch.ones(300, dtype=torch.bfloat16, device="cuda")
    q, scale = norms.to_8bit(x)
    assert scale[0] == 2.0 ** -126 and (q[0].float() == 0).all()
    assert scale[1] == inf and q[1, 17].float().isnan() and (q[1, :17].float() == 0).all()
    assert scale[2].isnan() and q[2].float().isnan().all() and scale[3] == inf
    assert scale[4:].isfinite().all()
    y = norms.rms_norm(x, w)
    n = x.float() * (x.float().square().mean(1, keepdim=True) + 1e-6).rsqrt()
    assert torch.equal(y.isnan(), n.isnan()) and (y[0] == 0).all() and y[4:].isfinite().all()
    q, scale = norms.rms_norm_8bit(x, w)
    assert scale[0] == 2.0 ** -126 and (q[0].float() == 0).all() and q[2].float().isnan().all() and scale[1:4].isnan().all() and scale[4:].isfinite().all()
    assert norms.rms_norm(x[:1], w, eps=0.0).isnan().all()           # 0 / 0


def test_more_than_2_32_elements():
    from lmz_b200 import norms
    rows, dim = 1_050_000, 4104
    x = torch.empty((rows, dim), dtype=torch.bfloat16, device="cuda").fill_(1.0)
    at = torch.tensor([0, 1, rows // 2, rows - 2, rows - 1], device="cuda")
    x[at] = _randn(14, (5, dim), torch.bfloat16)
    w = _randn(15, dim, torch.bfloat16)
    y = norms.rms_norm(x, w, eps=EPS)
    close(y[at], want_norms(x[at], w, eps=EPS)["y"])
    del y
    q, scale = norms.to_8bit(x)
    want, by = norms.to_8bit(x[at])
    assert torch.equal(q.view(torch.uint8)[at], want.view(torch.uint8)) and torch.equal(scale[at], by)


def test_captured_and_on_another_stream():
    from lmz_b200 import norms
    x, r, w = _inputs(50, 1000, torch.bfloat16)
    dy = _randn(4, (50, 1000), torch.bfloat16)
    w.requires_grad_(True)

    def step():
        y, s = norms.rms_norm(x, w, r)
        q = norms.rms_norm_8bit(x, w.detach(), r)
        return (y, s, *q, *torch.autograd.grad(y, w, dy))

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step()
    torch.cuda.current_stream().wait_stream(side)
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        kept = step()
    x.copy_(_randn(16, (50, 1000), torch.bfloat16))
    g.replay()
    g.replay()
    for a, b in zip(kept, step()):
        assert torch.equal(a.detach().view(torch.uint8), b.detach().view(torch.uint8))


def test_differences():
    """Gradients against differences of the definition in 64 bits."""
    from lmz_b200 import norms
    x, r, w = (t.requires_grad_(True) for t in _inputs(4, 12, torch.float32))
    dy, ds = _randn(4, (4, 12), torch.float32), _randn(5, (4, 12), torch.float32)
    got = torch.autograd.grad(norms.rms_norm(x, w, r, eps=EPS), (x, r, w), (dy, ds))

    def loss(x, r, w):
        s = x + r
        return ((s * (s.square().mean(1, keepdim=True) + EPS).rsqrt() * w) * dy.double()).sum() + (s * ds.double()).sum()

    at = [t.detach().double() for t in (x, r, w)]
    h = 1e-5
    for i, t in enumerate(at):
        for j in range(t.numel()):
            d = torch.zeros_like(t).view(-1)
            d[j] = h
            hi, lo = ([v + d.view_as(v) * sign if k == i else v for k, v in enumerate(at)] for sign in (1, -1))
            # (x + r is rounded to 32 bits, and differences are good to h^2)
            assert abs(float(loss(*hi) - loss(*lo)) / (2 * h) - float(got[i].reshape(-1)[j])) < 1e-4


def test_steps_are_as_many_as_said():
    assert norm_steps(16384) == 64 and norm_steps(16385) == 80
