"""Calls of norms, products and experts' products that their documentation allows: the same tensor twice, broadcast inputs, gradients that accumulate, threads,
streams, padded batches, sizes at the ends of their ranges, tensors beyond 32 bits."""
import threading

import pytest
import torch

from layers import close, norms as want_norms, products as want_products

pytestmark = pytest.mark.gpu

BF16 = torch.bfloat16


@pytest.fixture(autouse=True)
def _library(gpu):
    yield gpu
    from lmz_b200 import adapters
    adapters.check()


def _randn(seed, shape, dtype=BF16, std=1.0):
    g = torch.Generator(device="cuda")
    g.manual_seed(seed)
    return (torch.randn(shape, generator=g, device="cuda") * std).to(dtype)


def _off(a, b):
    return float((a.detach().double() - b.detach().double()).norm() / b.detach().double().norm())


def test_one_tensor_in_several_places():
    from lmz_b200 import linear, norms
    x, w, dy = _randn(1, (40, 64)), _randn(2, (64, 64), std=0.1), _randn(3, (40, 64))
    gamma = _randn(4, 64)
    lone = x.clone().requires_grad_(True)
    y, s = norms.rms_norm(lone, gamma, lone)
    (d,) = torch.autograd.grad(y, lone, dy)
    apart = [x.clone().requires_grad_(True) for _ in range(2)]
    a, b = torch.autograd.grad(norms.rms_norm(apart[0], gamma, apart[1])[0], apart, dy)
    assert torch.equal(d, a + b)
    lone = x.clone().requires_grad_(True)
    (d,) = torch.autograd.grad(linear.project(lone, w, activation="silu", times=lone, residual=lone), lone, dy)
    apart = [x.clone().requires_grad_(True) for _ in range(3)]
    a, b, c = torch.autograd.grad(linear.project(apart[0], w, activation="silu", times=apart[1], residual=apart[2]), apart, dy)
    # (three gradients of 16 bits are added up, in whichever order: two roundings)
    assert ((d.double() - (a.double() + b.double() + c.double())).abs() <= 2 ** -7 * (a.double().abs() + b.double().abs() + c.double().abs())).all()
    square = linear.project(w, w)                           # (x and the weight)
    close(square, want_products(w, w)["y"])


def test_gradients_that_accumulate_share_nothing():
    from lmz_b200 import linear, norms
    x, r, w, g = (t.requires_grad_(True) for t in (_randn(1, (24, 32)), _randn(2, (24, 32)), _randn(3, (32, 32), std=0.2), _randn(4, 32)))
    dy = _randn(5, (24, 32))
    kept = dy.clone()
    y, s = norms.rms_norm(x, g, r)
    linear.project(y, w, residual=s).backward(dy)
    first = [t.grad.clone() for t in (x, r, w, g)]
    with torch.no_grad():
        x.grad.zero_()
    assert torch.equal(r.grad, first[1]) and torch.equal(dy, kept)
    with torch.no_grad():
        x.grad.copy_(first[0])
    y, s = norms.rms_norm(x, g, r)
    linear.project(y, w, residual=s).backward(dy)
    for t, once in zip((x, r, w, g), first):
        assert torch.equal(t.grad, (once.float() * 2).to(BF16))


def test_broadcast_inputs():
    from lmz_b200 import linear, norms
    row, w, dy = _randn(1, (1, 48)).requires_grad_(True), _randn(2, (48, 48), std=0.2), _randn(3, (30, 48))
    m = _randn(4, (48,)).requires_grad_(True)
    y = linear.project(row.expand(30, 48), w, activation="gelu", times=m.expand(30, 48), residual=row.expand(30, 48))
    got = torch.autograd.grad(y, (row, m), dy)
    whole = [row.detach().repeat(30, 1).requires_grad_(True), m.detach().repeat(30, 1).requires_grad_(True)]
    other = torch.autograd.grad(linear.project(whole[0], w, activation="gelu", times=whole[1], residual=whole[0]), whole, dy)
    assert torch.equal(y, linear.project(whole[0].detach(), w, activation="gelu", times=whole[1].detach(), residual=whole[0].detach()))
    assert _off(got[0], other[0].double().sum(0, keepdim=True)) < 4 * 2 ** -8 and _off(got[1], other[1].double().sum(0)) < 4 * 2 ** -8
    g = _randn(5, 48)
    assert torch.equal(norms.rms_norm(row.detach().expand(7, 48), g), norms.rms_norm(row.detach().repeat(7, 1), g))


def test_second_derivatives_are_refused():
    from lmz_b200 import linear, norms
    x, w, g = (t.requires_grad_(True) for t in (_randn(1, (8, 16)), _randn(2, (16, 16)), _randn(3, 16)))
    for y in (norms.rms_norm(x, g), linear.project(x, w, activation="silu")):
        (d,) = torch.autograd.grad(y.float().square().sum(), x, create_graph=True)
        with pytest.raises(RuntimeError, match="once_differentiable|differentiated twice"):
            d.float().sum().backward()


def test_what_the_gradients_need_may_not_be_changed():
    from lmz_b200 import linear, norms
    x, w = _randn(1, (8, 16)).requires_grad_(True), _randn(2, (16, 16)).requires_grad_(True)
    y, s = norms.rms_norm(x, w[0], _randn(3, (8, 16)))
    with torch.no_grad():
        s.zero_()
    with pytest.raises(RuntimeError, match="modified by an inplace"):
        y.float().sum().backward()
    y = linear.project(x, w, activation="silu")
    with torch.no_grad():
        w.zero_()
    with pytest.raises(RuntimeError, match="modified by an inplace"):
        y.float().sum().backward()


def test_several_threads_at_once():
    from lmz_b200 import experts, linear, norms
    x, w, g = _randn(1, (130, 264)), _randn(2, (200, 264), std=0.1), _randn(3, 264)
    ws, offsets = _randn(4, (3, 200, 264), std=0.1), torch.tensor([0, 60, 60, 130], device="cuda")
    dy = _randn(5, (130, 200))

    def work():
        v, u = x.clone().requires_grad_(True), w.clone().requires_grad_(True)
        y = linear.project(norms.rms_norm(v, g), u, activation="gelu_tanh")
        return [y.detach(), *torch.autograd.grad(y, (v, u), dy), experts.project(x, ws, offsets), *norms.rms_norm_8bit(x, g)]

    want = work()
    torch.cuda.synchronize()
    bad = []

    def run(k):
        try:
            with torch.cuda.stream(torch.cuda.Stream()):
                for _ in range(20):
                    if not all(torch.equal(a.view(torch.uint8), b.view(torch.uint8)) for a, b in zip(work(), want)):
                        bad.append(k)
        except Exception as e:                              # noqa: BLE001
            bad.append(e)

    threads = [threading.Thread(target=run, args=(k,)) for k in range(4)]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    assert not bad, bad


def test_two_captured_graphs_replayed_in_turn():
    from lmz_b200 import linear, norms
    inputs = [(_randn(k, (90, 77)), _randn(k + 10, (33, 77), std=0.1).requires_grad_(True), _randn(k + 20, 77).requires_grad_(True), _randn(k + 30, (90, 33))) for k in range(2)]

    def step(x, w, g, dy):
        y = linear.project(norms.rms_norm(x, g), w, activation="silu")
        return [y.detach(), *torch.autograd.grad(y, (w, g), dy)]

    graphs, kept = [], []
    for i in inputs:
        side = torch.cuda.Stream()
        side.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(side):
            step(*i)
        torch.cuda.current_stream().wait_stream(side)
        graphs.append(torch.cuda.CUDAGraph())
        with torch.cuda.graph(graphs[-1], pool=graphs[0].pool() if kept else None):
            kept.append(step(*i))
    for _ in range(3):
        for k, g in enumerate(graphs):
            g.replay()
            torch.cuda.synchronize()
            for a, b in zip([t.clone() for t in kept[k]], step(*inputs[k])):
                assert torch.equal(a, b)


def test_the_kernel_in_front_may_write_what_is_multiplied():
    """Weights and rows that a kernel writes right in front of a product, time after time: tiles that are sent for early are not stale."""
    from lmz_b200 import adapters, linear
    x, base = _randn(1, (4, 4096)), _randn(2, (4096, 4096), std=0.02)
    a, b = _randn(3, (16, 4096), std=0.02), _randn(4, (4096, 16), std=0.5)
    w, other = base.clone(), base.clone()
    for k in range(30):
        scale = 0.25 * (k % 5)
        adapters.merge(base, a, b, scale=scale, out=w)
        y = linear.project(x, w)
        w.mul_(2)
        z = linear.project(x, w)
        torch.cuda.synchronize()
        adapters.merge(base, a, b, scale=scale, out=other)
        torch.cuda.synchronize()
        assert torch.equal(y, linear.project(x, other)) and torch.equal(z, linear.project(x, other * 2))


def test_results_and_rows_beyond_32_bits():
    from lmz_b200 import experts, linear
    rows, inp, out = 300_001, 32, 14_400                    # 4.3e9 results
    x, w = _randn(1, (rows, inp)), _randn(2, (out, inp), std=0.2)
    at = torch.tensor([0, 1, 149_130, 149_131, 298_261, 298_262, rows - 2, rows - 1], device="cuda")
    y = linear.project(x, w, activation="relu")
    want = want_products(x[at], w, kind="relu")["y"]
    close(y[at], want)
    del y
    ws = torch.stack((w, -w))
    y = experts.project(x, ws, torch.tensor([0, 298_262, rows - 1], device="cuda"), activation="relu", times=x[:, :1].expand(rows, out))
    assert (y[-1] == 0).all()
    for t in at.tolist()[:-1]:
        close(y[t:t + 1], want_products(x[t:t + 1], ws[1] if t >= 298_262 else ws[0], kind="relu", times=x[t:t + 1, :1].expand(1, out))["y"])


def test_a_gradient_beyond_32_bits():
    from lmz_b200 import linear
    rows, inp, out = 270_000, 16_000, 8                     # 4.3e9 elements of x and of its gradient
    x, w = torch.empty((rows, inp), dtype=BF16, device="cuda").fill_(0.5), _randn(2, (out, inp), std=0.01)
    dy = _randn(3, (rows, out))
    x.requires_grad_(True)
    y = linear.project(x, w)
    (dx,) = torch.autograd.grad(y, x, dy)
    with torch.no_grad():
        for t in (0, 134_217, 268_436, rows - 1):
            got = want_products(x[t:t + 1], w, dy=dy[t:t + 1])
            close(y[t:t + 1], got["y"]), close(dx[t:t + 1], got["dx"])


@pytest.mark.parametrize("inp, out", [(1, 70_000), (70_000, 1), (16, 100_003), (100_008, 24)])
def test_long_and_thin_weights(inp, out):
    from lmz_b200 import linear
    x, w, dy = _randn(1, (3, inp)).requires_grad_(True), _randn(2, (out, inp), std=0.02).requires_grad_(True), _randn(3, (3, out))
    y = linear.project(x, w, activation="gelu")
    dx, dw = torch.autograd.grad(y, (x, w), dy)
    with torch.no_grad():
        want = want_products(x, w, kind="gelu", dy=dy)
        close(y, want["y"]), close(dx, want["dx"]), close(dw, want["dweight"])


def test_long_rows_normed():
    from lmz_b200 import norms
    dim = 300_001
    x, w, dy = _randn(1, (3, dim)).requires_grad_(True), _randn(2, dim).requires_grad_(True), _randn(3, (3, dim))
    y = norms.rms_norm(x, w)
    dx, dw = torch.autograd.grad(y, (x, w), dy)
    with torch.no_grad():
        want = want_norms(x, w, None, 1e-6, dy)
        close(y, want["y"]), close(dx, want["dx"]), close(dw, want["dweight"])


def test_infinities_in_one_row_or_feature():
    """What is not finite reaches its own row and its own feature, and nothing else."""
    from lmz_b200 import linear
    inf, nan = float("inf"), float("nan")
    for rows, inp, out in ((40, 72, 50), (300, 128, 256), (1, 64, 64)):
        x, w, b, m = _randn(1, (rows, inp)), _randn(2, (out, inp), std=0.2), _randn(3, out), _randn(4, (rows, out))
        fine = linear.project(x, w, b, "silu", m)
        x2, w2, b2 = x.clone(), w.clone(), b.clone()
        row, feature = rows // 2, out // 3
        x2[row, 0], w2[feature, inp - 1], b2[feature + 1] = inf, nan, inf
        got = linear.project(x2, w2, b2, "silu", m)
        keep = torch.ones((rows, out), dtype=torch.bool, device="cuda")
        keep[row], keep[:, feature], keep[:, feature + 1] = False, False, False
        assert torch.equal(got[keep], fine[keep]) and got[:, feature].isnan().all()


def test_activations_at_the_ends_of_their_range():
    """Where exponentials over- and underflow: z itself, zero, or what lies between, and never NaN for a finite z."""
    from lmz_b200 import linear
    z = torch.tensor([0.0, -0.0, 1e-30, -1e-30, 3.0, -3.0, 20.0, -20.0, 88.0, -88.0, 89.0, -89.0, 120.0, -120.0, 1e4, -1e4, 1e15, -1e15, 3e38, -3e38], dtype=BF16, device="cuda")
    x, w, dy = z[:, None].clone().requires_grad_(True), torch.ones((1, 1), dtype=BF16, device="cuda"), torch.ones((len(z), 1), dtype=BF16, device="cuda")
    for kind in ("relu", "silu", "gelu", "gelu_tanh"):
        y = linear.project(x, w, activation=kind)
        (dx,) = torch.autograd.grad(y, x, dy)
        with torch.no_grad():
            assert y.isfinite().all() and dx.isfinite().all()
            small = z.abs() < 1e5                            # (of larger ones z itself and zero are exact)
            want = want_products(x[small], w, kind=kind, dy=dy[small])
            close(y[small], want["y"]), close(dx[small], want["dx"])
            assert torch.equal(y[~small][:, 0], z[~small].clamp_min(0)) and torch.equal(dx[~small][:, 0], (z[~small] > 0).to(BF16))


def test_experts_weights_in_other_orders():
    """Side by side instead of behind each other, one for all of them, in reverse, every other one."""
    from lmz_b200 import experts
    x, dy, offsets, starts = _randn(1, (90, 64)), _randn(2, (90, 48)), torch.tensor([0, 30, 41, 90], device="cuda"), [0, 30, 41, 90]
    block = _randn(3, (48, 3, 64), std=0.2)
    for w in (block.transpose(0, 1), block[:, :1].transpose(0, 1).expand(3, 48, 64), _randn(4, (6, 48, 64), std=0.2)[::2], _randn(5, (3, 96, 64), std=0.2)[:, ::2], _randn(6, (3, 48, 80), std=0.2)[:, :, 8:72]):
        leaf = w.detach().requires_grad_(True)
        v = x.clone().requires_grad_(True)
        y = experts.project(v, leaf, offsets)
        dx, dw = torch.autograd.grad(y, (v, leaf), dy)
        with torch.no_grad():
            want = want_products(x, w, dy=dy, starts=starts)
            close(y, want["y"]), close(dx, want["dx"]), close(dw, want["dweight"])


def test_a_padded_batch():
    """Rows behind the last sequence: zeros out, none of theirs in any gradient, whatever they hold."""
    from lmz_b200 import experts
    x, w, dy, m = _randn(1, (200, 40)), _randn(2, (4, 24, 40), std=0.2), _randn(3, (200, 24)), _randn(4, (200, 24))
    offsets = torch.tensor([0, 50, 50, 120, 137], dtype=torch.int32, device="cuda")
    x[137:], dy[137:], m[137:] = float("nan"), float("inf"), float("nan")
    leaves = [t.requires_grad_(True) for t in (x, w, m)]
    y = experts.project(x, w, offsets, activation="gelu", times=m)
    grads = torch.autograd.grad(y, leaves, dy)
    assert (y[137:] == 0).all() and (grads[0][137:] == 0).all() and (grads[2][137:] == 0).all() and all(g.isfinite().all() for g in grads)
    short = [t.detach()[:137].clone().requires_grad_(True) if t.dim() == 2 else t for t in leaves]
    again = experts.project(short[0], short[1], offsets, activation="gelu", times=short[2])
    for a, b in zip((y, *grads), (again, *torch.autograd.grad(again, short, dy[:137]))):
        assert torch.equal(a[:137], b) if a.dim() == 2 else torch.equal(a, b)
