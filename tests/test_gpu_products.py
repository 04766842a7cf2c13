"""Products with bias, activation, factor and residual in their epilogue, in 16 and in 8 bits, with experts' weights, and their gradients,
against their definitions in 64 bits (tolerances: layers.py)."""
import itertools

import numpy as np
import pytest
import torch

from layers import act, close, products as want_products

pytestmark = pytest.mark.gpu

DTYPES = [torch.bfloat16, torch.float16]
ACTS = [None, "relu", "silu", "gelu", "gelu_tanh"]


@pytest.fixture(autouse=True)
def _library(gpu):
    yield gpu
    from lmz_b200 import adapters
    adapters.check()                                       # (no kernel has given up waiting)


def _randn(seed, shape, dtype, std=1.0):
    g = torch.Generator(device="cuda")
    g.manual_seed(seed)
    return (torch.randn(shape, generator=g, device="cuda") * std).to(dtype)


def _check(got, want):
    for name, t in got.items():
        if t is not None:
            try:
                close(t, want[name])
            except AssertionError as e:
                raise AssertionError(f"{name}: {e}") from None


# rows, in, out: one of each, a tile of the tensor core and its neighbours, sizes that no vector fits, few rows and wide weights, many rows
SHAPES = [(1, 1, 1), (1, 8, 8), (3, 5, 7), (1, 64, 128), (2, 72, 136), (16, 64, 128), (17, 65, 129), (31, 200, 96), (64, 128, 256), (100, 250, 331), (127, 512, 127),
          (128, 256, 128), (129, 264, 384), (255, 129, 513), (256, 320, 256), (257, 1000, 264), (333, 777, 1001), (1, 4096, 1024), (1, 1001, 4097), (8, 2048, 512), (600, 64, 64),
          (1000, 96, 2050), (2049, 512, 300), (40, 3000, 40), (5000, 33, 17),
          # (pairs of CTAs: forwards, for the rows' gradient, for the weight's)
          (2304, 512, 2304), (2301, 520, 2311), (2304, 2304, 512), (2305, 2312, 505), (512, 2304, 2304), (501, 2312, 2307)]


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("rows, inp, out", SHAPES)
def test_product(dtype, rows, inp, out):
    from lmz_b200 import linear
    x, w = _randn(1, (rows, inp), dtype), _randn(2, (out, inp), dtype, inp ** -0.5)
    _check({"y": linear.project(x, w)}, want_products(x, w))
    b, m, r = _randn(3, out, dtype), _randn(4, (rows, out), dtype), _randn(5, (rows, out), dtype, 3.0)
    y = linear.project(x, w, bias=b, activation="silu", times=m, residual=r)
    assert y.is_contiguous() and y.dtype == dtype and y.shape == (rows, out)
    _check({"y": y}, want_products(x, w, b, "silu", m, r))


@pytest.mark.parametrize("kind", ACTS)
@pytest.mark.parametrize("with_bias, with_times, with_residual", list(itertools.product([False, True], repeat=3)))
def test_every_epilogue(kind, with_bias, with_times, with_residual):
    from lmz_b200 import linear
    for dtype, (rows, inp, out) in ((torch.bfloat16, (70, 96, 200)), (torch.float16, (19, 50, 77))):
        x, w = _randn(1, (rows, inp), dtype), _randn(2, (out, inp), dtype, inp ** -0.5 * 2)
        b = _randn(3, out, dtype) if with_bias else None
        m = _randn(4, (rows, out), dtype) if with_times else None
        r = _randn(5, (rows, out), dtype) if with_residual else None
        dy = _randn(6, (rows, out), dtype)
        plain = linear.project(x, w, bias=b, activation=kind, times=m, residual=r)
        given = {"x": x, "weight": w, "bias": b, "times": m, "residual": r}
        leaves = [t.requires_grad_(True) for t in given.values() if t is not None]
        y = linear.project(x, w, bias=b, activation=kind, times=m, residual=r)
        assert torch.equal(y, plain)
        got = dict(zip(("d" + k for k, t in given.items() if t is not None), torch.autograd.grad(y, leaves, dy)))
        with torch.no_grad():
            if with_residual:
                assert torch.equal(got.pop("dresidual"), dy)
            _check({"y": y} | got, want_products(x, w, b, kind, m, r, dy))


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("rows, inp, out", SHAPES + [(0, 64, 32)])
def test_gradients(dtype, rows, inp, out):
    from lmz_b200 import linear
    x, w, b = _randn(1, (rows, inp), dtype), _randn(2, (out, inp), dtype, inp ** -0.5), _randn(3, out, dtype)
    dy = _randn(6, (rows, out), dtype)
    leaves = [t.requires_grad_(True) for t in (x, w, b)]
    for kind in (None, "gelu"):
        first = torch.autograd.grad(linear.project(x, w, bias=b, activation=kind), leaves, dy)
        again = torch.autograd.grad(linear.project(x, w, bias=b, activation=kind), leaves, dy)
        assert all(torch.equal(p, q) for p, q in zip(first, again))
        with torch.no_grad():
            _check(dict(zip(("dx", "dweight", "dbias"), first)), want_products(x, w, b, kind, dy=dy))


def test_only_the_gradients_that_are_wanted():
    from lmz_b200 import linear
    x, w, b = _randn(1, (50, 72), torch.bfloat16), _randn(2, (90, 72), torch.bfloat16, 0.2), _randn(3, 90, torch.bfloat16)
    m, r, dy = _randn(4, (50, 90), torch.bfloat16), _randn(5, (50, 90), torch.bfloat16), _randn(6, (50, 90), torch.bfloat16)
    every = [t.clone().requires_grad_(True) for t in (x, w, b, m, r)]
    full = torch.autograd.grad(linear.project(every[0], every[1], every[2], "silu", every[3], every[4]), every, dy)
    for i in range(5):
        leaves = [x, w, b, m, r]
        leaves[i] = leaves[i].clone().requires_grad_(True)
        (got,) = torch.autograd.grad(linear.project(leaves[0], leaves[1], leaves[2], "silu", leaves[3], leaves[4]), leaves[i], dy)
        assert torch.equal(got, full[i])


@pytest.mark.parametrize("rows, inp, out", [(1, 16, 16), (1, 4096, 512), (5, 20, 9), (16, 128, 128), (40, 1000, 333), (130, 256, 384), (257, 1040, 264), (3, 17, 8), (1000, 96, 2050)])
@pytest.mark.parametrize("dtype", DTYPES)
def test_product_in_8_bits(rows, inp, out, dtype):
    from lmz_b200 import linear, norms
    q, s = norms.to_8bit(_randn(1, (rows, inp), torch.float32, 3.0))
    wq, ws = norms.to_8bit(_randn(2, (out, inp), torch.float32, 0.02))
    b, m, r = _randn(3, out, dtype), _randn(4, (rows, out), dtype), _randn(5, (rows, out), dtype)
    if dtype is torch.bfloat16:
        _check({"y": linear.project_8bit(q, s, wq, ws)}, want_products(q.float(), wq.float(), x_scale=s, weight_scale=ws, dtype=dtype))
    got = linear.project_8bit(q, s, wq, ws, bias=b, activation="gelu", times=m, residual=r, dtype=dtype)
    assert got.dtype == dtype
    _check({"y": got}, want_products(q.float(), wq.float(), b, "gelu", m, r, x_scale=s, weight_scale=ws, dtype=dtype))


def _starts(seed, rows, experts, how):
    rng = np.random.default_rng(seed)
    if how == "one":
        counts = np.zeros(experts, dtype=np.int64)
        counts[experts // 2] = rows
    elif how == "even":
        counts = np.full(experts, rows // experts)
    else:
        p = np.exp(rng.standard_normal(experts))
        p[1::3] = 0
        counts = rng.multinomial(rows, p / p.sum())
    lead = 3 if how == "inside" else 0
    return [lead, *(lead + np.cumsum(counts)).tolist()]


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("rows, experts, inp, out, how", [(1, 1, 8, 8, "one"), (1, 4, 64, 128, "any"), (7, 3, 33, 19, "any"), (64, 64, 128, 72, "any"), (50, 8, 96, 130, "one"),
                                                          (128, 16, 512, 264, "any"), (300, 4, 200, 100, "inside"), (300, 3, 64, 256, "even"), (900, 5, 136, 520, "any"),
                                                          (2000, 6, 256, 384, "any"), (40, 1024, 40, 24, "any"), (1500, 2, 77, 333, "inside"), (0, 5, 16, 16, "even"),
                                                          (777, 7, 1024, 512, "any"),
                                                          # (pairs of CTAs)
                                                          (5000, 3, 512, 2304, "any"), (4000, 4, 2304, 520, "any"), (1500, 6, 1536, 1544, "any"), (5000, 3, 515, 2307, "inside")])
def test_experts(dtype, rows, experts, inp, out, how):
    from lmz_b200 import experts as ex
    starts = _starts(1, rows, experts, how)
    total = starts[-1] + (5 if how in ("inside", "any") else 0)
    x, w, b = _randn(1, (total, inp), dtype), _randn(2, (experts, out, inp), dtype, inp ** -0.5), _randn(3, (experts, out), dtype)
    m, dy = _randn(4, (total, out), dtype), _randn(6, (total, out), dtype)
    offsets = torch.tensor(starts, dtype=torch.int32 if inp % 2 else torch.int64, device="cuda")
    _check({"y": ex.project(x, w, offsets)}, want_products(x, w, starts=starts))
    leaves = [t.requires_grad_(True) for t in (x, w, b, m)]
    for given in (dict(), dict(bias=b, activation="silu", times=m)):
        names = ("x", "weight", "bias", "times") if given else ("x", "weight")
        wanted = leaves[:len(names)]
        y = ex.project(x, w, offsets, **given)
        first = torch.autograd.grad(y, wanted, dy)
        again = torch.autograd.grad(ex.project(x, w, offsets, **given), wanted, dy)
        assert all(torch.equal(p, q) for p, q in zip(first, again))
        with torch.no_grad():
            want = want_products(x, w, given.get("bias"), given.get("activation"), given.get("times"), dy=dy, starts=starts)
            _check({"y": y} | dict(zip(("d" + n for n in names), first)), want)


def test_nothing_of_an_expert_reaches_another():
    """Infinities and NaN in rows and weights stay with their expert, and those in rows of no expert reach nothing."""
    from lmz_b200 import experts as ex
    inf, nan = float("inf"), float("nan")
    for dtype, (inp, out) in itertools.product(DTYPES, ((72, 40), (64, 128), (33, 50))):
        starts, total = [2, 21, 21, 85, 100], 107
        x, w = _randn(1, (total, inp), dtype), _randn(2, (4, out, inp), dtype, 0.1)
        dy = _randn(3, (total, out), dtype)
        bad_x, bad_w, bad_dy = x.clone(), w.clone(), dy.clone()
        bad_x[:2], bad_x[100:], bad_x[21:85] = nan, inf, inf
        bad_w[1], bad_w[2] = nan, inf
        bad_dy[:2], bad_dy[100:], bad_dy[21:85] = nan, inf, nan
        offsets = torch.tensor(starts, device="cuda")
        got, want = [], []
        for to, v, u, d in ((got, bad_x, bad_w, bad_dy), (want, x, w, dy)):
            v, u = v.requires_grad_(True), u.requires_grad_(True)
            for kind in (None, "relu"):
                y = ex.project(v, u, offsets, activation=kind)
                to += [y.detach(), *torch.autograd.grad(y, (v, u), d)]
        fine = torch.ones(total, dtype=torch.bool, device="cuda")
        fine[21:85] = False
        for g, t in zip(got, want):
            keep = [0, 1, 3] if g.dim() == 3 else fine
            assert torch.equal(g[keep], t[keep])
        y = got[0]
        assert (y[:2] == 0).all() and (y[100:] == 0).all() and not y[21:85].isfinite().any()


def test_offsets_of_any_kind_stay_within_the_rows():
    from lmz_b200 import experts as ex
    x, w = _randn(1, (90, 64), torch.bfloat16), _randn(2, (4, 48, 64), torch.bfloat16, 0.1)
    for offsets, as_if in (([-5, 10, 2 ** 40, 3, 2 ** 50], [0, 10, 90, 90, 90]), ([20, 10, 30, 25, 60], [20, 20, 30, 30, 60]), ([-9, -8, -7, -6, -5], [0] * 5),
                           ([2 ** 33] * 5, [90] * 5)):
        v, u = x.clone().requires_grad_(True), w.clone().requires_grad_(True)
        y = ex.project(v, u, torch.tensor(offsets, device="cuda"), activation="silu")
        dy = _randn(3, (90, 48), torch.bfloat16)
        dx, dw = torch.autograd.grad(y, (v, u), dy)
        with torch.no_grad():
            _check({"y": y, "dx": dx, "dweight": dw}, want_products(v, u, kind="silu", dy=dy, starts=as_if))


@pytest.mark.parametrize("n, experts, dtype", [(0, 4, torch.int32), (1, 1, torch.int64), (1000, 7, torch.int32), (5000, 1023, torch.int64), (5000, 1024, torch.int32), (40, 8, torch.int64)])
def test_sort(n, experts, dtype):
    from lmz_b200 import experts as ex
    rng = np.random.default_rng(3)
    ids = rng.integers(-1, experts + 1, n)
    order, offsets = ex.sort(torch.from_numpy(ids).to(dtype).cuda(), experts)
    keys = np.where((ids < 0) | (ids >= experts), experts, ids)
    assert order.tolist() == np.argsort(keys, kind="stable").tolist()
    assert offsets.tolist() == np.searchsorted(np.sort(keys), np.arange(experts + 1)).tolist()


@pytest.mark.parametrize("offset, stride", [(0, 264), (1, 257), (2, 258), (4, 260), (8, 272), (0, 0)])
def test_rows_of_any_stride_and_alignment(offset, stride):
    from lmz_b200 import experts as ex, linear
    dtype = torch.bfloat16
    block = _randn(1, (70 * max(stride, 256) + 300,), dtype)
    x = block[offset:].as_strided((70, 256), (stride, 1))
    w = _randn(2, (96 * 300,), dtype, 0.06)[offset:].as_strided((96, 256), (max(stride, 256), 1))
    m = _randn(4, (70, 120), dtype)[:, offset:offset + 96]
    r = _randn(5, (70, 121), dtype)[:, offset:offset + 96]
    b, dy = _randn(3, 110, dtype)[offset:offset + 96], _randn(6, (96, 70), dtype).t()
    leaves = [t.detach().requires_grad_(True) for t in (x, w, b, m)]
    y = linear.project(leaves[0], leaves[1], leaves[2], "gelu_tanh", leaves[3], r)
    got = torch.autograd.grad(y, leaves, dy)
    with torch.no_grad():
        _check({"y": y} | dict(zip(("dx", "dweight", "dbias", "dtimes"), got)), want_products(x, w, b, "gelu_tanh", m, r, dy))
        cube = _randn(7, (5, 256, 14), dtype).transpose(1, 2)
        assert torch.equal(linear.project(cube, w), linear.project(cube.contiguous().reshape(70, 256), w).reshape(5, 14, 96))
        line = linear.project(x[3], w, times=m[3])
        assert line.shape == (96,) and torch.equal(line, linear.project(x[3:4], w, times=m[3:4])[0])
        ws = _randn(8, (3 * 100 * 300,), dtype, 0.06)[offset:].as_strided((3, 96, 256), (100 * max(stride, 256) + offset, max(stride, 256), 1))
        offsets = torch.tensor([0, 30, 30, 65], dtype=torch.int32, device="cuda")
        _check({"y": ex.project(x, ws, offsets, times=m)}, want_products(x, ws, times=m, starts=[0, 30, 30, 65]))


def test_in_8_bits_at_any_stride_and_alignment():
    from lmz_b200 import linear, norms
    for offset, stride in ((0, 272), (1, 257), (8, 264), (16, 272), (0, 0)):
        q, _ = norms.to_8bit(_randn(1, (1, 70 * 300), torch.float32))
        x = q.reshape(-1)[offset:].as_strided((70, 256), (stride, 1))
        wq, _ = norms.to_8bit(_randn(2, (1, 96 * 300), torch.float32))
        w = wq.reshape(-1)[offset:].as_strided((96, 256), (max(stride, 256), 1))
        xs, ws = _randn(3, 140, torch.float32).abs()[::2], _randn(4, 192, torch.float32).abs()[::2]
        _check({"y": linear.project_8bit(x, xs, w, ws)}, want_products(x.float(), w.float(), x_scale=xs, weight_scale=ws, dtype=torch.bfloat16))


def test_captured_and_on_another_stream():
    from lmz_b200 import experts as ex, linear
    x, w, b = _randn(1, (300, 264), torch.bfloat16), _randn(2, (200, 264), torch.bfloat16, 0.06), _randn(3, 200, torch.bfloat16)
    dy = _randn(6, (300, 200), torch.bfloat16)
    ws, offsets = _randn(7, (4, 200, 264), torch.bfloat16, 0.06), torch.tensor([0, 100, 100, 170, 290], device="cuda")
    w.requires_grad_(True), ws.requires_grad_(True), x.requires_grad_(True)

    def step():
        y = linear.project(x, w, bias=b, activation="silu")
        e = ex.project(x, ws, offsets, activation="gelu")
        return y, e, *torch.autograd.grad(y, (x, w), dy), *torch.autograd.grad(e, (x, ws), dy)

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step()
    torch.cuda.current_stream().wait_stream(side)
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        kept = step()
    with torch.no_grad():
        x.copy_(_randn(16, (300, 264), torch.bfloat16))
        offsets.copy_(torch.tensor([5, 60, 200, 201, 300]))    # (experts' rows are found on the device)
    g.replay()
    g.replay()
    for a, b2 in zip(kept, step()):
        assert torch.equal(a, b2)


def test_differences():
    """Gradients against differences of the definition in 64 bits, at points of 16 bits."""
    from lmz_b200 import experts as ex
    dtype = torch.float16
    x, w, b = _randn(1, (6, 5), dtype), _randn(2, (2, 4, 5), dtype), _randn(3, (2, 4), dtype)
    m, dy = _randn(4, (6, 4), dtype), _randn(5, (6, 4), dtype)
    starts = [1, 3, 6]
    leaves = [t.requires_grad_(True) for t in (x, w, b, m)]
    for kind in ACTS:
        got = torch.autograd.grad(ex.project(x, w, torch.tensor(starts, device="cuda"), bias=b, activation=kind, times=m), leaves, dy)

        def loss(x, w, b, m):
            z = torch.cat([x[lo:hi] @ w[e].t() + b[e] for e, (lo, hi) in enumerate(zip(starts, starts[1:]))])
            return (act(kind, z)[0] * m[starts[0]:] * dy[starts[0]:].double()).sum()

        at, h = [t.detach().double() for t in leaves], 1e-5
        with torch.no_grad():
            want = want_products(x, w, b, kind, m, dy=dy, starts=starts)
        for i, name in enumerate(("dx", "dweight", "dbias", "dtimes")):
            for j in range(at[i].numel()):
                d = torch.zeros_like(at[i]).view(-1)
                d[j] = h
                hi, lo = ([v + d.view_as(v) * sign if k == i else v for k, v in enumerate(at)] for sign in (1, -1))
                off = float(want[name][1].reshape(-1)[j])
                assert abs(float(loss(*hi) - loss(*lo)) / (2 * h) - float(got[i].reshape(-1)[j])) <= off + 1e-6, (kind, name, j)


def test_a_layers_feed_forward_half_from_an_archives_tensors():
    """Norm, gated products and back into the stream, forwards and backwards, in 8 bits, and by experts, on weights that an archive was decoded to."""
    from oracle import archive as oa, synth

    from lmz_b200 import decode, embed, experts as ex, linear, norms
    dec = decode.ArchiveDecoder(oa.write_archive([("m.safetensors", synth.llama_shard([0], 5, scale=0.125, vocab=2000, embed=True))], mapped=True))
    dec.run()
    dec.check()
    t = {name: v for (_, name), v in dec.tensors().items()}
    up, gate, down = (t[f"model.layers.0.mlp.{n}_proj.weight"] for n in ("up", "gate", "down"))
    norm, table = t["model.layers.0.post_attention_layernorm.weight"], t["model.embed_tokens.weight"]
    ids = torch.arange(0, 250, 3, device="cuda")
    stream = embed.lookup(table, ids)
    side = _randn(1, stream.shape, torch.bfloat16)

    def block(stream, side, norm, up, gate, down):
        y, s = norms.rms_norm(side, norm, stream, eps=1e-5)
        return linear.project(linear.project(y, gate, activation="silu", times=linear.project(y, up)), down, residual=s)

    def plain(stream, side, norm, up, gate, down):
        s = side + stream
        y = s * (s.square().mean(1, keepdim=True) + 1e-5).rsqrt() * norm
        return (act("silu", y @ gate.t())[0] * (y @ up.t())) @ down.t() + s

    leaves = [v.detach().clone().requires_grad_(True) for v in (stream, side, norm, up, gate, down)]
    wide = [v.detach().double().requires_grad_(True) for v in leaves]
    got, want = block(*leaves), plain(*wide)
    dy = _randn(2, got.shape, torch.bfloat16)
    # six roundings to 16 bits between the ends, each of half a step, and what they do on their way: under sixteen of them in the 2-norm
    off = lambda a, b: float((a.detach().double() - b.detach()).norm() / b.detach().norm())                      # noqa: E731
    assert off(got, want) < 16 * 2 ** -8
    for a, b in zip(torch.autograd.grad(got, leaves, dy), torch.autograd.grad(want, wide, dy.double())):
        assert off(a, b) < 16 * 2 ** -8
    with torch.no_grad():
        q, scale, s = norms.rms_norm_8bit(side, norm, stream, eps=1e-5)
        (gq, gs), (uq, us), (dq, ds) = (norms.to_8bit(v) for v in (gate, up, down))
        h, hs = norms.to_8bit(linear.project_8bit(q, scale, gq, gs, activation="silu", times=linear.project_8bit(q, scale, uq, us)))
        # four tensors of 8 bits, half a step of 2^-4 each
        assert off(linear.project_8bit(h, hs, dq, ds, residual=s), want) < 4 * 2 ** -4
        # two experts, this layer's and a smaller one of the same shapes; every token goes to both
        both = lambda v: torch.stack((v, v * 0.5))                                     # noqa: E731
        order, offsets = ex.sort(torch.tensor([[0, 1]] * len(ids), device="cuda"), 2)
        y, s = norms.rms_norm(side, norm, stream, eps=1e-5)
        rows = embed.lookup(y, order // 2)
        rows = ex.project(ex.project(rows, both(gate), offsets, activation="silu", times=ex.project(rows, both(up), offsets)), both(down), offsets)
        back = torch.empty_like(order).scatter_(0, order.long(), torch.arange(order.numel(), dtype=torch.int32, device="cuda"))
        one = linear.project(linear.project(y, gate, activation="silu", times=linear.project(y, up)), down)
        # (the same products, rounded at the same places; their sums may have another order)
        assert off(embed.lookup(rows, back.reshape(-1, 2))[:, 0], one.double()) < 2 * 2 ** -8
