"""Operators on a checkpoint's tensors against their definitions in 64 bits.

Tolerances, per element: half a step of the result's type (u * |exact|), and what sums in 32 bits can lose: a sum of n terms
is off by at most n * 2^-23 times the sum of the terms' magnitudes (tensor cores cut where an addition would round).  The
thin products h = s x A^T and g = s dy B are kept in 16 bits at least (an error of 2^-16 of their magnitude, for F16 also
2^-24 absolutely, the step of its smallest numbers), which the second product carries on.
"""
import math

import numpy as np
import pytest
import torch

pytestmark = pytest.mark.gpu

DTYPES = [torch.bfloat16, torch.float16]
ALL = DTYPES + [torch.float32]


@pytest.fixture(autouse=True)
def _library(gpu):
    return gpu


def _u(dtype):
    return torch.finfo(dtype).eps / 2


def _randn(seed, shape, dtype, std=1.0):
    g = torch.Generator(device="cuda")
    g.manual_seed(seed)
    return (torch.randn(shape, generator=g, device="cuda") * std).to(dtype)


def _ids(seed, n, rows, dtype=torch.int64, shape=None):
    rng = np.random.default_rng(seed)
    v = torch.from_numpy(rng.integers(0, rows, n)).to(dtype).cuda()
    return v if shape is None else v.reshape(shape)


def _bits(t):
    return t.contiguous().view({2: torch.int16, 4: torch.int32}[t.element_size()])


# ------------------------------------------------------------------------------------------- rows

@pytest.mark.parametrize("dtype", ALL)
@pytest.mark.parametrize("rows, dim, n", [(1, 1, 1), (10, 8, 1), (10, 7, 5), (997, 250, 3001), (300, 4096, 64), (5, 1024, 333), (100, 33, 4096), (50, 6000, 9)])
def test_rows(dtype, rows, dim, n):
    from lmz_b200 import embed
    table, ids = _randn(1, (rows, dim), dtype), _ids(2, n, rows)
    assert torch.equal(_bits(embed.lookup(table, ids)), _bits(table[ids]))
    scale = math.sqrt(dim) * 0.7
    want = table.double()[ids] * float(np.float32(scale))
    got = embed.lookup(table, ids.to(torch.int32), scale=scale)
    # one product in 32 bits, one rounding
    assert ((got.double() - want).abs() <= (_u(dtype) + 2 ** -23) * want.abs() + torch.finfo(dtype).smallest_normal * torch.finfo(dtype).eps).all()


def test_rows_keep_every_bit_and_pad_with_zeros():
    from lmz_b200 import embed
    every = torch.arange(-32768, 32768, dtype=torch.int32).to(torch.int16).cuda().view(torch.bfloat16).reshape(64, 1024)
    ids = torch.tensor([[0, -1, 63], [64, 5, -2 ** 40], [2 ** 40, 63, 1]], device="cuda")
    got = embed.lookup(every, ids)
    inside = (ids >= 0) & (ids < 64)
    want = torch.where(inside[..., None], _bits(every)[ids.clamp(0, 63)], torch.zeros((), dtype=torch.int16, device="cuda"))
    assert got.shape == (3, 3, 1024) and torch.equal(_bits(got), want)
    got = embed.lookup(every, ids, scale=2.0)
    assert (_bits(got)[~inside] == 0).all()


@pytest.mark.parametrize("dtype", ALL)
@pytest.mark.parametrize("offset, stride", [(0, 264), (1, 257), (2, 258), (4, 260), (0, 256)])
def test_rows_of_any_stride_and_alignment(dtype, offset, stride):
    from lmz_b200 import embed
    block = _randn(3, (40 * stride + 8,), dtype)
    table = block[offset:].as_strided((40, 256), (stride, 1))
    ids = _ids(4, 100, 40).reshape(4, 25).t()              # (ids that do not follow each other either)
    assert torch.equal(_bits(embed.lookup(table, ids)), _bits(table[ids]))
    one = table[3:4].expand(7, 256)                        # rows that are one
    assert torch.equal(_bits(embed.lookup(one, _ids(5, 9, 7))), _bits(table[3:4].expand(9, 256)))


def test_rows_beyond_32_bits():
    from lmz_b200 import embed
    rows, dim = 140_000, 16_384                            # 4.6 GB
    table = torch.empty((rows, dim), dtype=torch.bfloat16, device="cuda")
    ids = torch.tensor([0, rows - 1, 131_072, 131_071, 70_000], device="cuda")
    table[ids] = _randn(6, (5, dim), torch.bfloat16)
    assert torch.equal(embed.lookup(table, ids), table[ids])
    y = embed.lookup(table, ids.repeat(30_000)[:140_001])  # (and a result beyond them)
    assert torch.equal(y[-3:], table[ids.repeat(30_000)[139_998:140_001]])


def _rows_grad(table_shape, ids, dy, scale):
    want = torch.zeros(table_shape, dtype=torch.float64, device="cuda")
    size = torch.zeros(table_shape, dtype=torch.float64, device="cuda")
    inside = ((ids >= 0) & (ids < table_shape[0])).flatten()
    flat, d = ids.flatten()[inside].long(), dy.reshape(-1, dy.shape[-1])[inside].double()
    want.index_add_(0, flat, d)
    size.index_add_(0, flat, d.abs())
    most = int(torch.bincount(flat, minlength=1).max()) if flat.numel() else 0
    scale = float(np.float32(scale))
    return want * scale, size * abs(scale), most


@pytest.mark.parametrize("dtype", ALL)
@pytest.mark.parametrize("rows, dim, n, how", [(1, 1, 1, "any"), (10, 8, 0, "any"), (10, 7, 5, "any"), (997, 250, 3001, "any"), (300, 4096, 64, "any"),
                                               (3, 264, 5000, "any"), (70_000, 40, 4097, "any"), (50, 2056, 2500, "one"), (20, 64, 33, "one"), (20, 64, 32, "one"),
                                               (300, 96, 20_000, "few"), (1000, 48, 9000, "padded"), (20, 6000, 200, "few"), (256, 24, 3000, "any"), (255, 24, 3000, "any")])
def test_rows_gradient(dtype, rows, dim, n, how):
    from lmz_b200 import embed
    ids = _ids(7, n, rows)
    if how == "one":
        ids[:] = rows - 1
    elif how == "few":
        ids = torch.where(_ids(8, n, 10) < 6, ids % 3, ids)
    elif how == "padded":
        ids = torch.where(_ids(8, n, 10) < 6, _ids(9, n, 3) * 2000 - 2000, ids)           # -2000, 0 and 2000
    table, dy = _randn(10, (rows, dim), dtype).requires_grad_(True), _randn(11, (n, dim), dtype)
    scale = 0.37
    (got,) = torch.autograd.grad(embed.lookup(table, ids, scale=scale), table, dy)
    want, size, most = _rows_grad((rows, dim), ids, dy, scale)
    assert got.dtype == dtype and got.shape == table.shape and got.is_contiguous()
    assert ((got.double() - want).abs() <= _u(dtype) * want.abs() + (most + 1) * 2 ** -23 * size + torch.finfo(dtype).smallest_normal * torch.finfo(dtype).eps).all()
    assert (got[torch.bincount(ids.clamp(0, rows - 1), minlength=rows) == 0] == 0).all()
    (again,) = torch.autograd.grad(embed.lookup(table, ids, scale=scale), table, dy)
    assert torch.equal(_bits(got), _bits(again))


def test_rows_gradient_of_many_tokens():
    """A quarter of a million tokens, half of them padding with one id: windows of more than 32 tokens."""
    from lmz_b200 import embed
    n, rows, dim = 250_001, 5000, 64
    ids = torch.where(_ids(12, n, 2) == 0, torch.zeros((), dtype=torch.int64, device="cuda"), _ids(13, n, rows)).to(torch.int32)
    table, dy = _randn(14, (rows, dim), torch.float32).requires_grad_(True), _randn(15, (n, dim), torch.float32)
    (got,) = torch.autograd.grad(embed.lookup(table, ids), table, dy)
    want, size, most = _rows_grad((rows, dim), ids, dy, 1.0)
    # sums of sums: no term goes through more additions than a window's and the windows'
    steps = 2 * math.ceil(math.sqrt(n)) + 4096
    assert ((got.double() - want).abs() <= 2 ** -24 * want.abs() + steps * 2 ** -24 * size).all()


def test_rows_gradient_takes_any_upstream_gradient():
    """A sum's gradient is one number expanded: no memory of its own; and differences, exact for a linear map."""
    from lmz_b200 import embed
    table, ids = _randn(16, (30, 16), torch.float32).requires_grad_(True), _ids(17, 50, 30)
    (g,) = torch.autograd.grad(embed.lookup(table, ids).sum(), table)
    assert torch.equal(g, torch.bincount(ids, minlength=30)[:, None].expand(30, 16).float())
    t = torch.randint(-8, 8, (30, 16), device="cuda").float().requires_grad_(True)
    w = torch.randint(-8, 8, (50, 16), device="cuda").float()
    (g,) = torch.autograd.grad((embed.lookup(t, ids, scale=2.0) * w).sum(), t)
    for at in ((0, 0), (7, 3), (29, 15)):
        up, down = t.detach().clone(), t.detach().clone()
        up[at] += 1
        down[at] -= 1
        diff = ((embed.lookup(up, ids, scale=2.0) * w).sum() - (embed.lookup(down, ids, scale=2.0) * w).sum()) / 2
        assert float(diff) == float(g[at])
    dy = _randn(18, (16, 50), torch.float32).t()           # columns that are rows
    (g,) = torch.autograd.grad(embed.lookup(table, ids), table, dy)
    (h,) = torch.autograd.grad(embed.lookup(table, ids), table, dy.contiguous())
    assert torch.equal(g, h)


def test_rows_refusals():
    from lmz_b200 import embed
    t, i = torch.zeros((4, 8), device="cuda"), torch.zeros(3, dtype=torch.int64, device="cuda")
    for args, kind in (((t[0], i), ValueError), ((t.double(), i), TypeError), ((t, i.float()), TypeError), ((t, i.to(torch.int16)), TypeError),
                       ((t.t(), i), ValueError), ((t, i.cpu()), ValueError), ((t, i, math.nan), ValueError), ((t, [0, 1]), TypeError)):
        with pytest.raises(kind):
            embed.lookup(*args)
    assert embed.lookup(t, i[:0]).shape == (0, 8) and embed.lookup(t[:, :0], i).shape == (3, 0)
    assert (embed.lookup(t[:0], i) == 0).all()


# ------------------------------------------------------------------------------------------- projections

def _index(kind, tokens, n, seed=20):
    rng = np.random.default_rng(seed)
    if kind == "none":
        return None
    if kind == "mixed":
        v = rng.integers(-1, n, tokens)
    elif kind == "short":                                  # many runs in every tile
        v = np.repeat(rng.integers(0, n, tokens // 32 + 1), 32)[:tokens]
    elif kind == "off":
        v = np.full(tokens, -1)
    elif kind == "far":                                    # outside on both sides
        v = rng.integers(-3, n + 3, tokens)
    else:                                                  # runs
        cuts = np.sort(rng.integers(0, tokens + 1, 5))
        v = np.repeat(rng.integers(-1, n, 6), np.diff(np.concatenate(([0], cuts, [tokens]))))
    return torch.from_numpy(v.astype(np.int32)).cuda()


def _inputs(tokens, inp, out, rank, n, dtype, seed=30):
    x, w = _randn(seed, (tokens, inp), dtype), _randn(seed + 1, (out, inp), dtype, 0.05)
    a, b = _randn(seed + 2, (n, rank, inp), dtype, inp ** -0.5), _randn(seed + 3, (n, out, rank), dtype, 0.3)
    scales = 0.5 + torch.rand(n, generator=torch.Generator(device="cuda").manual_seed(seed + 4), device="cuda")
    return x, w, a, b, scales


def _rows_of(index, tokens, i):
    return torch.arange(tokens, device="cuda") if index is None and i == 0 else torch.nonzero(index == i).flatten() if index is not None else \
        torch.zeros(0, dtype=torch.int64, device="cuda")


def _carried(t, up, dtype):
    """What thin products kept in 16 bits cost: |t| 2^-16 (and F16's smallest step) times the second factor."""
    return (t.abs() * 2 ** -16 + (2 ** -24 if dtype == torch.float16 else 0)) @ up.abs()


def _check(got, want, size, carried, terms, what):
    u = _u(got.dtype)
    least = torch.finfo(got.dtype).smallest_normal * torch.finfo(got.dtype).eps
    bound = u * want.abs() + (1 + u) * (terms * 2 ** -23 * size + carried) + least
    off = (got.double() - want).abs()
    assert torch.isfinite(got).all(), what
    worst = (off / bound).max()
    assert worst <= 1, f"{what}: {float(worst)} of its bound at {int((off / bound).argmax())}"


def _check_project(x, w, a, b, scales, index, y, dy=None, grads=None):
    """Results against the definition in 64 bits, adapter by adapter."""
    dtype, tokens = x.dtype, x.shape[0]
    xd, wd, ad, bd = (t.detach().double() for t in (x, w, a, b))
    want, size = xd @ wd.t(), xd.abs() @ wd.abs().t()
    carried = torch.zeros_like(want)
    (n, rank, inp), out = a.shape, b.shape[1]
    eye = torch.eye(rank, dtype=torch.float64, device="cuda")
    if dy is not None:
        dyd = dy.double()
        dx, dxs, dxc = dyd @ wd, dyd.abs() @ wd.abs(), torch.zeros_like(xd)
        da, das, dac = (torch.zeros_like(ad) for _ in range(3))
        db, dbs, dbc = (torch.zeros_like(bd) for _ in range(3))
    for i in range(n):
        at, s = _rows_of(index, tokens, i), float(scales[i])
        if not at.numel():
            continue
        h = s * (xd[at] @ ad[i].t())
        hs = s * (xd[at].abs() @ ad[i].abs().t())
        want[at] += h @ bd[i].t()
        size[at] += hs @ bd[i].abs().t()
        carried[at] = _carried(h, bd[i].t(), dtype)
        if dy is not None:
            g = s * (dyd[at] @ bd[i])
            gs = s * (dyd[at].abs() @ bd[i].abs())
            dx[at] += g @ ad[i]
            dxs[at] += gs @ ad[i].abs()
            dxc[at] = _carried(g, ad[i], dtype)
            da[i], das[i], dac[i] = g.t() @ xd[at], gs.t() @ xd[at].abs(), _carried(g, eye, dtype).t() @ xd[at].abs()
            db[i], dbs[i], dbc[i] = dyd[at].t() @ h, dyd[at].abs().t() @ hs, dyd[at].abs().t() @ _carried(h, eye, dtype)
    _check(y, want, size, carried, inp + rank + 8, "y")
    if dy is not None:
        _check(grads[0], dx, dxs, dxc, out + rank + 8, "dx")
        _check(grads[1], da, das, dac, tokens + out + 8, "da")
        _check(grads[2], db, dbs, dbc, tokens + inp + 8, "db")


SHAPES = [
    # tokens, in, out, rank, adapters, index
    (1, 64, 64, 16, 1, "none"), (1, 256, 192, 8, 4, "runs"), (2, 64, 130, 1, 3, "mixed"), (7, 136, 264, 4, 2, "mixed"), (16, 512, 128, 16, 3, "runs"),
    (17, 72, 200, 64, 5, "mixed"), (33, 1024, 384, 24, 6, "runs"), (64, 320, 640, 16, 48, "mixed"), (100, 128, 96, 128, 3, "mixed"),
    (129, 200, 264, 256, 2, "runs"), (255, 192, 520, 32, 9, "runs"), (300, 448, 128, 16, 1, "none"), (513, 256, 512, 40, 4, "runs"),
    (640, 128, 1032, 16, 70, "mixed"), (1000, 512, 256, 64, 2, "runs"), (257, 128, 256, 16, 3, "off"), (40, 128, 256, 16, 3, "far"), (1500, 64, 136, 8, 7, "far"),
    # more tiles than multiprocessors, more steps than a ring has stages, more runs than that too
    (2600, 64, 2200, 16, 5, "runs"), (2600, 648, 2056, 40, 30, "short"), (4700, 1400, 1288, 8, 3, "runs"), (900, 1032, 5000, 100, 12, "short"),
    (2300, 776, 2200, 16, 40, "mixed"), (200, 2048, 264, 64, 6, "short"),
    (4000, 200, 640, 16, 5, "runs"), (4100, 328, 600, 24, 9, "short"), (2000, 136, 6000, 16, 30, "mixed"), (9000, 256, 1400, 32, 3, "runs"),
    (1500, 777, 501, 100, 6, "mixed"), (5000, 1032, 1000, 16, 9, "far"), (700, 1100, 1200, 128, 20, "mixed"), (300, 1000, 2000, 256, 2, "mixed"),
    # sizes where rows do not start on a boundary
    (5, 1, 1, 1, 1, "none"), (9, 33, 65, 3, 2, "mixed"), (333, 777, 501, 5, 5, "runs"), (70, 250, 1001, 7, 4, "mixed"), (600, 100, 77, 12, 3, "runs"),
]


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("tokens, inp, out, rank, n, kind", SHAPES)
def test_project_and_its_gradients(dtype, tokens, inp, out, rank, n, kind):
    from lmz_b200 import adapters
    x, w, a, b, scales = _inputs(tokens, inp, out, rank, n, dtype)
    index = _index(kind, tokens, n)
    with torch.no_grad():
        y = adapters.project(x, w, a, b, index, scale=scales)
    dy = _randn(40, (tokens, out), dtype)
    for t in (x, a, b):
        t.requires_grad_(True)
    z = adapters.project(x, w, a, b, index, scale=scales)
    assert torch.equal(_bits(z.detach()), _bits(y))
    grads = torch.autograd.grad(z, (x, a, b), dy)
    assert [g.dtype for g in grads] == [dtype] * 3 and [g.shape for g in grads] == [x.shape, a.shape, b.shape]
    _check_project(x, w, a, b, scales, index, y, dy, grads)
    again = torch.autograd.grad(adapters.project(x, w, a, b, index, scale=scales), (x, a, b), dy)
    for g, h in zip(grads, again):
        assert torch.equal(_bits(g), _bits(h))


@pytest.mark.parametrize("tokens", [3, 40, 300, 700])
def test_bad_values_stay_with_their_own_tokens(tokens):
    """Infinities and NaN in one adapter's factors, and in rows of x that belong to nobody, reach nobody else."""
    from lmz_b200 import adapters
    n, bad = 5, 2
    x, w, a, b, scales = _inputs(tokens, 256, 264, 16, n, torch.bfloat16)
    index = _index("runs" if tokens > 100 else "mixed", tokens, n)
    index[0], index[tokens // 2:tokens // 2 + 1 + tokens // 50] = bad, -1
    index[-1] = 1
    dy = _randn(41, (tokens, 264), torch.bfloat16)
    good = adapters.project(x, w, a, b, index, scale=scales)
    want = torch.autograd.grad(adapters.project(x.requires_grad_(True), w, a.requires_grad_(True), b.requires_grad_(True), index, scale=scales), (x, a, b), dy)
    x, a, b, dy = x.detach().clone(), a.detach().clone(), b.detach().clone(), dy.clone()
    a[bad], b[bad] = math.inf, math.nan
    x[index == -1] = math.nan
    dy[index == -1] = math.inf
    others = (index != bad) & (index != -1)
    y = adapters.project(x, w, a, b, index, scale=scales)
    assert torch.equal(y[others], good[others])
    assert torch.isnan(y[index == bad]).all() and torch.isnan(y[index == -1]).all()
    got = torch.autograd.grad(adapters.project(x.requires_grad_(True), w, a.requires_grad_(True), b.requires_grad_(True), index, scale=scales), (x, a, b), dy)
    assert torch.equal(got[0][others], want[0][others])
    keep = [i for i in range(n) if i != bad]
    assert torch.equal(got[1][keep], want[1][keep]) and torch.equal(got[2][keep], want[2][keep])


@pytest.mark.parametrize("tokens, inp, out, rank, n", [(130, 256, 512, 16, 5), (300, 1024, 2056, 8, 9), (700, 264, 1288, 24, 12), (2500, 512, 4104, 72, 7),
                                                       (1100, 320, 1096, 16, 200)])
def test_bad_values_among_tokens_in_any_order(tokens, inp, out, rank, n):
    """The same where every sixteen tokens have several adapters, in tiles of a few adapters and of very many."""
    from lmz_b200 import adapters
    x, w, a, b, scales = _inputs(tokens, inp, out, rank, n, torch.bfloat16)
    index, dy = _index("mixed", tokens, n), _randn(41, (tokens, out), torch.bfloat16)
    index[:3] = torch.tensor([1, -1, 3])

    def both():
        leaves = [t.detach().clone().requires_grad_(True) for t in (x, a, b)]
        y = adapters.project(leaves[0], w, leaves[1], leaves[2], index, scale=scales)
        return y.detach(), torch.autograd.grad(y, leaves, dy)

    good, want = both()
    _check_project(x, w, a, b, scales, index, good, dy, want)
    a[1, -1, -1], b[1, 0, 0], a[3, 0, 0], b[3, -1, -1] = math.nan, math.inf, -math.inf, math.nan
    x[index == -1] = math.nan
    dy[index == -1] = math.inf
    others = (index != 1) & (index != 3) & (index != -1)
    y, got = both()
    assert torch.equal(y[others], good[others]) and torch.equal(got[0][others], want[0][others])
    for i in (1, 3):
        assert torch.isnan(y[index == i]).any() and torch.isnan(got[0][index == i]).any()
    keep = [i for i in range(n) if i not in (1, 3)]
    assert torch.equal(got[1][keep], want[1][keep]) and torch.equal(got[2][keep], want[2][keep])
    # a row of x with infinities is its own token's alone
    x, w, a, b, scales = _inputs(tokens, inp, out, rank, n, torch.bfloat16)
    dy = _randn(41, (tokens, out), torch.bfloat16)
    x[0], dy[0] = math.inf, math.nan
    y, got = both()
    assert torch.equal(y[1:], good[1:]) and torch.equal(got[0][1:], want[0][1:])


def test_one_adapter_without_a_stack():
    from lmz_b200 import adapters
    x, w, a, b, _ = _inputs(20, 64, 96, 8, 1, torch.bfloat16)
    want = adapters.project(x, w, a, b, scale=0.5)
    got = adapters.project(x.reshape(4, 5, 64), w, a[0], b[0], scale=0.5)
    assert torch.equal(got.reshape(20, 96), want)
    zeros = torch.zeros((4, 5), dtype=torch.int64, device="cuda")
    assert torch.equal(adapters.project(x.reshape(4, 5, 64), w, a, b, zeros, scale=torch.tensor([0.5], device="cuda")), got)
    a1, b1 = a[0].clone().requires_grad_(True), b[0].clone().requires_grad_(True)
    da, db = torch.autograd.grad(adapters.project(x, w, a1, b1, scale=0.5).float().sum(), (a1, b1))
    assert da.shape == a1.shape and db.shape == b1.shape


@pytest.mark.parametrize("tokens", [3, 300])
@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("offset, pad", [(4, 0), (1, 0), (0, 1), (4, 4), (0, 8), (3, 5)])
def test_project_of_any_stride_and_alignment(dtype, offset, pad, tokens):
    """Weights where an archive put them: on a boundary of 8 bytes, of 2, and as a part of a wider tensor; x likewise."""
    from lmz_b200 import adapters
    x, w, a, b, scales = _inputs(tokens, 256, 136, 16, 3, dtype)
    index = _index("mixed", tokens, 3).long()

    def elsewhere(t):
        rows, cols = t.shape
        block = torch.full((rows * (cols + pad) + offset + 16,), math.nan, dtype=dtype, device="cuda")
        view = block[offset:].as_strided((rows, cols), (cols + pad, 1))
        view.copy_(t)
        return view

    want = adapters.project(x, w, a, b, index, scale=scales)
    dy = _randn(42, (tokens, 136), dtype)
    want_grads = torch.autograd.grad(adapters.project(x.requires_grad_(True), w, a.requires_grad_(True), b.requires_grad_(True), index, scale=scales), (x, a, b), dy)
    x2, w2 = elsewhere(x.detach()), elsewhere(w)
    a2, b2 = elsewhere(a.detach().reshape(-1, 256)).reshape(a.shape), elsewhere(b.detach().reshape(-1, 16)).reshape(b.shape)
    assert torch.equal(adapters.project(x2, w2, a2, b2, index, scale=scales), want)
    got = torch.autograd.grad(adapters.project(x2.requires_grad_(True), w2, a2.requires_grad_(True), b2.requires_grad_(True), index, scale=scales), (x2, a2, b2), dy)
    for g, h in zip(got, want_grads):
        assert torch.equal(g, h)


def test_project_gradients_by_differences():
    """Whole numbers small enough that every product and sum is exact in BF16: differences of the linear parts are too."""
    from lmz_b200 import adapters
    g = torch.Generator(device="cuda").manual_seed(5)
    small = lambda *s: torch.randint(-1, 2, s, generator=g, device="cuda").to(torch.bfloat16)      # noqa: E731
    x, w, a, b = small(6, 8), small(8, 8), small(2, 2, 8), small(2, 8, 2)
    index = torch.tensor([0, 1, 1, -1, 0, 1], device="cuda")
    dy = small(6, 8)
    args = [x, a, b]
    loss = lambda x, a, b: (adapters.project(x, w, a, b, index, scale=2.0).double() * dy.double()).sum()      # noqa: E731
    leaves = [t.clone().requires_grad_(True) for t in args]
    grads = torch.autograd.grad(adapters.project(leaves[0], w, leaves[1], leaves[2], index, scale=2.0), leaves, dy)
    for k, t in enumerate(args):
        for at in ((0,) * t.dim(), tuple(n - 1 for n in t.shape), tuple(n // 2 for n in t.shape)):
            sides = []
            for d in (1, -1):
                moved = [v.clone() for v in args]
                moved[k][at] += d
                sides.append(float(loss(*moved)))
            assert (sides[0] - sides[1]) / 2 == float(grads[k][at])


def test_only_the_gradients_asked_for():
    from lmz_b200 import adapters
    x, w, a, b, scales = _inputs(50, 64, 64, 8, 3, torch.bfloat16)
    index, dy = _index("mixed", 50, 3), _randn(43, (50, 64), torch.bfloat16)
    full = torch.autograd.grad(adapters.project(x.requires_grad_(True), w, a.requires_grad_(True), b.requires_grad_(True), index, scale=scales), (x, a, b), dy)
    for k in range(3):
        args = [t.detach().clone().requires_grad_(i == k) for i, t in enumerate((x, a, b))]
        (g,) = torch.autograd.grad(adapters.project(args[0], w, args[1], args[2], index, scale=scales), args[k], dy)
        assert torch.equal(g, full[k])


def test_only_the_gradients_asked_for_of_tokens_in_any_order():
    """(How many CTAs share a factor's tokens, and so the order of its sums in 32 bits, goes by how many factors are wanted:
    within the bounds of the definition, not bit for bit.)"""
    from lmz_b200 import adapters
    x, w, a, b, scales = _inputs(1500, 392, 400, 128, 5, torch.bfloat16)
    index, dy = _index("mixed", 1500, 5), _randn(43, (1500, 400), torch.bfloat16)

    def grads(which):
        leaves = [t.detach().requires_grad_(i in which) for i, t in enumerate((x, a, b))]
        y = adapters.project(leaves[0], w, leaves[1], leaves[2], index, scale=scales)
        return y.detach(), torch.autograd.grad(y, [leaves[i] for i in which], dy)

    y, every = grads((0, 1, 2))
    for which in ((0,), (1,), (2,), (0, 1), (1, 2)):
        got = list(every)
        for i, g in zip(which, grads(which)[1]):
            got[i] = g
        _check_project(x, w, a, b, scales, index, y, dy, got)


def test_no_tokens():
    from lmz_b200 import adapters
    x, w, a, b, scales = _inputs(0, 64, 96, 8, 3, torch.bfloat16)
    index = torch.zeros(0, dtype=torch.int32, device="cuda")
    for t in (x, a, b):
        t.requires_grad_(True)
    y = adapters.project(x, w, a, b, index, scale=scales)
    assert y.shape == (0, 96)
    dx, da, db = torch.autograd.grad(y, (x, a, b), torch.zeros_like(y))
    assert dx.shape == (0, 64) and (da == 0).all() and (db == 0).all() and da.shape == a.shape and db.shape == b.shape


def test_project_refusals():
    from lmz_b200 import adapters
    x, w, a, b, scales = _inputs(6, 64, 96, 8, 3, torch.bfloat16)
    index = torch.zeros(6, dtype=torch.int32, device="cuda")
    big = torch.zeros((1, 257, 64), dtype=torch.bfloat16, device="cuda"), torch.zeros((1, 96, 257), dtype=torch.bfloat16, device="cuda")
    for args, kw, kind in (((x.float(), w, a, b), {}, TypeError), ((x, w.half(), a, b), {}, TypeError), ((x, w, a.float(), b), {}, TypeError),
                           ((x[:, :32], w, a, b), {}, ValueError), ((x, w.t(), a, b), {}, ValueError), ((x, w, a[0], b), {}, ValueError),
                           ((x, w, a[:2], b), {}, ValueError), ((x, w, a[:, :4], b), {}, ValueError), ((x, w, *big), {}, ValueError),
                           ((x, w, a[:0], b[:0]), {}, ValueError), ((x, w, a, b, index[:5]), {}, ValueError), ((x, w, a, b, index.float()), {}, TypeError),
                           ((x, w, a, b, index.cpu()), {}, ValueError), ((x, w, a, b, index), dict(scale=scales[:2]), ValueError),
                           ((x, w, a, b, index), dict(scale=scales.double()), ValueError), ((x, w, a, b, index), dict(scale=math.inf), ValueError),
                           ((x, w.clone().requires_grad_(True), a, b), {}, ValueError),
                           ((x, w, a, b, index), dict(scale=scales.clone().requires_grad_(True)), ValueError)):
        with pytest.raises(kind):
            adapters.project(*args, **kw)
    wide = torch.zeros((96, 128), dtype=torch.bfloat16, device="cuda")
    with pytest.raises(ValueError, match="next to each other"):
        adapters.project(x, wide[:, ::2], a, b)


# ------------------------------------------------------------------------------------------- merges

@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("out, inp, rank", [(1, 1, 1), (8, 8, 8), (130, 264, 16), (1000, 771, 5), (256, 1024, 64), (129, 512, 256), (70, 2000, 100), (66_000, 16, 4), (3000, 2600, 8), (2900, 1900, 72), (5000, 1032, 200), (2500, 1001, 33)])
def test_merge(dtype, out, inp, rank):
    from lmz_b200 import adapters
    w, a, b = _randn(50, (out, inp), dtype), _randn(51, (rank, inp), dtype, inp ** -0.5), _randn(52, (out, rank), dtype)
    scale = 1.7
    s = float(np.float32(scale))
    want = w.double() + s * (b.double() @ a.double())
    size = w.double().abs() + s * (b.double().abs() @ a.double().abs())
    got = adapters.merge(w, a, b, scale=scale)
    zero = torch.zeros_like(want)
    _check(got, want, size, zero, rank + 4, "merge")
    wide = torch.full((out, inp + 3), math.nan, dtype=dtype, device="cuda")
    wide[:, 1:inp + 1] = w
    assert torch.equal(adapters.merge(wide[:, 1:inp + 1], a, b, scale=scale), got)
    assert torch.equal(adapters.merge(wide[:, 1:inp + 1], a, b, scale=scale, out=torch.empty_like(w)), got)
    assert adapters.merge(w, a, b, scale=scale, out=w) is w and torch.equal(w, got)


def test_merge_refusals():
    from lmz_b200 import adapters
    w, a, b = _randn(50, (16, 24), torch.bfloat16), _randn(51, (4, 24), torch.bfloat16), _randn(52, (16, 4), torch.bfloat16)
    for args, kw, kind in (((w.float(), a, b), {}, TypeError), ((w, a.half(), b), {}, TypeError), ((w, a, b.t()), {}, ValueError), ((w.t(), a, b), {}, ValueError),
                           ((w, a[:3], b), {}, ValueError), ((w, a[:0], b[:, :0]), {}, ValueError), ((w, a, b, math.nan), {}, ValueError),
                           ((w, a, b), dict(out=w.t()), ValueError), ((w, a, b), dict(out=w.half()), ValueError), ((w, a.clone().requires_grad_(True), b), {}, ValueError)):
        with pytest.raises(kind):
            adapters.merge(*args, **kw)
    block = torch.zeros(16 * 24 + 24, dtype=torch.bfloat16, device="cuda")
    one, other = block[:384].view(16, 24), block[24:].view(16, 24)
    with pytest.raises(ValueError, match="overlap"):
        adapters.merge(one, a, b, out=other)
    assert adapters.merge(w[:0], a, b[:0]).shape == (0, 24)


# ------------------------------------------------------------------------------------------- streams, graphs

def test_on_a_stream_of_its_own_and_captured():
    """Each operator on a side stream, then captured: replays take what the inputs hold by then, and two graphs whose
    replays overlap do not disturb each other."""
    from lmz_b200 import adapters, embed
    x, w, a, b, scales = _inputs(300, 256, 136, 16, 3, torch.bfloat16)
    table, ids, index = _randn(60, (500, 256), torch.bfloat16), _ids(61, 300, 500), _index("runs", 300, 3)
    dy = _randn(62, (300, 136), torch.bfloat16)

    def step():
        t, p, q = table.detach().requires_grad_(True), a.detach().requires_grad_(True), b.detach().requires_grad_(True)
        e = embed.lookup(t, ids, scale=3.0)
        y = adapters.project(e, w, p, q, index, scale=scales)
        return (y, *torch.autograd.grad(y, (t, p, q), dy), adapters.merge(w, a[0], b[0], scale=0.5))

    want = step()
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        got = step()
    side.synchronize()
    for g, v in zip(got, want):
        assert torch.equal(g, v)
    graphs, outs = [], []
    for _ in range(2):
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            outs.append(step())
        graphs.append(graph)
    ids.copy_(_ids(63, 300, 500))
    table.mul_(2)
    index.copy_(_index("mixed", 300, 3))
    want = step()
    torch.cuda.synchronize()
    other = torch.cuda.Stream()
    for _ in range(3):
        with torch.cuda.stream(side):
            graphs[0].replay()
        with torch.cuda.stream(other):
            graphs[1].replay()
    torch.cuda.synchronize()
    for out in outs:
        for g, v in zip(out, want):
            assert torch.equal(g, v)


def test_captured_for_any_order_of_the_tokens():
    """One graph for tokens in runs and in any order: which it is shows only on the device."""
    from lmz_b200 import adapters
    x, w, a, b, scales = _inputs(1500, 392, 400, 128, 6, torch.bfloat16)
    dy, index = _randn(62, (1500, 400), torch.bfloat16), _index("runs", 1500, 6).long()

    def step():
        leaves = [t.detach().requires_grad_(True) for t in (x, a, b)]
        y = adapters.project(*leaves[:1], w, *leaves[1:], index, scale=scales)
        return (y.detach(), *torch.autograd.grad(y, leaves, dy))

    step()
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = step()
    for kind in ("mixed", "runs", "far", "off"):
        index.copy_(_index(kind, 1500, 6, seed=64))
        for t in out:
            t.fill_(7)
        graph.replay()
        torch.cuda.synchronize()
        for g, v in zip(out, step()):
            assert torch.equal(g, v)
        _check_project(x, w, a, b, scales, index, out[0], dy, out[1:])


def test_captured_behind_copies_and_from_other_streams():
    """What stands in front of an operator in a graph may be a copy, or work of another stream that it waits for."""
    from lmz_b200 import adapters, embed
    x, w, a, b, scales = _inputs(40, 256, 136, 16, 3, torch.bfloat16)
    table, ids, index = _randn(60, (500, 256), torch.bfloat16), _ids(61, 40, 500), _index("runs", 40, 3)
    mine, weight, out = torch.empty_like(table), torch.empty_like(w), torch.empty_like(w)

    def step():
        mine.copy_(table)
        e = embed.lookup(mine, ids, scale=3.0)
        other.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(other):
            weight.copy_(w)
            merged = adapters.merge(weight, a[0], b[0], scale=0.5)
        torch.cuda.current_stream().wait_stream(other)
        y = adapters.project(e, merged, a, b, index, scale=scales)
        out.copy_(merged)
        return y, adapters.merge(out, a[1], b[1], scale=0.25, out=out)

    other = torch.cuda.Stream()
    want = [t.clone() for t in step()]
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got = step()
    for t in (mine, weight, out, *got):
        t.fill_(7)
    for _ in range(3):
        graph.replay()
    torch.cuda.synchronize()
    for g, v in zip(got, want):
        assert torch.equal(g, v)


def test_no_wait_has_run_out():
    from lmz_b200 import adapters
    x, w, a, b, scales = _inputs(300, 256, 264, 16, 3, torch.bfloat16)
    adapters.project(x, w, a, b, _index("runs", 300, 3), scale=scales)
    adapters.check()
    adapters.check(torch.device("cuda", 0))


def test_inputs_changed_between_the_passes_are_noticed():
    from lmz_b200 import adapters, embed
    x, w, a, b, scales = _inputs(6, 64, 96, 8, 3, torch.bfloat16)
    index = torch.zeros(6, dtype=torch.int32, device="cuda")
    y = adapters.project(x, w, a.requires_grad_(True), b, index, scale=scales)
    index.add_(1)
    with pytest.raises(RuntimeError, match="modified by an inplace operation"):
        y.float().sum().backward()
    table, ids = _randn(60, (5, 8), torch.float32).requires_grad_(True), _ids(61, 3, 5)
    y = embed.lookup(table, ids)
    ids.zero_()
    with pytest.raises(RuntimeError, match="modified by an inplace operation"):
        y.sum().backward()


def test_gradients_have_no_gradient():
    """A graph of the gradients may be asked for (other parts of a loss may need it); going through it is refused."""
    from lmz_b200 import adapters, embed
    table, ids = _randn(60, (5, 8), torch.float32).requires_grad_(True), _ids(61, 3, 5)
    (g,) = torch.autograd.grad(embed.lookup(table, ids).square().sum(), table, create_graph=True)
    want = torch.autograd.grad(embed.lookup(table, ids).square().sum(), table)[0]
    assert torch.equal(g, want)
    with pytest.raises(RuntimeError, match="once_differentiable"):
        g.sum().backward()
    x, w, a, b, scales = _inputs(6, 64, 96, 8, 3, torch.bfloat16)
    (g,) = torch.autograd.grad(adapters.project(x.requires_grad_(True), w, a, b, scale=0.5).float().square().sum(), x, create_graph=True)
    with pytest.raises(RuntimeError, match="once_differentiable"):
        g.float().sum().backward()


# ------------------------------------------------------------------------------------------- with archives

def _safetensors(tensors):
    import json
    import struct
    meta, body, at = {}, b"", 0
    names = {torch.bfloat16: "BF16", torch.float16: "F16", torch.float32: "F32"}
    for name, t in tensors.items():
        raw = t.cpu().contiguous().view(torch.uint8).numpy().tobytes()
        meta[name] = {"dtype": names[t.dtype], "shape": list(t.shape), "data_offsets": [at, at + len(raw)]}
        at += len(raw)
        body += raw
    head = json.dumps(meta).encode()
    head += b" " * (-len(head) % 8)
    return np.frombuffer(struct.pack("<Q", len(head)) + head + body, dtype=np.uint8)


def _archive(tensors, **kw):
    from oracle import archive as oa
    return oa.write_archive([("m.safetensors", _safetensors(tensors))], **kw)


@pytest.mark.parametrize("dtype, dim", [(torch.bfloat16, 250), (torch.bfloat16, 1024), (torch.float32, 100)])
def test_rows_of_an_archive(dtype, dim):
    from lmz_b200 import archive, decode
    rows = 700_000 // dim
    tensors = {"norm": _randn(70, (33,), dtype), "emb": _randn(71, (rows, dim), dtype, 0.02), "head": _randn(72, (50, dim), dtype)}
    ar = archive.Archive(_archive(tensors, mapped=True))
    rng = np.random.default_rng(5)
    for ids in (np.array([0]), np.array([rows - 1]), rng.integers(0, rows, (3, 17)), np.array([5, 5, 6, 7, rows // 2, rows // 2 + 1, 3]), []):
        got = decode.decode_rows(ar, "emb", ids, scale=1.5)
        want = tensors["emb"][torch.as_tensor(np.asarray(ids, dtype=np.int64)).cuda()].float() * 1.5
        assert got.dtype == dtype and torch.equal(got, want.to(dtype))
    part = decode._decode_ranges(ar, [(0, 1)], None, True)[0].plan.chunks.size
    assert part < ar.records.size                          # (only what is needed was decoded)
    for bad, kind in (([rows], IndexError), ([-1], IndexError), ([0.5], TypeError)):
        with pytest.raises(kind):
            decode.decode_rows(ar, "emb", bad)
    with pytest.raises(ValueError):
        decode.decode_rows(ar, "norm", [0])
    with pytest.raises(KeyError):
        decode.decode_rows(ar, "nothing", [0])


def test_a_base_and_its_adapters_from_archives_to_gradients():
    """As they are used together: a base archive and three adapters' archives; embeddings, a projection for a batch of
    requests, its gradients, and a fine-tune restored by merging, saved, and read back."""
    import os
    import tempfile

    from lmz_b200 import adapters, archive, decode, embed, save
    vocab, dim, out, dtype = 600, 256, 384, torch.bfloat16
    base = {"emb.weight": _randn(80, (vocab, dim), dtype, 0.5), "odd": _randn(81, (3,), dtype), "proj.weight": _randn(82, (out, dim), dtype, 0.05)}
    tuned = []
    for i, rank in enumerate((16, 4, 8)):
        tuned.append({f"base_model.proj.lora_A.weight": _randn(83 + i, (rank, dim), dtype, dim ** -0.5),
                      f"base_model.proj.lora_B.weight": _randn(93 + i, (out, rank), dtype, 0.3)})
    ar, parts = archive.Archive(_archive(base)), [archive.Archive(_archive(t)) for t in tuned]
    dec = decode.ArchiveDecoder(ar)
    dec.run()
    dec.check()
    views = {k[1]: v for k, v in dec.tensors().items()}
    a, b = adapters.load(parts, "proj.weight")
    assert a.shape == (3, 16, dim) and b.shape == (3, out, 16) and (a[1, 4:] == 0).all() and (b[2, :, 8:] == 0).all()
    ids, index = _ids(84, 90, vocab), _index("runs", 90, 3)
    scales = torch.tensor([2.0, 0.5, 1.0], device="cuda")
    table = views["emb.weight"].requires_grad_(True)
    a.requires_grad_(True)
    b.requires_grad_(True)
    x = embed.lookup(table, ids, scale=2.0)
    y = adapters.project(x, views["proj.weight"], a, b, index, scale=scales)
    dy = _randn(85, (90, out), dtype)
    dt, dx, da, db = torch.autograd.grad(y, (table, x, a, b), dy)
    _check_project(x.detach(), base["proj.weight"], a, b, scales, index, y.detach(), dy, (dx, da, db))
    want, size, most = _rows_grad((vocab, dim), ids, dx, 2.0)
    assert ((dt.double() - want).abs() <= _u(dtype) * want.abs() + (most + 1) * 2 ** -23 * size).all()
    # the first fine-tune as a checkpoint of its own
    got = decode.decode_tensors(ar, ["proj.weight", "emb.weight"], adapter=parts[0], scale=2.0)
    got = {k[1]: v for k, v in got.items()}
    assert torch.equal(got["emb.weight"], base["emb.weight"])
    assert torch.equal(got["proj.weight"], adapters.merge(base["proj.weight"], tuned[0]["base_model.proj.lora_A.weight"],
                                                          tuned[0]["base_model.proj.lora_B.weight"], scale=2.0))
    path = os.path.join(tempfile.mkdtemp(), "tuned.lmz")
    member = torch.from_numpy(_safetensors(got).copy()).cuda()
    save.save_archive(path, [("m.safetensors", member)])
    back = {k[1]: v for k, v in decode.decode_tensors(path, ["proj.weight", "emb.weight"]).items()}
    assert all(torch.equal(back[k], got[k]) for k in got)


def test_adapters_that_do_not_fit():
    from lmz_b200 import adapters, archive
    one = lambda **t: archive.Archive(_archive({k.replace("__", "."): v for k, v in t.items()}))      # noqa: E731
    a, b = _randn(1, (4, 64), torch.bfloat16), _randn(2, (32, 4), torch.bfloat16)
    good, none = one(p__lora_A__weight=a, p__lora_B__weight=b), one(q__lora_A__weight=a, q__lora_B__weight=b)
    p, q = adapters.load([good, none], "p.weight")
    assert torch.equal(p[0], a) and (p[1] == 0).all() and torch.equal(q[0], b)
    with pytest.raises(KeyError):
        adapters.load([none], "p.weight")
    with pytest.raises(KeyError, match="one factor"):
        adapters.load([one(p__lora_A__weight=a)], "p.weight")
    with pytest.raises(ValueError):
        adapters.load([good, one(p__lora_A__weight=a[:, :32].contiguous(), p__lora_B__weight=b)], "p.weight")
    with pytest.raises(ValueError):
        adapters.load([one(p__lora_A__weight=a, p__lora_B__weight=b[:, :2].contiguous())], "p.weight")
    with pytest.raises(TypeError, match="dtype"):
        adapters.load([good, one(p__lora_A__weight=a.float(), p__lora_B__weight=b.float())], "p.weight")
    p, q = adapters.load([good, one(p__lora_A__weight=a.float(), p__lora_B__weight=b.float())], "p.weight", dtype=torch.bfloat16)
    assert torch.equal(p[0], p[1]) and torch.equal(q[0], q[1])
