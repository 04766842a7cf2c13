"""Products and their gradients in every tile that they are worked out in: pairs of CTAs at 160 to 256 columns, one at 16 to 128, clusters of two to eight
that share a sum, with one weight and with several, against their definitions in 64 bits (tolerances: layers.py).

Shapes at which a different tile is chosen for one of the three products each; what is measured decides about that, so that they cover
most tiles whatever is chosen."""
import pytest
import torch

from layers import close, products as want_products

pytestmark = pytest.mark.gpu

# rows, in, out, experts
SHAPES = [
           (8, 8, 865, 1), (8, 396, 2394, 1), (8, 848, 8, 1), (8, 2393, 8, 1), (9, 8, 2355, 1), (597, 9, 1436, 1), (620, 1457, 8, 1), (636, 1131, 8, 1),
           (673, 8, 987, 1), (859, 8, 8, 1), (1149, 8, 2390, 1), (1207, 1363, 8, 1), (1214, 8, 2362, 1), (1260, 2294, 9, 1), (1296, 8, 1360, 1), (1527, 392, 2516, 1),
           (1812, 538, 1868, 1), (1941, 532, 1299, 1), (1995, 8, 521, 1), (2069, 514, 526, 1), (2371, 1092, 524, 1), (2398, 8, 8, 1), (2408, 556, 401, 1),
           (2431, 410, 8, 1), (2477, 148, 2671, 1), (2490, 8, 264, 1), (2514, 2715, 160, 1), (2531, 8, 2135, 1), (2561, 1905, 8, 1), (2716, 1086, 542, 1),
           (2774, 130, 2603, 1), (2804, 259, 8, 1), (8, 910, 8, 2), (578, 8, 985, 2), (689, 8, 1488, 2), (1262, 8, 2435, 2), (2009, 8, 8, 2), (2142, 9, 1190, 2),
           (2600, 1941, 8, 2), (8, 2360, 8, 3), (1170, 8, 1462, 3), (2359, 2629, 149, 3), (2543, 276, 8, 3), (8, 8, 1891, 5), (8, 8, 2396, 5), (9, 8, 855, 5),
           (9, 1815, 65, 5), (339, 2465, 258, 5), (355, 310, 2750, 5), (433, 8, 2829, 5), (440, 2840, 9, 5), (491, 2087, 12, 5), (538, 1423, 8, 5), (560, 9, 1937, 5),
           (575, 1046, 8, 5), (575, 2066, 8, 5), (631, 8, 1930, 5), (648, 1194, 8, 5), (660, 8, 1222, 5), (1137, 2248, 8, 5), (1171, 1415, 8, 5),
           (2286, 149, 2773, 5), (2371, 9, 269, 5), (2501, 8, 8, 5), (2548, 8, 1870, 5)
]
# the same in 8 bits
SHAPES_8 = [(657, 2061, 8), (9, 1737, 8), (2609, 8, 8), (1188, 2733, 9), (636, 3137, 8), (2418, 8, 277), (3271, 1112, 280), (2005, 1069, 1389), (2020, 1104, 1552), (3300, 8, 270),
            (64, 2048, 2048), (130, 8192, 1024), (1, 14336, 256)]


@pytest.fixture(autouse=True)
def _library(gpu):
    yield gpu
    from lmz_b200 import adapters
    adapters.check()


def _randn(seed, shape, dtype=torch.bfloat16, std=1.0):
    g = torch.Generator(device="cuda")
    g.manual_seed(seed)
    return (torch.randn(shape, generator=g, device="cuda") * std).to(dtype)


def _check(got, want):
    for name, t in got.items():
        try:
            close(t, want[name])
        except AssertionError as e:
            raise AssertionError(f"{name}: {e}") from None


@pytest.mark.parametrize("rows, inp, out, experts", SHAPES)
def test_tiles(rows, inp, out, experts):
    from lmz_b200 import experts as ex, linear
    x, b, r, dy = _randn(1, (rows, inp)), _randn(3, (experts, out)), _randn(5, (rows, out)), _randn(6, (rows, out))
    w = _randn(2, (experts, out, inp), std=inp ** -0.5)
    # (shares that differ by a few rows, so that they end inside of tiles)
    each = rows // experts
    starts = [min(rows, e * each + min(each, 3) * (e % 2)) for e in range(experts)] + [rows]
    if experts == 1:
        with torch.no_grad():
            _check({"y": linear.project(x, w[0], b[0], "silu", residual=r)}, want_products(x, w[0], b[0], "silu", residual=r))
            _check({"y": linear.project(x, w[0], b[0], "relu")}, want_products(x, w[0], b[0], "relu"))
    x.requires_grad_(True), w.requires_grad_(True)
    y = linear.project(x, w[0]) if experts == 1 else ex.project(x, w, torch.tensor(starts, device="cuda"), bias=b)
    dx, dw = torch.autograd.grad(y, (x, w), dy)
    with torch.no_grad():
        want = want_products(x, w, None if experts == 1 else b, dy=dy, starts=starts)
        _check({"y": y, "dx": dx, "dweight": dw}, want)


@pytest.mark.parametrize("rows, inp, out", SHAPES_8)
def test_tiles_in_8_bits(rows, inp, out):
    from lmz_b200 import linear, norms
    q, s = norms.to_8bit(_randn(1, (rows, inp), torch.float32, 3.0))
    wq, ws = norms.to_8bit(_randn(2, (out, inp), torch.float32, 0.02))
    b, r = _randn(3, out), _randn(5, (rows, out))
    _check({"y": linear.project_8bit(q, s, wq, ws, bias=b, activation="silu")}, want_products(q.float(), wq.float(), b, "silu", x_scale=s, weight_scale=ws, dtype=torch.bfloat16))
    _check({"y": linear.project_8bit(q, s, wq, ws, residual=r)}, want_products(q.float(), wq.float(), residual=r, x_scale=s, weight_scale=ws, dtype=torch.bfloat16))
