"""Operators with adapters at the ranks where their kernels change layout, against the definition in 64 bits (bounds as in
test_gpu_ops)."""
import pytest
import torch

from test_gpu_ops import DTYPES, _check, _check_project, _index, _inputs, _randn

pytestmark = pytest.mark.gpu


@pytest.fixture(autouse=True)
def _library(gpu):
    return gpu


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("out, inp", [(264, 520), (130, 251)])
@pytest.mark.parametrize("rank", [127, 128, 129, 136, 144, 145, 160, 161, 176, 191, 192, 193, 208, 209, 224, 240, 255, 256])
def test_merge_of_every_layout(dtype, out, inp, rank):
    from lmz_b200 import adapters
    w, a, b = _randn(50, (out, inp), dtype), _randn(51, (rank, inp), dtype, inp ** -0.5), _randn(52, (out, rank), dtype)
    want = w.double() + 0.5 * (b.double() @ a.double())
    size = w.double().abs() + 0.5 * (b.double().abs() @ a.double().abs())
    got = adapters.merge(w, a, b, scale=0.5)
    _check(got, want, size, torch.zeros_like(want), rank + 4, "merge")
    assert adapters.merge(w, a, b, scale=0.5, out=w) is w and torch.equal(w, got)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("tokens, inp, out, n, kind", [(1, 264, 520, 1, "none"), (90, 264, 392, 3, "mixed"), (700, 200, 320, 2, "runs"), (500, 136, 1288, 1, "none"),
                                                       (333, 131, 203, 4, "runs"), (1800, 264, 2056, 5, "mixed")])
@pytest.mark.parametrize("rank", [120, 129, 136, 144, 160, 192, 200, 247, 255])
def test_project_and_its_gradients_of_every_layout(dtype, tokens, inp, out, n, kind, rank):
    from lmz_b200 import adapters
    x, w, a, b, scales = _inputs(tokens, inp, out, rank, n, dtype)
    index, dy = _index(kind, tokens, n), _randn(40, (tokens, out), dtype)
    leaves = [t.requires_grad_(True) for t in (x, a, b)]
    y = adapters.project(x, w, a, b, index, scale=scales)
    _check_project(x, w, a, b, scales, index, y.detach(), dy, torch.autograd.grad(y, leaves, dy))


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("tokens, inp, out, rank, n, kind", [(1, 72, 136, 8, 40, "runs"), (17, 264, 392, 5, 2, "runs"), (200, 136, 264, 16, 70, "runs"), (200, 136, 264, 16, 13, "short"),
                                                             (600, 264, 1032, 24, 38, "short"), (900, 72, 328, 40, 500, "runs"), (5000, 72, 136, 8, 300, "short"),
                                                             (5000, 72, 136, 8, 312, "short"), (5000, 72, 136, 8, 313, "short")])
def test_more_and_fewer_adapters_than_sixteens(dtype, tokens, inp, out, rank, n, kind):
    from lmz_b200 import adapters
    x, w, a, b, scales = _inputs(tokens, inp, out, rank, n, dtype)
    index, dy = _index(kind, tokens, n), _randn(40, (tokens, out), dtype)
    leaves = [t.requires_grad_(True) for t in (x, a, b)]
    y = adapters.project(x, w, a, b, index, scale=scales)
    _check_project(x, w, a, b, scales, index, y.detach(), dy, torch.autograd.grad(y, leaves, dy))
