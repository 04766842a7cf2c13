"""Calls of the operators that their documentation allows, or that they have to refuse, beside the sizes of test_gpu_ops."""
import numpy as np
import pytest
import torch

from test_gpu_ops import _archive, _check_project, _inputs, _randn

pytestmark = pytest.mark.gpu


@pytest.fixture(autouse=True)
def _library(gpu):
    return gpu


def test_tangents_are_refused_beside_a_scale_and_in_a_gradient():
    from torch.autograd import forward_ad

    from lmz_b200 import adapters, embed
    x, w, a, b, scales = _inputs(6, 64, 96, 8, 3, torch.bfloat16)
    index, dy = torch.zeros(6, dtype=torch.int32, device="cuda"), _randn(1, (6, 96), torch.bfloat16)
    table, ids = _randn(2, (5, 8), torch.float32).requires_grad_(True), torch.zeros(3, dtype=torch.int64, device="cuda")
    y, e = adapters.project(x.requires_grad_(True), w, a, b, index, scale=scales), embed.lookup(table, ids)
    with forward_ad.dual_level():
        with pytest.raises(NotImplementedError, match="tangent"):
            adapters.project(x, w, a, b, index, scale=forward_ad.make_dual(scales, torch.ones_like(scales)))
        with pytest.raises(NotImplementedError, match="tangent"):
            torch.autograd.grad(y, x, forward_ad.make_dual(dy, dy.clone()))
        with pytest.raises(NotImplementedError, match="tangent"):
            torch.autograd.grad(e, table, forward_ad.make_dual(e.detach(), e.detach().clone()))
        assert adapters.project(x, w, a, b, index, scale=scales).shape == (6, 96)


def test_one_row_of_an_archive_by_its_number():
    """Row numbers of any shape: of none, too."""
    from lmz_b200 import archive, decode
    table = _randn(71, (900, 250), torch.bfloat16, 0.02)
    ar = archive.Archive(_archive({"norm": _randn(70, (33,), torch.bfloat16), "emb": table}, mapped=True))
    for row in (7, np.int64(7), np.array(7, dtype=np.uint8), torch.tensor(7)):
        got = decode.decode_rows(ar, "emb", row)
        assert got.shape == (250,) and torch.equal(got, table[7])
    assert decode.decode_rows(ar, "emb", torch.tensor([[899], [0]])).shape == (2, 1, 250)
    with pytest.raises(IndexError):
        decode.decode_rows(ar, "emb", 900)


@pytest.mark.parametrize("n", [3, 33])
def test_rows_gradient_of_the_widest_rows(n):
    """2^24 - 1 elements of 16 bits, which move one at a time: more slices of a row than a grid has along y."""
    from lmz_b200 import embed
    dim = (1 << 24) - 1
    table = torch.zeros((2, dim), dtype=torch.float16, device="cuda").requires_grad_(True)
    ids = torch.ones(n, dtype=torch.int64, device="cuda")
    ids[1] = 0
    dy = torch.randint(-8, 9, (n, dim), generator=torch.Generator(device="cuda").manual_seed(3), device="cuda", dtype=torch.int8).to(torch.float16)
    (got,) = torch.autograd.grad(embed.lookup(table, ids), table, dy)
    assert torch.equal(got[0], dy[1])
    want = torch.zeros(dim, device="cuda")                 # (whole numbers up to 33 * 8: exact in F16 too)
    for t in range(n):
        if t != 1:
            want += dy[t]
    assert torch.equal(got[1].float(), want)


def test_a_merge_in_place_is_noticed():
    """As any operator of torch that writes to a tensor which a gradient still needs; and a leaf is not written to."""
    from lmz_b200 import adapters
    w, a, b = _randn(50, (16, 24), torch.bfloat16), _randn(51, (4, 24), torch.bfloat16), _randn(52, (16, 4), torch.bfloat16)
    v = torch.ones_like(w).requires_grad_(True)
    y = (v * w).sum()
    adapters.merge(w, a, b, out=torch.empty_like(w))       # (leaves w alone)
    (g,) = torch.autograd.grad(y, v, retain_graph=True)
    assert torch.equal(g, w)
    adapters.merge(w, a, b, out=w)
    with pytest.raises(RuntimeError, match="modified by an inplace operation"):
        y.backward()
    leaf = torch.empty_like(w).requires_grad_(True)
    with pytest.raises(ValueError, match="gradient"):
        adapters.merge(w, a, b, out=leaf)
    with torch.no_grad():
        assert adapters.merge(w, a, b, out=leaf) is leaf
    with torch.inference_mode():
        out = torch.empty_like(w)
        assert torch.equal(adapters.merge(w, a, b, out=out), leaf)


def test_merged_tensors_are_checked(monkeypatch):
    from lmz_b200 import adapters, archive, decode, gpu
    w, a, b = _randn(50, (32, 64), torch.bfloat16), _randn(51, (4, 64), torch.bfloat16), _randn(52, (32, 4), torch.bfloat16)
    ar, tuned = archive.Archive(_archive({"p.weight": w})), archive.Archive(_archive({"p.lora_A.weight": a, "p.lora_B.weight": b}))
    (got,) = decode.decode_tensors(ar, ["p.weight"], adapter=tuned).values()
    assert torch.equal(got, adapters.merge(w, a, b))
    monkeypatch.setattr(gpu.library(), "lmz_gpu_ops_gave_up", lambda: 1)      # a merge whose wait has run out
    with pytest.raises(RuntimeError, match="gave up"):
        decode.decode_tensors(ar, ["p.weight"], adapter=tuned)
    (plain,) = decode.decode_tensors(ar, ["p.weight"]).values()
    assert torch.equal(plain, w)


@pytest.mark.parametrize("tokens", [1, 64, 700])
@pytest.mark.parametrize("n", [2, 5])
def test_without_an_index_only_the_first_adapter_has_gradients(tokens, n):
    from lmz_b200 import adapters
    x, w, a, b, scales = _inputs(tokens, 64, 136, 8, n, torch.bfloat16)
    dy = _randn(40, (tokens, 136), torch.bfloat16)
    leaves = [t.requires_grad_(True) for t in (x, a, b)]
    y = adapters.project(x, w, a, b, scale=scales)
    grads = torch.autograd.grad(y, leaves, dy)
    _check_project(x, w, a, b, scales, None, y.detach(), dy, grads)
    zeros = torch.zeros(tokens, dtype=torch.int32, device="cuda")
    for g, h in zip(grads, torch.autograd.grad(adapters.project(x, w, a, b, zeros, scale=scales), leaves, dy)):
        assert torch.equal(g, h)
    assert (grads[1][1:] == 0).all() and (grads[2][1:] == 0).all()
