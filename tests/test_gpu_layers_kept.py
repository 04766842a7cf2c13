"""What a product keeps for its gradients: the sums in 32 bits where a slope or a factor's gradient goes by them, and nothing elsewhere."""
import itertools

import pytest
import torch

pytestmark = pytest.mark.gpu

BF16 = torch.bfloat16
NAMES = ("x", "weight", "bias", "times", "residual")


def _randn(seed, shape, std=1.0):
    g = torch.Generator(device="cuda")
    g.manual_seed(seed)
    return (torch.randn(shape, generator=g, device="cuda") * std).to(BF16)


def _kept(y):
    """Bytes that a result's autograd node holds beside the tensors that were given."""
    return sum(t.numel() for t in y.grad_fn.saved_tensors if t is not None and t.dtype is torch.uint8)


@pytest.mark.parametrize("kind", [None, "silu"])
@pytest.mark.parametrize("with_times", [False, True])
@pytest.mark.parametrize("by_experts", [False, True])
def test_sums_are_kept_where_a_gradient_goes_by_them(gpu, kind, with_times, by_experts):
    from lmz_b200 import experts, linear
    rows, inp, out = 45, 72, 80
    given = dict(x=_randn(1, (rows, inp)), weight=_randn(2, (2, out, inp) if by_experts else (out, inp), 0.2), bias=_randn(3, (2, out) if by_experts else out))
    if with_times:
        given["times"] = _randn(4, (rows, out))
    if not by_experts:
        given["residual"] = _randn(5, (rows, out))
    dy, offsets = _randn(6, (rows, out)), torch.tensor([0, 20, 41], device="cuda")

    def call(leaves):
        return experts.project(offsets=offsets, activation=kind, **leaves) if by_experts else linear.project(activation=kind, **leaves)

    every = {k: t.clone().requires_grad_(True) for k, t in given.items()}
    y = call(every)
    full = dict(zip(given, torch.autograd.grad(y, list(every.values()), dy)))
    for k in range(1, len(given)):
        for wanted in itertools.combinations(given, k):
            leaves = {n: t.clone().requires_grad_(n in wanted) for n, t in given.items()}
            z = call(leaves)
            assert torch.equal(z, y)
            assert _kept(z) == (rows * out * 4 if "times" in wanted or (kind and set(wanted) - {"residual"}) else 0), wanted
            for n, g in zip(wanted, torch.autograd.grad(z, [leaves[n] for n in wanted], dy)):
                assert torch.equal(g, full[n]), (wanted, n)
