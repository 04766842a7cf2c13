"""Calls that the operators refuse, as far as it can be said without a GPU."""
import ctypes

import pytest
import torch

from lmz_b200 import _ops, adapters, build, embed


@pytest.fixture(scope="module")
def lib():
    path = build.build()
    assert path, build.last_error
    lib = ctypes.CDLL(path)
    _ops.bind(lib)
    return lib


def test_tangents_are_refused():
    """(Before anything is asked of a device: an operator that ran would lose them.)"""
    from torch.autograd import forward_ad
    t, i = torch.ones((8, 8), dtype=torch.bfloat16), torch.zeros(8, dtype=torch.int64)
    with forward_ad.dual_level():
        d, s = forward_ad.make_dual(t, torch.ones_like(t)), forward_ad.make_dual(torch.ones(1), torch.ones(1))
        for call in (lambda: embed.lookup(d, i), lambda: adapters.project(d, t, t, t), lambda: adapters.project(t, d, t, t),
                     lambda: adapters.project(t, t, d, t), lambda: adapters.project(t, t, t, d), lambda: adapters.merge(d, t, t),
                     lambda: adapters.merge(t, d, t), lambda: adapters.merge(t, t, d), lambda: adapters.merge(t, t, t, out=d),
                     lambda: _ops.no_tangents("x scale", t, s), lambda: embed._rows_grad(d, i, 8, 1.0),
                     lambda: adapters._backward(0, d, t, t, t, t, None, None, 1.0, None, (True, True, True))):
            with pytest.raises(NotImplementedError, match="tangent"):
                call()
        with pytest.raises(ValueError, match="CUDA"):      # (others are taken, or refused for what they lack)
            adapters.merge(t, t, t)


@pytest.mark.parametrize("out, inp, rank, dtype", [(8, 8, 0, 0), (8, 8, 257, 2), (8, 8, 4, 3), (0, 8, 4, 2), (8, 1 << 21, 4, 2)])
def test_wide_merges_the_library_refuses(lib, out, inp, rank, dtype):
    assert lib.lmz_gpu_merge_wide_dev(None, out, inp, inp, None, None, rank, 1.0, dtype, None, None) == -2
