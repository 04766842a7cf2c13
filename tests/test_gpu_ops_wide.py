"""Merges of adapters in FP32, into weights of every type.

Tolerance, per element: half a step of the result's type, and a sum of `rank` products in 32 bits, each added by a fused
multiplication (2^-24 of the sum of the magnitudes, each time), the weight's addition among them."""
import math

import pytest
import torch

from test_gpu_ops import ALL, _archive, _randn, _safetensors

pytestmark = pytest.mark.gpu


@pytest.fixture(autouse=True)
def _library(gpu):
    return gpu


def _check_merge(got, w, a, b, scale):
    want = w.double() + scale * (b.double() @ a.double())
    size = w.double().abs() + abs(scale) * (b.double().abs() @ a.double().abs())
    t = torch.finfo(got.dtype)
    bound = t.eps / 2 * want.abs() + (1 + t.eps) * (a.shape[0] + 3) * 2 ** -24 * size + t.smallest_normal * t.eps
    off = ((got.double() - want).abs() / bound).max()
    assert off <= 1, float(off)


@pytest.mark.parametrize("dtype", ALL)
@pytest.mark.parametrize("out, inp, rank", [(1, 1, 1), (8, 8, 8), (128, 128, 16), (130, 264, 17), (1000, 771, 5), (256, 1024, 64), (129, 512, 256), (70, 2000, 100), (257, 127, 15),
                                            (3, 4097, 33)])
def test_merge(dtype, out, inp, rank):
    from lmz_b200 import adapters
    w, a, b = _randn(50, (out, inp), dtype), _randn(51, (rank, inp), torch.float32, inp ** -0.5), _randn(52, (out, rank), torch.float32)
    got = adapters.merge(w, a, b, scale=1.5)
    assert got.dtype == dtype
    _check_merge(got, w, a, b, 1.5)
    for pad, at in ((3, 1), (4, 4), (4, 0)):               # rows of any stride and alignment
        block = torch.full((out, inp + pad), math.nan, dtype=dtype, device="cuda")
        block[:, at:inp + at] = w
        if at + inp <= block.shape[1]:
            assert torch.equal(adapters.merge(block[:, at:inp + at], a, b, scale=1.5), got)
    strided = torch.zeros((2 * rank, inp), device="cuda")
    strided[::2] = a
    assert torch.equal(adapters.merge(w, strided[::2], b.t().contiguous().t(), scale=1.5), got)
    assert adapters.merge(w, a, b, scale=1.5, out=w) is w and torch.equal(w, got)


def test_infinities_stay_in_their_row_and_column():
    from lmz_b200 import adapters
    w, a, b = torch.zeros((140, 150), device="cuda"), torch.ones((5, 150), device="cuda"), torch.ones((140, 5), device="cuda")
    b[3, 1], a[4, 7] = -math.inf, math.inf
    got = adapters.merge(w, a, b)
    want = torch.full((140, 150), 5.0, device="cuda")
    want[3] = -math.inf
    want[:, 7] = math.inf
    want[3, 7] = math.nan
    assert torch.equal(torch.nan_to_num(got, nan=7.0), torch.nan_to_num(want, nan=7.0))


def test_refusals():
    from lmz_b200 import adapters
    w, a, b = _randn(50, (16, 24), torch.bfloat16), _randn(51, (4, 24), torch.float32), _randn(52, (16, 4), torch.float32)
    for args, kind in (((w, a, b.bfloat16()), TypeError), ((w, a.bfloat16(), b), TypeError), ((w.float(), a.bfloat16(), b.bfloat16()), TypeError), ((w.double(), a, b), TypeError),
                       ((w, a.double(), b.double()), TypeError), ((w, a[:3], b), ValueError), ((w, a[:, :8], b), ValueError)):
        with pytest.raises(kind):
            adapters.merge(*args)
    assert adapters.merge(w[:0], a, b[:0]).shape == (0, 24)


@pytest.mark.parametrize("weight, factors", [(torch.float32, torch.float32), (torch.bfloat16, torch.float32), (torch.float32, torch.bfloat16), (torch.bfloat16, torch.float16),
                                             (torch.float16, torch.bfloat16), (torch.float16, torch.float16)])
def test_fine_tunes_from_archives(weight, factors):
    """Factors meet the weight as they are stored: nothing is rounded before the result is."""
    from lmz_b200 import archive, decode
    w, a, b = _randn(60, (264, 200), weight), _randn(61, (16, 200), factors, 0.07), _randn(62, (264, 16), factors, 0.3)
    ar, tuned = archive.Archive(_archive({"p.weight": w})), archive.Archive(_archive({"x.p.lora_A.weight": a, "x.p.lora_B.weight": b}))
    (got,) = decode.decode_tensors(ar, ["p.weight"], adapter=tuned, scale=2.0).values()
    assert got.dtype == weight
    if weight == factors != torch.float32:                 # (the tensor core's sums: test_gpu_ops)
        assert (got.double() - (w.double() + 2 * (b.double() @ a.double()))).abs().max() < 0.05
    else:
        _check_merge(got, w, a, b, 2.0)


def test_factors_of_two_types():
    from lmz_b200 import archive, decode
    w, a, b = _randn(60, (32, 24), torch.bfloat16), _randn(61, (4, 24), torch.float32), _randn(62, (32, 4), torch.bfloat16)
    ar, mixed = archive.Archive(_archive({"p.weight": w})), archive.Archive(_archive({"p.lora_A.weight": a, "p.lora_B.weight": b}))
    (got,) = decode.decode_tensors(ar, ["p.weight"], adapter=mixed).values()
    _check_merge(got, w, a, b.float(), 1.0)


@pytest.mark.parametrize("weight, pad", [(torch.bfloat16, 1), (torch.float32, 2), (torch.float32, 1), (torch.float16, 2)])
def test_a_weight_off_the_boundary_of_its_elements(weight, pad):
    """A safetensors header of any length puts a tensor at any byte: it comes as bytes then, and merged as what it is; so with
    an adapter's factors."""
    import struct

    import numpy as np

    from lmz_b200 import adapters, archive, decode
    from oracle import archive as oa

    def shifted(tensors):
        whole = _safetensors(tensors).tobytes()
        n = struct.unpack("<Q", whole[:8])[0]
        head = whole[8:8 + n].rstrip()
        head += b" " * ((pad - len(head)) % 8)
        member = struct.pack("<Q", len(head)) + head + whole[8 + n:]
        return archive.Archive(oa.write_archive([("m.safetensors", np.frombuffer(member, dtype=np.uint8))]))

    w, a, b = _randn(60, (64, 40), weight), _randn(61, (8, 40), weight, 0.2), _randn(62, (64, 8), weight)
    ar, tuned = shifted({"p.weight": w}), shifted({"p.lora_A.weight": a, "p.lora_B.weight": b})
    (plain,) = decode.decode_tensors(ar, ["p.weight"]).values()
    assert torch.equal(plain.clone().view(weight).view(64, 40), w)
    (got,) = decode.decode_tensors(ar, ["p.weight"], adapter=tuned, scale=0.5).values()
    assert torch.equal(got, adapters.merge(w, a, b, scale=0.5))
    p, q = adapters.load([tuned], "p.weight")
    assert torch.equal(p[0], a) and torch.equal(q[0], b)
