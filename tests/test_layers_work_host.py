"""Workspaces of the layer operators hold all that the kernels leave in them at a time: the sizes are worked out here from what each kernel writes."""
import ctypes
import itertools

import pytest

from lmz_b200 import _ops, build

BF16, F16, F32 = _ops.BF16, _ops.F16, _ops.F32


@pytest.fixture(scope="module")
def lib():
    path = build.build()
    assert path, build.last_error
    lib = ctypes.CDLL(path)
    _ops.bind(lib)
    return lib


def _up(n, to):
    return (n + to - 1) // to * to


def _product(**kw):
    p = _ops.Product(256, 256)                              # (nothing is read at these addresses)
    p.rows, p.in_, p.out, p.experts, p.dy = 4, 64, 64, 1, 256
    for k, v in kw.items():
        setattr(p, k, v)
    p.x_stride, p.weight_stride, p.weight_plane = p.in_, p.in_, p.in_ * p.out
    return p


@pytest.mark.parametrize("rows, inp, out, experts", [(1, 1, 1, 1), (4, 1024, 1000, 1), (5000, 1024, 1000, 1), (5000, 77, 1001, 1), (5000, 77, 1001, 7), (40, 33, 50, 1024), (60000, 64, 20000, 1),
                                                     (60000, 63, 20001, 64)])
@pytest.mark.parametrize("dtype", [BF16, F16])
@pytest.mark.parametrize("activation, times", list(itertools.product([0, 2], [None, 256])))
def test_products_gradients(lib, rows, inp, out, experts, dtype, activation, times):
    def size(**wanted):
        p = _product(rows=rows, in_=inp, out=out, experts=experts, dtype=dtype, result_dtype=dtype, activation=activation, times=times, **wanted)
        if experts > 1:
            p.offsets, p.offset_bytes = 256, 4
        return lib.lmz_gpu_product_work_bytes(p, 1)

    e, own = 2, activation or times or out % 8
    # dz in rows that start on 16 bytes
    dz = rows * _up(out, 8) * e if own else 0
    # a row of 32 bits for each chunk of rows and each expert that meet: chunks of 4 rows, 32 at most, and no more than give 1024 blocks
    each = 32
    while each > 4 and rows * out < 1024 * 128 * 8 * each:
        each //= 2
    partial = ((rows + each - 1) // each + experts) * out * 4
    x = rows * _up(inp, 16) * e if inp % 8 else 0
    w = experts * out * _up(inp, 16) * e if inp % 8 else 0
    powers = experts * 4 if dtype == F16 and (activation or times) else 0
    assert size(dx=256, dweight=256, dbias=256) >= dz + partial + x + w + powers
    assert size(dbias=256) >= partial
    assert size(dx=256) >= dz + w + powers and size(dweight=256) >= dz + x + powers
    assert size(dx=256, dweight=256) >= dz + x + w + powers
    # and little beside: five boundaries of 256 bytes
    assert size(dx=256, dweight=256, dbias=256) <= dz + partial + x + w + powers + 5 * 256


@pytest.mark.parametrize("rows, inp, out, experts", [(5, 77, 9, 1), (5000, 1024, 1000, 1), (300, 31, 50, 12)])
def test_products(lib, rows, inp, out, experts):
    p = _product(rows=rows, in_=inp, out=out, experts=experts)
    if experts > 1:
        p.offsets, p.offset_bytes = 256, 8
    assert lib.lmz_gpu_product_work_bytes(p, 0) >= ((rows + experts * out) * _up(inp, 16) * 2 if inp % 8 else 0)
    assert lib.lmz_gpu_product_z_bytes(p) == rows * out * 4
    # in 8 bits rows of 16 elements start on 16 bytes
    p.dtype, p.offsets, p.experts = _ops.E4M3, None, 1
    assert lib.lmz_gpu_product_work_bytes(p, 0) >= ((rows + out) * _up(inp, 16) if inp % 16 else 0)


@pytest.mark.parametrize("tokens, dim", [(1, 1), (1, 4096), (7, 96), (300, 997), (5000, 1000), (16384, 4096), (100000, 8), (3, 16385), (700, 100000), (149, 8192), (1200, 16384)])
@pytest.mark.parametrize("dtype", [BF16, F16, F32])
def test_norms_gradients(lib, tokens, dim, dtype):
    p = _ops.Norm()
    p.tokens, p.dim, p.x_stride, p.dtype, p.weight_dtype, p.eps = tokens, dim, dim, dtype, dtype, 1e-6
    size = lib.lmz_gpu_norm_grad_work_bytes(p)
    for each in (16, 8):                                    # elements of a thread: where vectors have 16 bytes, and where they are narrower
        lanes = 1
        while lanes < 1024 and each * lanes < dim:
            lanes *= 2
        turns = (tokens + max(256, lanes) // lanes - 1) // (max(256, lanes) // lanes)
        blocks = min(turns, max(148, min(592, (turns + 1) // 2)))
        assert size >= blocks * dim * 4                     # a row of 32 bits for each block
    assert size <= min(tokens, 592) * dim * 4
