"""Norms, products with an epilogue and experts' products: what can be said of them without a GPU."""
import ctypes
import os
import re
import subprocess

import pytest
import torch

from lmz_b200 import _ops, build, experts, linear, norms

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))


@pytest.fixture(scope="module")
def lib():
    path = build.build()
    assert path, build.last_error
    lib = ctypes.CDLL(path)
    _ops.bind(lib)
    lib.lmz_gpu_last_error.restype = ctypes.c_char_p
    return lib


@pytest.mark.parametrize("mirror, name", [(_ops.Norm, "lmz_norm"), (_ops.Product, "lmz_product")])
def test_structures_mirror_the_header(tmp_path, mirror, name):
    names = [n for n, _ in mirror._fields_]
    src = tmp_path / "layout.c"
    src.write_text("#include <stdio.h>\n#include \"lmz_b200.h\"\nint main(void) {\n" +
                   "".join(f'printf("%zu\\n", offsetof({name}, {n.rstrip("_")}));\n' for n in names) + f'printf("%zu\\n", sizeof({name})); return 0; }}\n')
    exe = tmp_path / "layout"
    subprocess.run(["gcc", "-I", os.path.join(ROOT, "include"), "-o", str(exe), str(src)], check=True)
    said = [int(v) for v in subprocess.run([str(exe)], capture_output=True, text=True, check=True).stdout.split()]
    assert said == [getattr(mirror, n).offset for n in names] + [ctypes.sizeof(mirror)]


def test_numbers_of_the_header():
    text = open(os.path.join(ROOT, "include", "lmz_b200.h")).read()
    said = {k: int(v) for k, v in re.findall(r"#define LMZ_GPU_(E4M3|MAX_EXPERTS|ACT_\w+) (\d+)", text)}
    assert said == {"E4M3": _ops.E4M3, "MAX_EXPERTS": experts.MAX_EXPERTS} | {"ACT_" + (k or "none").upper(): v for k, v in linear.ACTIVATIONS.items()}


def _norm(**kw):
    p = _ops.Norm()
    p.weight, p.tokens, p.dim, p.x_stride, p.eps = 64, 4, 64, 64, 1e-6    # (nothing is read at these addresses)
    for k, v in kw.items():
        setattr(p, k, v)
    return p


@pytest.mark.parametrize("bad", [dict(dtype=3), dict(weight_dtype=9), dict(dtype=2), dict(weight_dtype=1), dict(tokens=1 << 31), dict(dim=0), dict(dim=1 << 24), dict(eps=-1.0),
                                 dict(eps=float("nan")), dict(eps=float("inf"))])
def test_norms_the_library_refuses(lib, bad):
    assert lib.lmz_gpu_norm_dev(_norm(**bad), None) == -2 and lib.lmz_gpu_last_error()
    assert lib.lmz_gpu_norm_grad_dev(_norm(**bad), None) == -2


@pytest.mark.parametrize("without", [dict(), dict(x=64), dict(y=64), dict(x=64, y=64, q=64, scale=64), dict(x=64, q=64), dict(x=64, weight=None, y=64)])
def test_norms_without_what_they_write_to(lib, without):
    assert lib.lmz_gpu_norm_dev(_norm(**without), None) == -2 and lib.lmz_gpu_last_error()


@pytest.mark.parametrize("without", [dict(), dict(x=64, rstd=64), dict(x=64, dy=64), dict(x=64, rstd=64, dy=64, weight=None), dict(x=64, rstd=64, dy=64, dweight=64), dict(rstd=64, dy=64)])
def test_norms_gradients_without_what_they_go_by(lib, without):
    assert lib.lmz_gpu_norm_grad_dev(_norm(dx=64, **without), None) == -2 and lib.lmz_gpu_last_error()


def _product(**kw):
    p = _ops.Product()
    p.rows, p.in_, p.out, p.x_stride, p.weight_stride, p.experts = 4, 64, 64, 64, 64, 1
    for k, v in kw.items():
        setattr(p, k, v)
    return p


@pytest.mark.parametrize("bad", [dict(dtype=2), dict(dtype=9, result_dtype=9), dict(result_dtype=1), dict(dtype=3), dict(dtype=3, x_scale=64, weight_scale=64, offsets=64, offset_bytes=4),
                                 dict(dtype=3, x_scale=64, weight_scale=64, result_dtype=2), dict(offsets=64, offset_bytes=2), dict(offsets=64, offset_bytes=4, experts=0),
                                 dict(offsets=64, offset_bytes=4, experts=1025), dict(experts=2), dict(in_=0), dict(out=0), dict(in_=1 << 21), dict(out=1 << 21), dict(rows=1 << 31),
                                 dict(activation=5)])
def test_products_the_library_refuses(lib, bad):
    assert lib.lmz_gpu_product_dev(_product(**bad), None) == -2 and lib.lmz_gpu_last_error()
    assert lib.lmz_gpu_product_grad_dev(_product(**bad), None) == -2


def test_products_in_8_bits_have_no_gradients_in_the_library(lib):
    assert lib.lmz_gpu_product_grad_dev(_product(dtype=3, x_scale=64, weight_scale=64), None) == -2


@pytest.mark.parametrize("without", [dict(), dict(x=64, y=64), dict(weight=64, y=64), dict(x=64, weight=64), dict(x=2, weight=64, y=64)])
def test_products_without_what_they_go_by(lib, without):
    assert lib.lmz_gpu_product_dev(_product(**without), None) == -2 and lib.lmz_gpu_last_error()


@pytest.mark.parametrize("without", [dict(dx=64), dict(dx=64, dy=64), dict(dweight=64, dy=64), dict(dx=64, dy=64, weight=64, activation=2, work=256), dict(dx=64, dy=64, z=64, activation=2, weight=64),
                                     dict(dtimes=64, dy=64, times=64, work=256)])
def test_products_gradients_without_what_they_go_by(lib, without):
    assert lib.lmz_gpu_product_grad_dev(_product(**without), None) == -2 and lib.lmz_gpu_last_error()


@pytest.mark.parametrize("id_bytes, n, count", [(2, 1, 4), (4, 1, 0), (4, 1, 1025), (8, 1 << 31, 4)])
def test_orders_the_library_refuses(lib, id_bytes, n, count):
    assert lib.lmz_gpu_order_dev(None, id_bytes, n, count, None, None, None, None) == -2


class _OnGpu:
    """A stand-in for a CUDA tensor as far as the checks of arguments look: shapes, types and strides are a CPU tensor's."""
    def __init__(self, t):
        self.t = t

    def __getattr__(self, name):
        return getattr(self.t, name)

    def get_device(self):
        return 0


def _t(*shape, dtype=torch.bfloat16, grad=False):
    return _OnGpu(torch.zeros(shape, dtype=dtype, requires_grad=grad))


F8 = torch.float8_e4m3fn
REFUSED = [
    (TypeError, "x must be", lambda: norms.rms_norm(_t(4, 8, dtype=torch.int32), _t(8))),
    (TypeError, "weight must be", lambda: norms.rms_norm(_t(4, 8), _t(8, dtype=torch.float16))),
    (TypeError, "weight must be", lambda: norms.rms_norm(_t(4, 8, dtype=torch.float32), _t(8))),
    (ValueError, "weight \\[dim\\]", lambda: norms.rms_norm(_t(4, 8), _t(7))),
    (ValueError, "weight \\[dim\\]", lambda: norms.rms_norm(_t(4, 0), _t(0))),
    (ValueError, "residual must be", lambda: norms.rms_norm(_t(4, 8), _t(8), _t(4, 7))),
    (ValueError, "residual must be", lambda: norms.rms_norm(_t(4, 8), _t(8), _t(4, 8, dtype=torch.float16))),
    (ValueError, "eps", lambda: norms.rms_norm(_t(4, 8), _t(8), eps=-1.0)),
    (ValueError, "eps", lambda: norms.rms_norm(_t(4, 8), _t(8), eps=float("nan"))),
    (ValueError, "no gradient", lambda: norms.rms_norm_8bit(_t(4, 8, grad=True), _t(8))),
    (ValueError, "no gradient", lambda: norms.to_8bit(_t(4, 8, grad=True))),
    (ValueError, "x must be", lambda: norms.to_8bit(_t(4, 0))),
    (TypeError, "x must be", lambda: norms.to_8bit(_t(4, 8, dtype=torch.float64))),
    (TypeError, "x must be", lambda: linear.project(_t(4, 8, dtype=torch.float32), _t(6, 8, dtype=torch.float32))),
    (TypeError, "weight is", lambda: linear.project(_t(4, 8), _t(6, 8, dtype=torch.float16))),
    (TypeError, "bias is", lambda: linear.project(_t(4, 8), _t(6, 8), bias=_t(6, dtype=torch.float32))),
    (ValueError, "activation", lambda: linear.project(_t(4, 8), _t(6, 8), activation="tanh")),
    (ValueError, "activation", lambda: linear.project(_t(4, 8), _t(6, 8), activation=[])),
    (ValueError, "do not fit", lambda: linear.project(_t(4, 8), _t(6, 7))),
    (ValueError, "do not fit", lambda: linear.project(_t(4, 8), _t(2, 6, 8))),
    (ValueError, "empty", lambda: linear.project(_t(4, 8), _t(0, 8))),
    (ValueError, "next to each other", lambda: linear.project(_t(4, 8), _OnGpu(torch.zeros(8, 6, dtype=torch.bfloat16).t()))),
    (ValueError, "bias must", lambda: linear.project(_t(4, 8), _t(6, 8), bias=_t(8))),
    (ValueError, "times must", lambda: linear.project(_t(4, 8), _t(6, 8), times=_t(6))),
    (ValueError, "residual must", lambda: linear.project(_t(4, 8), _t(6, 8), residual=_t(4, 8))),
    (TypeError, "dtype", lambda: linear.project_8bit(_t(4, 8, dtype=F8), _t(4, dtype=torch.float32), _t(6, 8, dtype=F8), _t(6, dtype=torch.float32), dtype=torch.float32)),
    (TypeError, "x must be", lambda: linear.project_8bit(_t(4, 8), _t(4, dtype=torch.float32), _t(6, 8, dtype=F8), _t(6, dtype=torch.float32))),
    (TypeError, "weight must be", lambda: linear.project_8bit(_t(4, 8, dtype=F8), _t(4, dtype=torch.float32), _t(6, 8, dtype=torch.uint8), _t(6, dtype=torch.float32))),
    (ValueError, "x_scale must", lambda: linear.project_8bit(_t(4, 8, dtype=F8), _t(5, dtype=torch.float32), _t(6, 8, dtype=F8), _t(6, dtype=torch.float32))),
    (ValueError, "weight_scale must", lambda: linear.project_8bit(_t(4, 8, dtype=F8), _t(4, dtype=torch.float32), _t(6, 8, dtype=F8), _t(6))),
    (TypeError, "residual is", lambda: linear.project_8bit(_t(4, 8, dtype=F8), _t(4, dtype=torch.float32), _t(6, 8, dtype=F8), _t(6, dtype=torch.float32),
                                                           residual=_t(4, 6, dtype=torch.float16))),
    (ValueError, "no gradient", lambda: linear.project_8bit(_t(4, 8, dtype=F8), _t(4, dtype=torch.float32, grad=True), _t(6, 8, dtype=F8), _t(6, dtype=torch.float32))),
    (TypeError, "index must", lambda: experts.sort(_t(4), 4)),
    (ValueError, "experts", lambda: experts.sort(_t(4, dtype=torch.int32), 0)),
    (ValueError, "experts", lambda: experts.sort(_t(4, dtype=torch.int32), 1025)),
    (TypeError, "x must be", lambda: experts.project(_t(4, 8, dtype=torch.float32), _t(2, 6, 8, dtype=torch.float32), _t(3, dtype=torch.int32))),
    (TypeError, "weight is", lambda: experts.project(_t(4, 8), _t(2, 6, 8, dtype=torch.float16), _t(3, dtype=torch.int32))),
    (TypeError, "offsets must", lambda: experts.project(_t(4, 8), _t(2, 6, 8), _t(3))),
    (ValueError, "offsets must", lambda: experts.project(_t(4, 8), _t(2, 6, 8), _t(2, dtype=torch.int32))),
    (ValueError, "do not fit", lambda: experts.project(_t(4, 8), _t(2, 6, 7), _t(3, dtype=torch.int32))),
    (ValueError, "do not fit", lambda: experts.project(_t(2, 4, 8), _t(2, 6, 8), _t(3, dtype=torch.int32))),
    (ValueError, "empty", lambda: experts.project(_t(4, 8), _t(0, 6, 8), _t(1, dtype=torch.int32))),
    (ValueError, "experts", lambda: experts.project(_t(4, 8), _t(1025, 6, 8), _t(1026, dtype=torch.int32))),
    (ValueError, "bias must", lambda: experts.project(_t(4, 8), _t(2, 6, 8), _t(3, dtype=torch.int32), bias=_t(6))),
    (ValueError, "times must", lambda: experts.project(_t(4, 8), _t(2, 6, 8), _t(3, dtype=torch.int32), times=_t(4, 8))),
    (ValueError, "next to each other", lambda: experts.project(_t(4, 8), _OnGpu(torch.zeros(2, 8, 6, dtype=torch.bfloat16).transpose(1, 2)), _t(3, dtype=torch.int32))),
    (ValueError, "activation", lambda: experts.project(_t(4, 8), _t(2, 6, 8), _t(3, dtype=torch.int32), activation="swish")),
]


@pytest.mark.parametrize("error, match, call", REFUSED)
def test_refused(error, match, call):
    with pytest.raises(error, match=match):
        call()


def test_tensors_that_are_not_on_one_gpu_are_refused():
    t = torch.ones((8, 8), dtype=torch.bfloat16)
    for call in (lambda: norms.rms_norm(t, t[0]), lambda: norms.rms_norm_8bit(t, t[0]), lambda: norms.to_8bit(t), lambda: linear.project(t, t),
                 lambda: linear.project_8bit(t, t, t, t), lambda: experts.sort(t, 4), lambda: experts.project(t, t, t)):
        with pytest.raises(ValueError, match="CUDA"):
            call()
    with pytest.raises(TypeError, match="torch tensor"):
        linear.project([1.0], t)


def test_tangents_are_refused():
    from torch.autograd import forward_ad
    t, v = torch.ones((8, 8), dtype=torch.bfloat16), torch.ones(8, dtype=torch.bfloat16)
    with forward_ad.dual_level():
        d, e = (forward_ad.make_dual(u, torch.ones_like(u)) for u in (t, v))
        for call in (lambda: norms.rms_norm(d, v), lambda: norms.rms_norm(t, e), lambda: norms.rms_norm(t, v, d), lambda: norms.rms_norm_8bit(d, v), lambda: norms.to_8bit(d),
                     lambda: linear.project(d, t), lambda: linear.project(t, d), lambda: linear.project(t, t, e), lambda: linear.project(t, t, times=d),
                     lambda: linear.project(t, t, residual=d), lambda: linear.project_8bit(t, e, t, v), lambda: experts.project(d, t, v), lambda: experts.project(t, d, v),
                     lambda: experts.project(t, t, v, bias=d), lambda: experts.project(t, t, v, times=d), lambda: norms._backward(t, v, v, d, None, 0.0, True, True),
                     lambda: norms._backward(t, v, v, t, d, 0.0, True, True), lambda: linear._backward(0, d, t, t, None, None, None, None, (True,) * 4)):
            with pytest.raises(NotImplementedError, match="tangent"):
                call()


@pytest.mark.parametrize("rows", [4, 5000])
def test_workspaces_hold_what_is_left_in_them(lib, rows):
    def size(**kw):
        return lib.lmz_gpu_product_work_bytes(_product(**(dict(rows=rows, in_=1024, out=1000, x_stride=1024, weight_stride=1024) | kw)), 1)
    assert size(activation=2) >= rows * 1000 * 2
    assert size(dbias=64) >= (rows + 31) // 32 * 1000 * 4
    p = _norm(tokens=rows, dim=1000)
    assert 0 < lib.lmz_gpu_norm_grad_work_bytes(p) <= rows * 1000 * 4 + 4000 * 4
