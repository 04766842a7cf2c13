"""Root-mean-square norms with the residual's addition in front, their output as it is or in 8 bits.

The weight is a checkpoint's tensor as `decode` leaves it in HBM; rows in 8 bits are what `linear.project_8bit` multiplies.
"""
from __future__ import annotations

from . import _ops, gpu


def rms_norm(x, weight, residual=None, eps: float = 1e-6):
    """`x / sqrt(mean(x^2) + eps) * weight` over the last dimension; with a residual `(norm of s, s)`, `s = x + residual`.

    `x`, `residual`: [..., dim], bfloat16, float16 or float32, the elements of a row next to each other.  `weight`: [dim], of their
    type or float32.  `s` is rounded to the tensors' type, and what is normed is the rounded one.  Squares are summed and
    the result is worked out in 32 bits and rounded once (so that a row's squares have to stay within float32's range).  Results are contiguous.

    Differentiable once, in x, residual and weight (and through s); the weight's gradient is summed in 32 bits in one order, and is the
    same in every run."""
    import torch
    index, code, wcode, eps = _checked(x, weight, residual, eps)
    if torch.is_grad_enabled() and (x.requires_grad or weight.requires_grad or (residual is not None and residual.requires_grad)):
        got = _function().apply(x, weight, residual, eps)
        return got if residual is not None else got[0]
    y, stream, _ = _forward(index, code, wcode, x, weight, residual, eps, False)
    return y if residual is None else (y, stream)


def rms_norm_8bit(x, weight, residual=None, eps: float = 1e-6):
    """The same in 8 bits: `(q, scale)`, with a residual `(q, scale, s)`.  `q`: [..., dim] float8_e4m3fn, the norm (in 32 bits) divided by its row's
    scale and rounded once; `scale`: x's leading shape in float32, the row's largest magnitude / 448, but no less than 2^-126.  A row with
    infinities or NaN among its results has a scale that is not finite.  Not differentiable."""
    index, code, wcode, eps = _checked(x, weight, residual, eps)
    _no_gradient("rms_norm_8bit", x, weight, residual)
    q, scale, stream = _eight_bits(index, code, wcode, x, weight, residual, eps)
    return (q, scale) if residual is None else (q, scale, stream)


def to_8bit(x):
    """`(q, scale)`: rows in 8 bits as above, without a norm: a weight's rows, or what comes out of an activation.  Not differentiable."""
    index = _ops.on_cuda("x", x)
    code = _ops.type_code(x, "x")
    if x.dim() < 1 or not x.shape[-1]:
        raise ValueError(f"x must be [..., dim], not {list(x.shape)}")
    _no_gradient("to_8bit", x)
    return _eight_bits(index, code, code, x, None, None, 0.0)[:2]


def _checked(x, weight, residual, eps):
    index = _ops.on_cuda("x weight residual", x, weight, residual)
    code, wcode = _ops.type_code(x, "x"), _ops.type_code(weight, "weight")
    if wcode not in (code, _ops.F32):
        raise TypeError(f"weight must be {x.dtype}, as x is, or float32, not {weight.dtype}")
    if x.dim() < 1 or not x.shape[-1] or weight.shape != x.shape[-1:]:
        raise ValueError(f"x must be [..., dim] and weight [dim], not {list(x.shape)} and {list(weight.shape)}")
    if residual is not None and (residual.dtype is not x.dtype or residual.shape != x.shape):
        raise ValueError(f"residual must be like x, {x.dtype} {list(x.shape)}, not {residual.dtype} {list(residual.shape)}")
    eps = _ops.finite(eps, "eps")
    if eps < 0:
        raise ValueError("eps must not be below zero")
    return index, code, wcode, eps


def _no_gradient(name, *tensors):
    import torch
    if torch.is_grad_enabled() and _ops.trained(*tensors):
        raise ValueError(f"{name} has no gradient: call it under torch.no_grad()")


def _call(code, wcode, x, weight, residual, eps, y=None, q=None, scale=None, stream=None, rstd=None):
    p = _ops.Norm(x.data_ptr())                            # (set one by one, and only what there is: a third of the time of all at once)
    p.tokens, p.dim = x.shape
    p.x_stride, p.dtype, p.weight_dtype, p.eps = x.stride(0), code, wcode, eps
    if weight is not None:
        p.weight = weight.data_ptr()
    if residual is not None:
        p.residual, p.residual_stride = residual.data_ptr(), residual.stride(0)
    if y is not None:
        p.y = y.data_ptr()
    if q is not None:
        p.q, p.scale = q.data_ptr(), scale.data_ptr()
    if stream is not None:
        p.stream = stream.data_ptr()
    if rstd is not None:
        p.rstd = rstd.data_ptr()
    return p


def _forward(index, code, wcode, x, weight, residual, eps, keep):
    """(y, s, rstd): s is None without a residual, rstd unless `keep`."""
    y, stream, rstd = _ops.empty_like(x), None if residual is None else _ops.empty_like(x), None
    x, weight, residual = _ops.rows_of(x), _ops.packed(weight), _ops.rows_of(residual)
    if keep:
        import torch
        rstd = x.new_empty(x.shape[0], dtype=torch.float32)
    _ops.launch(index, "lmz_gpu_norm_dev", _call(code, wcode, x, weight, residual, eps, y, None, None, stream, rstd))
    return y, stream, rstd


def _eight_bits(index, code, wcode, x, weight, residual, eps):
    import torch
    q, stream = _ops.empty_like(x, torch.float8_e4m3fn), None if residual is None else _ops.empty_like(x)
    scale = x.new_empty(x.shape[0] if x.dim() == 2 else x.shape[:-1], dtype=torch.float32)
    x, weight, residual = _ops.rows_of(x), _ops.packed(weight), _ops.rows_of(residual)
    _ops.launch(index, "lmz_gpu_norm_dev", _call(code, wcode, x, weight, residual, eps, None, q, scale, stream))
    return q, scale, stream


def _backward(s, weight, rstd, dy, ds, eps, want_dx, want_dw):
    """(dx, dweight) for the normed tensor s; dy and ds may be None where nobody asked for them."""
    import torch
    _ops.no_tangents("dy ds", dy, ds)
    if dy is None:                                         # (only the stream was used)
        return (ds if want_dx else None), (torch.zeros_like(weight) if want_dw else None)
    dx, dw = _ops.empty_like(s) if want_dx else None, _ops.empty_like(weight) if want_dw else None
    flat, weight, dy, ds = _ops.rows_of(s), _ops.packed(weight), _ops.packed(dy), _ops.packed(ds)
    p = _call(_ops.type_code(s, "x"), _ops.type_code(weight, "weight"), flat, weight, None, eps, rstd=rstd)
    p.dy, p.dstream, p.dx, p.dweight = dy.data_ptr(), _ops.address(ds), _ops.address(dx), _ops.address(dw)
    if want_dw:
        work = s.new_empty(gpu.library().lmz_gpu_norm_grad_work_bytes(p), dtype=torch.uint8)
        p.work = work.data_ptr()
    _ops.launch(s.get_device(), "lmz_gpu_norm_grad_dev", p)
    return dx, dw


def _function():
    """The autograd function (made on first use: importing this package does not import torch)."""
    global _made
    if _made is None:
        import torch

        class Norm(torch.autograd.Function):
            @staticmethod
            def forward(ctx, x, weight, residual, eps):
                ctx.set_materialize_grads(False)
                code, wcode = _ops.type_code(x, "x"), _ops.type_code(weight, "weight")
                y, stream, rstd = _forward(x.get_device(), code, wcode, x, weight, residual, eps, True)
                ctx.save_for_backward(x if stream is None else stream, weight, rstd)
                ctx.eps = eps
                return y, stream

            @staticmethod
            @_ops.once
            def backward(ctx, dy, ds):
                s, weight, rstd = ctx.saved_tensors
                want_x, want_w, want_r, _ = ctx.needs_input_grad
                dx, dw = (None, None) if dy is None and ds is None else _backward(s, weight, rstd, dy, ds, ctx.eps, want_x or want_r, want_w)
                return dx if want_x else None, dw, dx if want_r else None, None

        _made = Norm
    return _made


_made = None
