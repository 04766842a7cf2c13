"""Products of activations with a checkpoint's weights, and what stands behind them in a layer: bias, activation, an
elementwise factor (the other half of a gated block) and the residual, in the product's own kernel.

`adapters.project` is the same for a frozen weight with adapters of many requests beside it, `experts.project` for rows that
have different weights.
"""
from __future__ import annotations

from . import _ops, gpu

ACTIVATIONS = {None: 0, "relu": 1, "silu": 2, "gelu": 3, "gelu_tanh": 4}


def project(x, weight, bias=None, activation=None, times=None, residual=None):
    """`act(x @ weight.T + bias) * times + residual`.

    `x`: [..., in], `weight`: [out, in], `bias`: [out], `times` and `residual`: [..., out], all bfloat16 or all float16; what is not given is left
    out.  `activation`: None, "relu", "silu", "gelu" (with the error function) or "gelu_tanh" (its approximation by tanh).

    Returns a contiguous [..., out], worked out in 32 bits and rounded once.  Differentiable once, in all five tensors; where an
    activation's slope or a factor's gradient is wanted the sums are kept for that in 32 bits; their own gradient, which is multiplied once more, is rounded to the tensors' type
    (float16: times a power of two that brings the largest to where that has room, so that its own range is no limit).  Gradients are the same in every run."""
    import torch
    index = _ops.on_cuda("x weight bias times residual", x, weight, bias, times, residual)
    code = _ops.type_code(x, "x", half_only=True)
    _ops.same_type(x.dtype, "x", weight=weight, bias=bias, times=times, residual=residual)
    kind = _activation(activation)
    _check_shapes(x, weight, bias, times, residual)
    if torch.is_grad_enabled() and _ops.trained(x, weight, bias, times, residual):
        return _function().apply(x, weight, bias, times, residual, None, kind)
    return _forward(index, code, code, kind, x, weight, bias, times, residual, None, None, None, False)[0]


def project_8bit(x, x_scale, weight, weight_scale, bias=None, activation=None, times=None, residual=None, dtype=None):
    """The same for rows and a weight in 8 bits: `act(x_scale * weight_scale * (x @ weight.T) + bias) * times + residual`.

    `x`: [..., in] and `weight`: [out, in], float8_e4m3fn; `x_scale`: x's leading shape, one per row, and `weight_scale`: [out], float32
    (what `norms.rms_norm_8bit` and `norms.to_8bit` return).  `dtype`: the result's, bfloat16 (the default) or float16; bias, times and residual
    are of it.  Products of 8 bits are exact and summed in 32 bits.  Not differentiable."""
    import torch
    index = _ops.on_cuda("x x_scale weight weight_scale bias times residual", x, x_scale, weight, weight_scale, bias, times, residual)
    dtype = torch.bfloat16 if dtype is None else dtype
    if dtype is not torch.bfloat16 and dtype is not torch.float16:
        raise TypeError(f"dtype must be bfloat16 or float16, not {dtype}")
    for name, t in (("x", x), ("weight", weight)):
        if t.dtype is not torch.float8_e4m3fn:
            raise TypeError(f"{name} must be float8_e4m3fn, not {t.dtype}")
    _ops.same_type(dtype, "the result", bias=bias, times=times, residual=residual)
    kind = _activation(activation)
    _check_shapes(x, weight, bias, times, residual)
    for name, t, shape in (("x_scale", x_scale, x.shape[:-1]), ("weight_scale", weight_scale, weight.shape[:1])):
        if t.dtype is not torch.float32 or t.shape != shape:
            raise ValueError(f"{name} must be float32 {list(shape)}, not {t.dtype} {list(t.shape)}")
    if torch.is_grad_enabled() and _ops.trained(x, x_scale, weight, weight_scale, bias, times, residual):
        raise ValueError("project_8bit has no gradient: call it under torch.no_grad()")
    return _forward(index, _ops.E4M3, _ops.BF16 if dtype is torch.bfloat16 else _ops.F16, kind, x, weight, bias, times, residual, None, x_scale, weight_scale, False)[0]


def _activation(name) -> int:
    try:
        return ACTIVATIONS[name]
    except (KeyError, TypeError):
        raise ValueError(f"activation must be one of {', '.join(map(repr, ACTIVATIONS))}, not {name!r}") from None


def _check_shapes(x, weight, bias, times, residual):
    shape, of_weight = x.shape, weight.shape
    if len(of_weight) != 2 or len(shape) < 1 or shape[-1] != of_weight[1]:
        raise ValueError(f"x {list(shape)} and weight {list(of_weight)} do not fit [..., in] and [out, in]")
    out, inp = of_weight
    if not out or not inp:
        raise ValueError("an empty weight")
    if weight.stride(1) != 1 and inp > 1:
        raise ValueError("the elements of a row of the weight must be next to each other")
    if bias is not None and bias.shape != (out,):
        raise ValueError(f"bias must be [{out}], not {list(bias.shape)}")
    if times is not None and times.shape != (*shape[:-1], out):
        raise ValueError(f"times must be {[*shape[:-1], out]}, not {list(times.shape)}")
    if residual is not None and residual.shape != (*shape[:-1], out):
        raise ValueError(f"residual must be {[*shape[:-1], out]}, not {list(residual.shape)}")


def _call(code, rcode, kind, x, weight, bias, times, residual, offsets, x_scale=None, weight_scale=None, y=None, z=None):
    """(`lmz_product`, copies that live as long as it) for x as [rows, in]."""
    x = _ops.rows_of(x)
    p = _ops.Product(x.data_ptr(), weight.data_ptr())      # (set one by one, and only what there is: a third of the time of all at once)
    p.rows, p.in_ = x.shape
    p.x_stride, p.dtype, p.result_dtype, p.activation, p.experts = x.stride(0), code, rcode, kind, 1
    if weight.dim() == 2:
        p.out, p.weight_stride = weight.shape[0], weight.stride(0)
    else:
        p.experts, p.out, _ = weight.shape
        p.weight_plane, p.weight_stride, _ = weight.stride()
    held = [x]
    if bias is not None:
        bias = _ops.packed(bias)
        p.bias = bias.data_ptr()
        held.append(bias)
    if times is not None:
        times = _ops.rows_of(times)
        p.times, p.times_stride = times.data_ptr(), times.stride(0)
        held.append(times)
    if residual is not None:
        residual = _ops.rows_of(residual)
        p.residual, p.residual_stride = residual.data_ptr(), residual.stride(0)
        held.append(residual)
    if offsets is not None:
        offsets = _ops.packed(offsets)
        p.offsets, p.offset_bytes = offsets.data_ptr(), offsets.element_size()
        held.append(offsets)
    if x_scale is not None:
        x_scale, weight_scale = _ops.packed(x_scale), _ops.packed(weight_scale)
        p.x_scale, p.weight_scale = x_scale.data_ptr(), weight_scale.data_ptr()
        held += x_scale, weight_scale
    if y is not None:
        p.y = y.data_ptr()
    if z is not None:
        p.z = z.data_ptr()
    return p, held


def _work(p, grad: int, like):
    size = gpu.library().lmz_gpu_product_work_bytes(p, grad)
    if not size:
        return None
    import torch
    work = like.new_empty(size, dtype=torch.uint8)
    p.work = work.data_ptr()
    return work


def _forward(index, code, rcode, kind, x, weight, bias, times, residual, offsets, x_scale, weight_scale, keep):
    """(y, the sums in 32 bits if `keep`)."""
    import torch
    like = times if times is not None else residual        # (of the result's shape and type)
    y = _ops.empty_like(like) if like is not None else x.new_empty((*x.shape[:-1], weight.shape[-2]), dtype=torch.bfloat16 if rcode == _ops.BF16 else torch.float16)
    p, held = _call(code, rcode, kind, x, weight, bias, times, residual, offsets, x_scale, weight_scale, y)
    z = None
    if keep:
        z = y.new_empty(gpu.library().lmz_gpu_product_z_bytes(p), dtype=torch.uint8)
        p.z = z.data_ptr()
    held = held, _work(p, 0, x)                            # (copies and workspace live until the launch)
    _ops.launch(index, "lmz_gpu_product_dev", p)
    return y, z


def _backward(kind, dy, x, weight, bias, times, offsets, z, wanted):
    """The gradients of x, weight, bias and times, where `wanted`."""
    _ops.no_tangents("dy", dy)
    code = _ops.type_code(x, "x", half_only=True)
    grads = [_ops.empty_like(t) if w else None for t, w in zip((x, weight, bias, times), wanted)]
    dy, at = _ops.packed(dy), _ops.address
    p, held = _call(code, code, kind, x, weight, bias, times, None, offsets, z=z)
    p.dy = dy.data_ptr()
    p.dx, p.dweight, p.dbias, p.dtimes = at(grads[0]), at(grads[1]), at(grads[2]), at(grads[3])
    held = held, _work(p, 1, x)
    _ops.launch(x.get_device(), "lmz_gpu_product_grad_dev", p)
    return grads


def _function():
    """The autograd function (made on first use: importing this package does not import torch)."""
    global _made
    if _made is None:
        import torch

        class Product(torch.autograd.Function):
            @staticmethod
            def forward(ctx, x, weight, bias, times, residual, offsets, kind):
                code = _ops.type_code(x, "x", half_only=True)
                wanted = ctx.needs_input_grad[:4]                # (a slope, or the factor's gradient, goes by the sums)
                y, z = _forward(x.get_device(), code, code, kind, x, weight, bias, times, residual, offsets, None, None, wanted[3] or (kind and any(wanted)))
                ctx.save_for_backward(x, weight, bias, times, offsets, z)
                ctx.kind = kind
                return y

            @staticmethod
            @_ops.once
            def backward(ctx, dy):
                x, weight, bias, times, offsets, z = ctx.saved_tensors
                wanted = ctx.needs_input_grad[:4]
                grads = _backward(ctx.kind, dy, x, weight, bias, times, offsets, z, wanted) if any(wanted) else [None] * 4
                return *grads, dy if ctx.needs_input_grad[4] else None, None, None

        _made = Product
    return _made


_made = None
