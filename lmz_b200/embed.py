"""Rows of an embedding table, and the table's gradient.

The table is a checkpoint's tensor as `decode` leaves it in HBM (a typed view of an archive's output, or any other
CUDA tensor); `decode.decode_rows` takes rows straight out of an archive with the same kernel.
"""
from __future__ import annotations

from . import _ops, gpu


def lookup(table, tokens, scale: float = 1.0):
    """`scale * table[tokens]`: a row of the table for every token.

    `table`: [rows, dim], bfloat16, float16 or float32, the elements of a row next to each other (rows may lie any
    stride apart).  `tokens`: int32 or int64 ids of any shape; an id outside [0, rows) -- the padding of a batch -- gives a
    row of zeros and takes no part in the gradient.  Returns a contiguous tensor of shape `tokens.shape + (dim,)`, rounded
    once from 32 bits (with a scale of one, the table's own bits).

    Differentiable in `table`, once: the gradient is dense and contiguous, summed in 32 bits over each row's tokens in their
    order, and the same in every run."""
    import torch
    index = _ops.on_cuda("table tokens", table, tokens)
    code = _ops.type_code(table, "table")
    id_bytes = _ops.whole_numbers(tokens, "tokens")
    if table.dim() != 2:
        raise ValueError(f"table must be [rows, dim], not {list(table.shape)}")
    if table.stride(1) != 1 and table.shape[1] > 1:
        raise ValueError("the elements of a row of the table must be next to each other")
    if scale != 1.0:
        scale = _ops.finite(scale)
    if table.requires_grad and torch.is_grad_enabled():
        return _function().apply(table, tokens, scale)
    return _rows(index, code, id_bytes, table, tokens, scale)


def _rows(index, code, id_bytes, table, tokens, scale):
    rows, dim = table.shape
    out = table.new_empty((*tokens.shape, dim))
    n = tokens.numel()
    if n and dim:
        ids = tokens if tokens.is_contiguous() else tokens.contiguous()
        _ops.launch(index, "lmz_gpu_rows_dev", table.data_ptr(), rows, dim, table.stride(0), code, ids.data_ptr(), id_bytes, n, scale, out.data_ptr())
    return out


def _rows_grad(dy, tokens, rows: int, scale):
    import torch
    _ops.no_tangents("dy", dy)
    dim = dy.shape[-1]
    grad = dy.new_empty((rows, dim))
    if grad.numel():
        ids, dy, n = tokens.contiguous(), dy.contiguous(), tokens.numel()
        work = dy.new_empty(gpu.library().lmz_gpu_rows_grad_work_bytes(n, rows, dim), dtype=torch.uint8)
        _ops.launch(dy.get_device(), "lmz_gpu_rows_grad_dev", dy.data_ptr(), n, dim, _ops.type_code(dy, "dy"), ids.data_ptr(), ids.element_size(), rows, scale,
                    grad.data_ptr(), work.data_ptr())
    return grad


def _function():
    """The autograd function (made on first use: importing this package does not import torch)."""
    global _made
    if _made is None:
        import torch

        class Rows(torch.autograd.Function):
            @staticmethod
            def forward(ctx, table, tokens, scale):
                ctx.save_for_backward(tokens)
                ctx.rows, ctx.scale = table.shape[0], scale
                return _rows(table.get_device(), _ops.type_code(table, "table"), tokens.element_size(), table, tokens, scale)

            @staticmethod
            @_ops.once
            def backward(ctx, dy):
                (tokens,) = ctx.saved_tensors
                return _rows_grad(dy, tokens, ctx.rows, ctx.scale), None, None

        _made = Rows
    return _made


_made = None
