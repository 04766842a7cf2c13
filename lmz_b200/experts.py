"""Products of rows with the weights of their experts: a layer in which every token goes through a few of many weights.

`sort` brings what a router chose into the experts' order; `project` runs the rows of every expert through its weight, all in one launch and
without the host knowing how many rows each has.

    order, offsets = experts.sort(chosen, weight.shape[0])                  # chosen: [tokens, k] expert ids
    rows = embed.lookup(x, order // chosen.shape[1])                       # a token's row for each expert it goes to
    y = experts.project(rows, weight, offsets)
"""
from __future__ import annotations

from . import _ops, gpu, linear

MAX_EXPERTS = 1024


def sort(index, experts: int):
    """`(order, offsets)`: the places of `index` (int32 or int64, of any shape, taken as one row) in the order of their experts, those of
    one expert in their own order, and where each expert's begin: int32 `[index.numel()]` and `[experts + 1]`.  Places whose index is outside
    [0, experts) come last, behind `offsets[experts]`."""
    import torch
    device = _ops.on_cuda("index", index)
    id_bytes = _ops.whole_numbers(index, "index")
    if not 1 <= experts <= MAX_EXPERTS:
        raise ValueError(f"between 1 and {MAX_EXPERTS} experts, not {experts}")
    ids, n = _ops.packed(index), index.numel()
    order, offsets = ids.new_empty(n, dtype=torch.int32), ids.new_empty(experts + 1, dtype=torch.int32)
    work = ids.new_empty(gpu.library().lmz_gpu_order_work_bytes(n), dtype=torch.uint8)
    _ops.launch(device, "lmz_gpu_order_dev", ids.data_ptr(), id_bytes, n, experts, order.data_ptr(), offsets.data_ptr(), work.data_ptr())
    return order, offsets


def project(x, weight, offsets, bias=None, activation=None, times=None):
    """`act(x[t] @ weight[e].T + bias[e]) * times[t]` for the rows t of every expert e: `offsets[e] <= t < offsets[e + 1]`.

    `x`: [rows, in], `weight`: [experts, out, in], `bias`: [experts, out], `times`: [rows, out], all bfloat16 or all float16.  `offsets`: int32 or
    int64 [experts + 1], on the device (as `sort` returns them), ascending; an offset below one before it, or outside [0, rows], counts as the nearest that is
    not.  Rows of no expert give zeros, take part in no gradient and get zeros for theirs.  `activation`: as for `linear.project`.

    Returns [rows, out], worked out in 32 bits and rounded once.  Differentiable once, in x, weight, bias and times, with zeros for an
    expert without rows; gradients are the same in every run."""
    import torch
    index = _ops.on_cuda("x weight offsets bias times", x, weight, offsets, bias, times)
    code = _ops.type_code(x, "x", half_only=True)
    _ops.same_type(x.dtype, "x", weight=weight, bias=bias, times=times)
    _ops.whole_numbers(offsets, "offsets")
    kind = linear._activation(activation)
    if x.dim() != 2 or weight.dim() != 3 or x.shape[1] != weight.shape[2]:
        raise ValueError(f"x {list(x.shape)} and weight {list(weight.shape)} do not fit [rows, in] and [experts, out, in]")
    experts, out, inp = weight.shape
    if not out or not inp or not 1 <= experts <= MAX_EXPERTS:
        raise ValueError(f"an empty weight, or not between 1 and {MAX_EXPERTS} experts")
    if weight.stride(2) != 1 and inp > 1:
        raise ValueError("the elements of a row of the weight must be next to each other")
    if offsets.shape != (experts + 1,):
        raise ValueError(f"offsets must be [{experts + 1}], not {list(offsets.shape)}")
    if bias is not None and bias.shape != (experts, out):
        raise ValueError(f"bias must be {[experts, out]}, not {list(bias.shape)}")
    if times is not None and times.shape != (x.shape[0], out):
        raise ValueError(f"times must be {[x.shape[0], out]}, not {list(times.shape)}")
    if torch.is_grad_enabled() and _ops.trained(x, weight, bias, times):
        return linear._function().apply(x, weight, bias, times, None, offsets, kind)
    return linear._forward(index, code, code, kind, x, weight, bias, times, None, offsets, None, None, False)[0]
