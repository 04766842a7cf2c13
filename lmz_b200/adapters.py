"""Low-rank adapters: many fine-tunes of one base checkpoint, each a pair of thin factors beside a shared weight.

`project` runs the shared projection of a batch whose tokens belong to different adapters, and its gradients; `merge`
makes a fine-tune's own weight out of base and adapter; `load` takes the factors out of adapter archives.
`decode.decode_tensors(..., adapter=...)` restores merged weights straight from a base archive and an adapter's.
"""
from __future__ import annotations

from . import _ops, gpu

MAX_RANK = 256


def project(x, weight, a, b, index=None, scale=1.0):
    """`x @ weight.T + s_i * (x @ a_i.T) @ b_i.T`, where every token of x has an adapter i of its own.

    `x`: [..., in], `weight`: [out, in] (frozen: it gets no gradient), `a`: [adapters, rank, in], `b`: [adapters, out, rank],
    all bfloat16 or all float16.  One adapter alone may be given as `a` [rank, in] and `b` [out, rank].  `index`: int32 or int64
    of x's leading shape, the adapter of each token; a token whose index is outside [0, adapters) has none, and without an
    index all tokens have adapter 0.  `scale`: a number, or a float32 tensor of one per adapter (alpha / rank).  Adapters of
    lower rank are padded with zeros.  Ranks go up to 256.  Tokens of one adapter next to each other are fastest.

    Returns [..., out], summed in 32 bits and rounded once; what comes of a_i goes to b_i with 16 bits or more (an error of 2^-16
    of its magnitude), over float32's range whatever the tensors' type.  An adapter's values, infinities and NaN among them, reach only
    its own tokens.  Differentiable once in x, a and b; gradients of a and b sum over each adapter's tokens, with zeros for
    an adapter that none has, and are the same in every run."""
    import torch
    _ops.on_cuda("x weight a b index", x, weight, a, b, index)
    code = _ops.type_code(x, "x", half_only=True)
    if weight.dtype is not x.dtype or a.dtype is not x.dtype or b.dtype is not x.dtype:
        raise TypeError(f"weight is {weight.dtype}, a {a.dtype} and b {b.dtype}, but x {x.dtype}")
    if weight.dim() != 2 or x.dim() < 1:
        raise ValueError(f"weight must be [out, in] and x [..., in], not {list(weight.shape)} and {list(x.shape)}")
    if a.dim() == 2 and b.dim() == 2:
        a, b = a.unsqueeze(0), b.unsqueeze(0)
    out, inp = weight.shape
    *lead, columns = x.shape
    n, rank, width = a.shape if a.dim() == 3 else (0, 0, 0)
    if columns != inp or width != inp or a.dim() != 3 or b.shape != (n, out, rank):
        raise ValueError(f"x {list(x.shape)}, weight {list(weight.shape)}, a {list(a.shape)} and b {list(b.shape)} do not fit "
                         "[..., in], [out, in], [adapters, rank, in] and [adapters, out, rank]")
    if weight.stride(1) != 1 and inp > 1:
        raise ValueError("the elements of a row of the weight must be next to each other")
    if not n or not inp or not out or not 1 <= rank <= MAX_RANK:
        raise ValueError(f"no adapter, an empty weight, or a rank outside 1..{MAX_RANK}")
    if index is not None:
        _ops.whole_numbers(index, "index")
        if [*index.shape] != lead:
            raise ValueError(f"index is {list(index.shape)}, x has tokens {lead}")
    scales = None
    if isinstance(scale, torch.Tensor):
        scales, scale = scale, 1.0
        _ops.on_cuda("x scale", x, scales)
        if scales.dtype is not torch.float32 or scales.shape != a.shape[:1]:
            raise ValueError(f"scale must be a number or float32 [{a.shape[0]}], not {scales.dtype} {list(scales.shape)}")
    else:
        scale = _ops.finite(scale)
    if torch.is_grad_enabled() and (x.requires_grad or a.requires_grad or b.requires_grad or weight.requires_grad or
                                    (scales is not None and scales.requires_grad)):
        if weight.requires_grad or (scales is not None and scales.requires_grad):
            raise ValueError("weight and scale are not trained beside an adapter: they must not require a gradient")
        return _function().apply(x, weight, a, b, index, scales, scale)
    return _forward(code, x, weight, a, b, index, scales, scale, False)[0]


def _flat(x):
    """x as [tokens, in] with the elements of a row next to each other, without a copy where it can be."""
    if x.dim() != 2:
        x = x.reshape(-1, x.shape[-1])
    return x if x.stride(1) == 1 or x.shape[1] == 1 else x.contiguous()


def _packed(t):
    return t if t is None or t.is_contiguous() else t.contiguous()


def _call(code, x, weight, a, b, index, scales, scale):
    (tokens, inp), (n, rank, _) = x.shape, a.shape
    return _ops.Projection(x.data_ptr(), weight.data_ptr(), a.data_ptr(), b.data_ptr(), None if index is None else index.data_ptr(),
                           None if scales is None else scales.data_ptr(), None, None, None, None, None, None, None, tokens, inp, weight.shape[0], x.stride(0),
                           weight.stride(0), n, rank, code, 0 if index is None else index.element_size(), scale)


def _run(name: str, grad: int, p, x):
    import torch
    size = gpu.library().lmz_gpu_project_work_bytes(p, grad)
    if size:
        work = x.new_empty(size, dtype=torch.uint8)
        p.work = work.data_ptr()
    _ops.launch(x.get_device(), name, p)


def _forward(code, x, weight, a, b, index, scales, scale, keep):
    """y, and what the gradients need of it if `keep`."""
    y = x.new_empty((*x.shape[:-1], weight.shape[0]))
    x, a, b, index, scales = _flat(x), _packed(a), _packed(b), _packed(index), _packed(scales)
    p, hidden = _call(code, x, weight, a, b, index, scales, scale), None
    p.y = y.data_ptr()
    if keep:
        import torch
        hidden = x.new_empty(gpu.library().lmz_gpu_project_hidden_bytes(p), dtype=torch.uint8)
        p.hidden = hidden.data_ptr()
    _run("lmz_gpu_project_dev", 0, p, x)
    return y, hidden


def _backward(code, dy, x, weight, a, b, index, scales, scale, hidden, wanted):
    _ops.no_tangents("dy", dy)
    dx, da, db = (t.new_empty(t.shape) if w else None for t, w in zip((x, a, b), wanted))
    x, dy = _flat(x), dy.reshape(-1, dy.shape[-1]).contiguous()
    a, b, index, scales = _packed(a), _packed(b), _packed(index), _packed(scales)      # (copies live until the launch)
    p = _call(code, x, weight, a, b, index, scales, scale)
    p.hidden, p.dy = hidden.data_ptr(), dy.data_ptr()
    p.dx, p.da, p.db = (None if t is None else t.data_ptr() for t in (dx, da, db))
    _run("lmz_gpu_project_grad_dev", 1, p, x)
    return dx, da, db


def _function():
    """The autograd function (made on first use: importing this package does not import torch)."""
    global _made
    if _made is None:
        import torch

        class Project(torch.autograd.Function):
            @staticmethod
            def forward(ctx, x, weight, a, b, index, scales, scale):
                code = _ops.type_code(x, "x", half_only=True)
                y, hidden = _forward(code, x, weight, a, b, index, scales, scale, True)
                ctx.save_for_backward(x, weight, a, b, index, scales, hidden)
                ctx.code, ctx.scale = code, scale
                return y

            @staticmethod
            @_ops.once
            def backward(ctx, dy):
                x, weight, a, b, index, scales, hidden = ctx.saved_tensors
                wanted = (ctx.needs_input_grad[0], ctx.needs_input_grad[2], ctx.needs_input_grad[3])
                dx, da, db = _backward(ctx.code, dy, x, weight, a, b, index, scales, ctx.scale, hidden, wanted)
                return dx, None, da, db, None, None, None

        _made = Project
    return _made


_made = None


def merge(weight, a, b, scale: float = 1.0, out=None):
    """`weight + scale * b @ a`, summed in 32 bits and rounded once: the weight of the fine-tune that an adapter is.

    `weight`: [out, in], `a`: [rank, in], `b`: [out, rank], all bfloat16 or all float16, or both factors float32 and the weight any
    of the three.  `out`: a contiguous tensor like the weight to write to, the weight itself among them; without it a new one.  Not differentiable."""
    import torch
    index = _ops.on_cuda("weight a b out", weight, a, b, out)
    code = _ops.type_code(weight, "weight")
    wide = a.dtype == torch.float32
    if a.dtype != b.dtype or not (wide or (a.dtype == weight.dtype)):
        raise TypeError(f"a is {a.dtype} and b {b.dtype}, the weight {weight.dtype}: the factors must be of its type, or float32")
    if weight.dim() != 2 or a.dim() != 2 or b.dim() != 2 or a.shape[1] != weight.shape[1] or b.shape[0] != weight.shape[0] or \
            a.shape[0] != b.shape[1]:
        raise ValueError(f"weight {list(weight.shape)}, a {list(a.shape)} and b {list(b.shape)} do not fit [out, in], [rank, in] and [out, rank]")
    if weight.stride(1) != 1 and weight.shape[1] > 1:
        raise ValueError("the elements of a row of the weight must be next to each other")
    if not 1 <= a.shape[0] <= MAX_RANK:
        raise ValueError(f"a rank outside 1..{MAX_RANK}")
    scale = _ops.finite(scale)
    if torch.is_grad_enabled() and any(t is not None and t.requires_grad for t in (weight, a, b, out)):
        raise ValueError("merge has no gradient: call it under torch.no_grad()")
    given = out is not None
    if not given:
        out = torch.empty(weight.shape, dtype=weight.dtype, device=weight.device)
    elif out.shape != weight.shape or out.dtype != weight.dtype or not out.is_contiguous():
        raise ValueError("out must be a contiguous tensor of the weight's shape and type")
    elif not _apart(out, a) or not _apart(out, b) or not (_apart(out, weight) or (out.data_ptr() == weight.data_ptr() and weight.is_contiguous())):
        raise ValueError("out may be the weight itself, but not overlap a, b or a part of the weight")
    if out.numel():
        a, b = _packed(a), _packed(b)
        _ops.launch(index, "lmz_gpu_merge_wide_dev" if wide else "lmz_gpu_merge_dev", weight.data_ptr(), weight.shape[0], weight.shape[1], weight.stride(0), a.data_ptr(), b.data_ptr(),
                    a.shape[0], scale, code, out.data_ptr())
        if given:                                          # (autograd notices where what was there is still needed)
            torch.autograd.graph.increment_version(out)
    return out


def check(device=None) -> None:
    """Synchronise the device, and raise if a kernel has given up waiting for one of its own copies there since the last
    check (every wait in them has a limit; none runs out unless the hardware fails).  What was computed since then is not to
    be used; calls after it are not touched by it."""
    import torch
    with torch.cuda.device(device if device is not None else torch.cuda.current_device()):
        rc = gpu.library().lmz_gpu_ops_gave_up()
    if rc:
        raise RuntimeError("a projection's kernel gave up waiting: its results are not to be used" if rc > 0 else gpu.last_error())


def _span(t):
    """The bytes from a tensor's first element to the end of its last."""
    lo = t.data_ptr()
    return lo, lo + (sum((n - 1) * s for n, s in zip(t.shape, t.stride())) + 1) * t.element_size() if t.numel() else lo


def _apart(t, u) -> bool:
    (a, b), (c, d) = _span(t), _span(u)
    return b <= c or d <= a


def load(archives, name: str, device=None, dtype=None):
    """(a, b): the factors that several adapters have for one weight, stacked for `project`.

    `archives`: an archive (or path, or bytes) per adapter.  `name`: the weight's name, as in the base checkpoint; an
    adapter's factors are the tensors whose names end in `<name without .weight>.lora_A.weight` and `...lora_B.weight`.  Adapters
    of lower rank are padded with zeros; one without factors for this weight gets zeros.  `dtype`: what to convert the
    factors to (they are all of one type where it is not given)."""
    import torch
    pairs = [_factors(ar, name, device) for ar in archives]
    have = [p for p in pairs if p is not None]
    if not have:
        raise KeyError(f"no archive has an adapter for {name!r}")
    if dtype is None and len({t.dtype for p in have for t in p}) > 1:
        raise TypeError("the adapters are of different types: give the dtype to convert them to")
    dtype = dtype or have[0][0].dtype
    rank, (_, inp), (out, _) = max(p[0].shape[0] for p in have), have[0][0].shape, have[0][1].shape
    a = torch.zeros((len(pairs), rank, inp), dtype=dtype, device=have[0][0].device)
    b = torch.zeros((len(pairs), out, rank), dtype=dtype, device=have[0][0].device)
    for i, p in enumerate(pairs):
        if p is None:
            continue
        if p[0].shape[1] != inp or p[1].shape[0] != out:
            raise ValueError(f"adapter {i} has factors {list(p[0].shape)} and {list(p[1].shape)} for {name!r}, another has [.., {inp}] and [{out}, ..]")
        a[i, :p[0].shape[0]] = p[0]
        b[i, :, :p[0].shape[0]] = p[1]
    return a, b


def _factors(ar, name: str, device=None):
    """(a, b) of one adapter archive for a weight, or None if it has none."""
    from . import archive as fmt, decode
    ar = ar if isinstance(ar, fmt.Archive) else fmt.Archive(ar)
    stem = name[:-len(".weight")] if name.endswith(".weight") else name
    found = []
    for part in ("lora_A", "lora_B"):
        end = f"{stem}.{part}.weight"
        keys = [k for k in ar.tensor_index() if k[1] == end or k[1].endswith("." + end)]
        if len(keys) > 1:
            raise KeyError(f"{len(keys)} tensors of the adapter end in {end!r}")
        found += keys
    if not found:
        return None
    if len(found) == 1:
        raise KeyError(f"the adapter has only one factor for {name!r}: {found[0][1]!r}")
    got = decode.decode_tensors(ar, found, device=device)
    a, b = (decode._typed(got[k], ar.tensor_index()[k]) for k in found)
    if a.dim() != 2 or b.dim() != 2 or a.shape[0] != b.shape[1]:
        raise ValueError(f"the factors for {name!r} are {list(a.shape)} and {list(b.shape)}, not [rank, in] and [out, rank]")
    return a, b
