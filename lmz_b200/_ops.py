"""ctypes view of the operators on a checkpoint's tensors (include/lmz_b200.h, section 3), and what their Python
layers share."""
from __future__ import annotations

import ctypes
import math

from . import gpu

_v, _u64, _u32, _int = ctypes.c_void_p, ctypes.c_uint64, ctypes.c_uint32, ctypes.c_int
BF16, F16, F32, E4M3 = 0, 1, 2, 3


class Projection(ctypes.Structure):
    """Mirror of `lmz_projection`."""
    _fields_ = [(n, _v) for n in ("x", "weight", "a", "b", "index", "scales", "y", "hidden", "dy", "dx", "da", "db", "work")] + \
        [(n, _u64) for n in ("tokens", "in_", "out", "x_stride", "weight_stride")] + \
        [(n, _u32) for n in ("adapters", "rank", "dtype", "index_bytes")] + [("scale", ctypes.c_float)]


class Norm(ctypes.Structure):
    """Mirror of `lmz_norm`."""
    _fields_ = [(n, _v) for n in ("x", "residual", "weight", "y", "q", "scale", "stream", "rstd", "dy", "dstream", "dx", "dweight", "work")] + \
        [(n, _u64) for n in ("tokens", "dim", "x_stride", "residual_stride")] + [("dtype", _u32), ("weight_dtype", _u32), ("eps", ctypes.c_float)]


class Product(ctypes.Structure):
    """Mirror of `lmz_product`."""
    _fields_ = [(n, _v) for n in ("x", "weight", "bias", "times", "residual", "offsets", "x_scale", "weight_scale", "y", "z", "dy", "dx", "dweight", "dbias", "dtimes", "work")] + \
        [(n, _u64) for n in ("rows", "in_", "out", "x_stride", "weight_stride", "weight_plane", "times_stride", "residual_stride")] + \
        [(n, _u32) for n in ("experts", "dtype", "result_dtype", "activation", "offset_bytes")]


def bind(lib) -> None:
    proj, norm, product = ctypes.POINTER(Projection), ctypes.POINTER(Norm), ctypes.POINTER(Product)
    for name, res, args in (
            ("lmz_gpu_rows_dev", _int, [_v, _u64, _u64, _u64, _int, _v, _int, _u64, ctypes.c_float, _v, _v]),
            ("lmz_gpu_rows_grad_work_bytes", ctypes.c_size_t, [_u64] * 3),
            ("lmz_gpu_rows_grad_dev", _int, [_v, _u64, _u64, _int, _v, _int, _u64, ctypes.c_float, _v, _v, _v]),
            ("lmz_gpu_project_hidden_bytes", ctypes.c_size_t, [proj]),
            ("lmz_gpu_project_work_bytes", ctypes.c_size_t, [proj, _int]),
            ("lmz_gpu_project_dev", _int, [proj, _v]),
            ("lmz_gpu_project_grad_dev", _int, [proj, _v]),
            ("lmz_gpu_norm_dev", _int, [norm, _v]),
            ("lmz_gpu_norm_grad_work_bytes", ctypes.c_size_t, [norm]),
            ("lmz_gpu_norm_grad_dev", _int, [norm, _v]),
            ("lmz_gpu_product_work_bytes", ctypes.c_size_t, [product, _int]),
            ("lmz_gpu_product_z_bytes", ctypes.c_size_t, [product]),
            ("lmz_gpu_product_dev", _int, [product, _v]),
            ("lmz_gpu_product_grad_dev", _int, [product, _v]),
            ("lmz_gpu_order_work_bytes", ctypes.c_size_t, [_u64]),
            ("lmz_gpu_order_dev", _int, [_v, _int, _u64, _u64, _v, _v, _v, _v]),
            ("lmz_gpu_ops_gave_up", _int, []),
            ("lmz_gpu_merge_dev", _int, [_v, _u64, _u64, _u64, _v, _v, ctypes.c_uint, ctypes.c_float, _int, _v, _v]),
            ("lmz_gpu_merge_wide_dev", _int, [_v, _u64, _u64, _u64, _v, _v, ctypes.c_uint, ctypes.c_float, _int, _v, _v])):
        fn = getattr(lib, name)
        fn.restype, fn.argtypes = res, args


_codes = {}


def _known():
    """Element types by the library's numbers (filled on first use: importing this package does not import torch)."""
    import torch
    _codes.update({torch.bfloat16: BF16, torch.float16: F16, torch.float32: F32})
    return _codes


def type_code(t, what: str, half_only: bool = False) -> int:
    """The library's number for a tensor's element type, or a TypeError."""
    code = (_codes or _known()).get(t.dtype)
    if code is None or (half_only and code == F32):
        raise TypeError(f"{what} must be {'bfloat16 or float16' if half_only else 'bfloat16, float16 or float32'}, not {t.dtype}")
    return code


def on_cuda(names: str, *tensors) -> int:
    """The index of the CUDA device that all given tensors are on (None for one that is not given), or an error that names
    who is not.  `names`: the tensors', by spaces.  Tensors with a forward-mode tangent are refused."""
    no_tangents(names, *tensors)
    device = None
    for t in tensors:
        if t is None:
            continue
        try:
            d = t.get_device()
        except AttributeError:
            d = -1
        if device is None:
            device = d
        if d < 0 or d != device:
            _refuse_place(names.split(), tensors)
    return device


_forward_mode = None


def no_tangents(names: str, *tensors) -> None:
    """The operators have gradients, but no forward-mode derivatives: a tangent would be lost without a word."""
    global _forward_mode
    if _forward_mode is None:
        from torch.autograd import forward_ad
        _forward_mode = forward_ad
    if _forward_mode._current_level < 0:                   # (nobody has made a dual tensor)
        return
    import torch
    for name, t in zip(names.split(), tensors):
        if isinstance(t, torch.Tensor) and _forward_mode.unpack_dual(t).tangent is not None:
            raise NotImplementedError(f"{name} has a tangent: this operator has no forward-mode derivative")


def _refuse_place(names, tensors):
    import torch
    device = None
    for name, t in zip(names, tensors):
        if t is None:
            continue
        if not isinstance(t, torch.Tensor):
            raise TypeError(f"{name} must be a torch tensor, not {type(t).__name__}")
        if not t.is_cuda:
            raise ValueError(f"{name} must be a CUDA tensor")
        if device is not None and t.device != device:
            raise ValueError(f"{name} is on {t.device}, the tensors before it on {device}")
        device = t.device


def whole_numbers(t, what: str) -> int:
    """Bytes of an id: int32 and int64 are taken."""
    import torch
    if t.dtype is not torch.int32 and t.dtype is not torch.int64:
        raise TypeError(f"{what} must be int32 or int64, not {t.dtype}")
    return 4 if t.dtype is torch.int32 else 8


def rows_of(t):
    """A tensor as [rows, columns] with the elements of a row next to each other, without a copy where it can be."""
    if t is None:
        return None
    if t.dim() != 2:
        t = t.reshape(-1, t.shape[-1])
    return t if t.stride(1) == 1 or t.shape[1] == 1 else t.contiguous()


def address(t):
    return None if t is None else t.data_ptr()


def trained(*tensors) -> bool:
    """Whether one of the tensors (None for one that is not given) wants a gradient."""
    for t in tensors:
        if t is not None and t.requires_grad:
            return True
    return False


def same_type(dtype, whose: str, **tensors) -> None:
    """A TypeError for the first of the tensors (None for one that is not given) of another type."""
    for name, t in tensors.items():
        if t is not None and t.dtype is not dtype:
            raise TypeError(f"{name} is {t.dtype}, but {whose} {dtype}")


def empty_like(t, dtype=None):
    """A contiguous tensor of the same shape."""
    import torch
    return torch.empty_like(t, dtype=dtype) if t.is_contiguous() else t.new_empty(t.shape, dtype=dtype)


def packed(t):
    return t if t is None or t.is_contiguous() else t.contiguous()


def finite(scale, what: str = "scale") -> float:
    scale = float(scale)
    if not math.isfinite(scale):
        raise ValueError(f"{what} must be finite")
    return scale


def once(backward):
    """A backward pass that has no gradient of its own: as torch's `once_differentiable`, without its cost where nobody asked
    for a graph of the gradients."""
    wrapped = None

    def run(ctx, *grads):
        nonlocal wrapped
        import torch
        if not torch.is_grad_enabled():
            return backward(ctx, *grads)
        if wrapped is None:
            from torch.autograd.function import once_differentiable
            wrapped = once_differentiable(backward)
        return wrapped(ctx, *grads)

    return run


def stream_of(index: int) -> int:
    """The device's current stream, as the library takes it."""
    import torch
    return torch._C._cuda_getCurrentRawStream(index)


_entries = {}


def launch(index: int, name: str, *args) -> None:
    """Call an entry point on the device's current stream (its last argument)."""
    import torch
    fn = _entries.get(name)
    if fn is None:
        fn = _entries[name] = getattr(gpu.library(), name)
    c = torch._C
    if c._cuda_getDevice() == index:
        rc = fn(*args, c._cuda_getCurrentRawStream(index))
    else:
        with torch.cuda.device(index):
            rc = fn(*args, c._cuda_getCurrentRawStream(index))
    if rc == 0:
        return
    if rc == gpu.EUNSUPPORTED:
        raise ValueError(gpu.last_error())
    raise RuntimeError(f"{name} failed ({rc}): {gpu.last_error()}")
