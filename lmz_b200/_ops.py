"""ctypes view of the operators on a checkpoint's tensors (include/lmz_b200.h, section 3), and what their Python
layers share."""
from __future__ import annotations

import ctypes

from . import gpu

_v, _u64, _u32, _int = ctypes.c_void_p, ctypes.c_uint64, ctypes.c_uint32, ctypes.c_int
BF16, F16, F32 = 0, 1, 2


class Projection(ctypes.Structure):
    """Mirror of `lmz_projection`."""
    _fields_ = [(n, _v) for n in ("x", "weight", "a", "b", "index", "scales", "y", "hidden", "dy", "dx", "da", "db", "work")] + \
        [(n, _u64) for n in ("tokens", "in_", "out", "x_stride", "weight_stride")] + \
        [(n, _u32) for n in ("adapters", "rank", "dtype", "index_bytes")] + [("scale", ctypes.c_float)]


def bind(lib) -> None:
    proj = ctypes.POINTER(Projection)
    for name, res, args in (
            ("lmz_gpu_rows_dev", _int, [_v, _u64, _u64, _u64, _int, _v, _int, _u64, ctypes.c_float, _v, _v]),
            ("lmz_gpu_rows_grad_work_bytes", ctypes.c_size_t, [_u64] * 3),
            ("lmz_gpu_rows_grad_dev", _int, [_v, _u64, _u64, _int, _v, _int, _u64, ctypes.c_float, _v, _v, _v]),
            ("lmz_gpu_project_hidden_bytes", ctypes.c_size_t, [proj]),
            ("lmz_gpu_project_work_bytes", ctypes.c_size_t, [proj, _int]),
            ("lmz_gpu_project_dev", _int, [proj, _v]),
            ("lmz_gpu_project_grad_dev", _int, [proj, _v]),
            ("lmz_gpu_ops_gave_up", _int, []),
            ("lmz_gpu_merge_dev", _int, [_v, _u64, _u64, _u64, _v, _v, ctypes.c_uint, ctypes.c_float, _int, _v, _v])):
        fn = getattr(lib, name)
        fn.restype, fn.argtypes = res, args


def type_code(t, what: str, half_only: bool = False) -> int:
    """The library's number for a tensor's element type, or a TypeError."""
    import torch
    code = {torch.bfloat16: BF16, torch.float16: F16, torch.float32: F32}.get(t.dtype)
    if code is None or (half_only and code == F32):
        raise TypeError(f"{what} must be {'bfloat16 or float16' if half_only else 'bfloat16, float16 or float32'}, not {t.dtype}")
    return code


def on_cuda(**tensors):
    """The CUDA device that all given tensors are on (None for one that is not given), or an error that names who is not."""
    import torch
    device = None
    for name, t in tensors.items():
        if t is None:
            continue
        if not isinstance(t, torch.Tensor):
            raise TypeError(f"{name} must be a torch tensor, not {type(t).__name__}")
        if not t.is_cuda:
            raise ValueError(f"{name} must be a CUDA tensor")
        if device is None:
            device = t.device
        elif t.device != device:
            raise ValueError(f"{name} is on {t.device}, the tensors before it on {device}")
    return device


def whole_numbers(t, what: str) -> int:
    """Bytes of an id: int32 and int64 are taken."""
    import torch
    if t.dtype not in (torch.int32, torch.int64):
        raise TypeError(f"{what} must be int32 or int64, not {t.dtype}")
    return t.element_size()


def finite(scale, what: str = "scale") -> float:
    import math
    scale = float(scale)
    if not math.isfinite(scale):
        raise ValueError(f"{what} must be finite")
    return scale


def launch(device, name: str, *args) -> None:
    """Call an entry point on the device's current stream (its last argument)."""
    import torch
    lib = gpu.library()
    if torch.cuda.current_device() == device.index:
        rc = getattr(lib, name)(*args, torch.cuda.current_stream(device).cuda_stream)
    else:
        with torch.cuda.device(device):
            rc = getattr(lib, name)(*args, torch.cuda.current_stream(device).cuda_stream)
    if rc == gpu.EUNSUPPORTED:
        raise ValueError(gpu.last_error())
    if rc != gpu.OK:
        raise RuntimeError(f"{name} failed ({rc}): {gpu.last_error()}")
