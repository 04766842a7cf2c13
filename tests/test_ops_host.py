"""Operators on a checkpoint's tensors: what can be said of them without a GPU."""
import ctypes
import os
import re
import subprocess
import sys

import numpy as np
import pytest
import torch

from lmz_b200 import _ops, adapters, build, embed

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))


@pytest.fixture(scope="module")
def lib():
    path = build.build()
    assert path, build.last_error
    lib = ctypes.CDLL(path)
    _ops.bind(lib)
    lib.lmz_gpu_last_error.restype = ctypes.c_char_p
    return lib


def test_projection_mirrors_the_header(tmp_path):
    names = [n for n, _ in _ops.Projection._fields_]
    c = "#include <stdio.h>\n#include \"lmz_b200.h\"\nint main(void) {\n" + "".join(
        f'printf("%zu\\n", offsetof(lmz_projection, {n.rstrip("_")}));\n' for n in names) + 'printf("%zu\\n", sizeof(lmz_projection)); return 0; }\n'
    src = tmp_path / "layout.c"
    src.write_text(c)
    exe = tmp_path / "layout"
    subprocess.run(["gcc", "-I", os.path.join(ROOT, "include"), "-o", str(exe), str(src)], check=True)
    said = [int(v) for v in subprocess.run([str(exe)], capture_output=True, text=True, check=True).stdout.split()]
    assert said == [getattr(_ops.Projection, n).offset for n in names] + [ctypes.sizeof(_ops.Projection)]


def test_numbers_of_the_header():
    text = open(os.path.join(ROOT, "include", "lmz_b200.h")).read()
    said = {k: int(v) for k, v in re.findall(r"#define LMZ_GPU_(BF16|F16|F32|MAX_RANK) (\d+)", text)}
    assert said == {"BF16": _ops.BF16, "F16": _ops.F16, "F32": _ops.F32, "MAX_RANK": adapters.MAX_RANK}


def _projection(**kw):
    p = _ops.Projection()
    p.tokens, p.in_, p.out, p.x_stride, p.weight_stride, p.adapters, p.rank, p.dtype = 4, 64, 64, 64, 64, 1, 8, _ops.BF16
    for k, v in kw.items():
        setattr(p, k, v)
    return p


@pytest.mark.parametrize("bad", [dict(dtype=_ops.F32), dict(dtype=9), dict(rank=0), dict(rank=257), dict(adapters=0), dict(adapters=1 << 16),
                                 dict(in_=0), dict(out=0), dict(in_=1 << 21), dict(out=1 << 21), dict(tokens=1 << 31), dict(index=64, index_bytes=2)])
def test_projections_the_library_refuses(lib, bad):
    p = _projection(**bad)
    assert lib.lmz_gpu_project_dev(p, None) == -2
    assert lib.lmz_gpu_last_error()
    assert lib.lmz_gpu_project_grad_dev(p, None) == -2


@pytest.mark.parametrize("rows, dim, dtype, id_bytes, n", [(10, 0, 0, 4, 1), (10, 1 << 24, 0, 4, 1), (1 << 31, 8, 0, 4, 1), (10, 8, 3, 4, 1),
                                                           (10, 8, 0, 2, 1), (10, 8, 0, 8, 1 << 31)])
def test_rows_the_library_refuses(lib, rows, dim, dtype, id_bytes, n):
    assert lib.lmz_gpu_rows_dev(None, rows, dim, dim, dtype, None, id_bytes, n, 1.0, None, None) == -2
    assert lib.lmz_gpu_rows_grad_dev(None, n, dim, dtype, None, id_bytes, rows, 1.0, None, None, None) == -2


@pytest.mark.parametrize("out, inp, rank, dtype", [(8, 8, 0, 0), (8, 8, 257, 0), (8, 8, 4, 2), (0, 8, 4, 0), (8, 1 << 21, 4, 0)])
def test_merges_the_library_refuses(lib, out, inp, rank, dtype):
    assert lib.lmz_gpu_merge_dev(None, out, inp, inp, None, None, rank, 1.0, dtype, None, None) == -2


@pytest.mark.parametrize("index", [None, 64])
@pytest.mark.parametrize("tokens", [4, 5000])
def test_workspaces_do_not_depend_on_the_gradients_wanted(lib, index, tokens):
    p = _projection(tokens=tokens, in_=1024, out=1024, x_stride=1024, weight_stride=1024, adapters=7, index=index, index_bytes=4, rank=16)
    size = lib.lmz_gpu_project_work_bytes(p, 1)
    for name in ("dx", "da", "db"):
        p.dx = p.da = p.db = None
        setattr(p, name, 4096)
        assert lib.lmz_gpu_project_work_bytes(p, 1) == size
    assert lib.lmz_gpu_project_work_bytes(p, 0) >= 4 * tokens * 16      # (the thin product)


def test_nothing_to_do_needs_no_gpu(lib):
    assert lib.lmz_gpu_rows_dev(None, 10, 8, 8, 0, None, 4, 0, 1.0, None, None) == 0
    assert lib.lmz_gpu_project_dev(_projection(tokens=0), None) == 0
    assert lib.lmz_gpu_rows_grad_dev(None, 5, 8, 0, None, 4, 0, 1.0, None, None, None) == 0


def test_work_sizes(lib):
    """Room for sorted ids twice, and for two sums per window of tokens."""
    for n, rows, dim in ((1, 10, 8), (5000, 128256, 4096), (1 << 20, 1000, 4096)):
        got = lib.lmz_gpu_rows_grad_work_bytes(n, rows, dim)
        window = -(-max(32, -(-n // 4096)) // 32) * 32
        partial = -(-n // window) * 2 * dim * 4 if n > window else 0
        least = 16 * n + partial
        assert least <= got <= least + 6 * 256


def test_cpu_tensors_are_refused():
    t = torch.zeros((4, 8), dtype=torch.bfloat16)
    with pytest.raises(ValueError, match="CUDA"):
        embed.lookup(t, torch.zeros(3, dtype=torch.int64))
    with pytest.raises(ValueError, match="CUDA"):
        adapters.project(t, t, t, t)
    with pytest.raises(ValueError, match="CUDA"):
        adapters.merge(t, t, t)
    with pytest.raises(TypeError, match="torch tensor"):
        embed.lookup(np.zeros((4, 8)), t)


def test_importing_the_package_imports_no_torch():
    code = "import sys, lmz_b200.embed, lmz_b200.adapters; sys.exit('torch' in sys.modules)"
    assert subprocess.run([sys.executable, "-c", code], cwd=ROOT).returncode == 0


def test_spans_of_strided_tensors():
    t = torch.zeros(100, dtype=torch.float16)
    w = t.as_strided((3, 4), (10, 1))
    lo, hi = adapters._span(w)
    assert (lo, hi) == (t.data_ptr(), t.data_ptr() + 48)
    assert adapters._apart(w, t[24:]) and not adapters._apart(w, t[23:])
