"""Rules of the operators' kernels that are plain arithmetic, checked on the CPU."""
import os
import shutil
import subprocess

import pytest

HERE = os.path.dirname(os.path.abspath(__file__))


def _compiled(tmp_path_factory, name):
    cxx = shutil.which("g++")
    if cxx is None:
        pytest.skip("no C++ compiler")
    exe = str(tmp_path_factory.mktemp("native") / name)
    subprocess.run([cxx, "-std=c++17", "-O1", "-g", "-I", os.path.join(HERE, "native"), "-o", exe, os.path.join(HERE, "native", name + ".cc")], check=True)
    return exe


def test_slots_between_a_projections_warps(tmp_path_factory):
    """Under every schedule the warps that fill slots and those that empty them get to their end."""
    done = subprocess.run([_compiled(tmp_path_factory, "slot_ring_check")], capture_output=True, text=True, timeout=120)
    assert done.returncode == 0, done.stderr


def test_a_merges_shared_memory(tmp_path_factory):
    """No rank takes more than the kernel is given leave for."""
    done = subprocess.run([_compiled(tmp_path_factory, "merge_layout_check")], capture_output=True, text=True, timeout=60)
    assert done.returncode == 0, done.stderr


def test_a_wait_that_ran_out_is_told_once(tmp_path_factory):
    """Whichever stream it was on, and to the check that follows it alone."""
    done = subprocess.run([_compiled(tmp_path_factory, "gave_up_check")], capture_output=True, text=True, timeout=60)
    assert done.returncode == 0, done.stderr
