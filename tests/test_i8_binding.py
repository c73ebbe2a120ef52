"""The Python binding of the 8-bit calls without a GPU and without the library: csrc/sgemm_py.cpp is compiled against a stand-in
(tests/i8_py_seam.cpp) that notes what reaches it.  CPU tensors lie on "device" -1."""
import ctypes
import importlib.util
import subprocess
import sysconfig
import threading
import time
from pathlib import Path

import pytest
import torch

from runner import api

ROOT = Path(__file__).resolve().parent.parent
CSRC = ROOT / "amdgpu-arch-gemm_b200" / "csrc"
A = 1 << 20          # an address; nothing is dereferenced


@pytest.fixture(scope="module")
def seam(tmp_path_factory):
    include = sysconfig.get_paths()["include"]
    if not (Path(include) / "Python.h").exists():
        pytest.skip("Python's headers are not here")
    out = tmp_path_factory.mktemp("binding") / "_sgemm_native.so"
    subprocess.run(["g++", "-O1", "-std=c++17", "-fPIC", "-shared", "-Wall", "-Wextra", f"-I{ROOT / 'include'}", f"-I{include}", "-o", str(out),
                    str(Path(__file__).parent / "i8_py_seam.cpp"), str(CSRC / "sgemm_py.cpp")], check=True)
    spec = importlib.util.spec_from_file_location("_sgemm_native", out)
    module = importlib.util.module_from_spec(spec)
    spec.loader.exec_module(module)
    module.setup(api._type_codes, api._type_code)
    module.state = ctypes.CDLL(str(out))
    return module


def value(seam, name, new=None):
    cell = ctypes.c_int.in_dll(seam.state, name)
    if new is not None:
        cell.value = new
    return cell.value


@pytest.fixture
def r():
    runner = api.SgemmRunner.__new__(api.SgemmRunner)
    runner.device, runner._h = -1, None
    return runner


CALLS = {
    "i8_linear": (A, A, A, A, A, 16, 4, 32, None, 0, 0, 0, 0, 0),
    "i8_quantize": (A, A, A, 32, 4, False, 0, 0, 0, 0),
    "i8_restore": (A, A, A, 32, 4, 0, 0, 0, 0),
    "i8_rmsnorm": (A, A, A, A, 32, 4, None, None, 1e-6, 0, 0, 0, 0, 0, 0),
    "i8_wgrad": (A, A, A, A, 16, 8, 4, None, 1.0, 0.0, 0, 0, 0, 0, 1, 0, 0),
}


@pytest.mark.parametrize("name", CALLS)
def test_other_threads_run_while_a_call_waits(seam, r, name):
    """A launch that waits for room in the queue must not hold back the thread whose host callback makes room."""
    value(seam, "seam_flag", 0)
    value(seam, "seam_wait", 1)

    def release():
        time.sleep(0.02)
        value(seam, "seam_flag", 1)

    other = threading.Thread(target=release)
    other.start()
    try:
        assert getattr(seam, name)(r, 0, -1, *CALLS[name]) == 0
    finally:
        other.join()
        value(seam, "seam_wait", 0)
