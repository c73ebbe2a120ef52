"""What the Makefile builds, without building it (make -n): the Python binding of the 8-bit calls is an addition where Python's headers are."""
import subprocess
import sys
from pathlib import Path

import pytest

from runner import api

RUNNER = Path(api.__file__).resolve().parent


def commands(*args):
    ret = subprocess.run(["make", "-C", str(RUNNER), "-n", "-B", f"PYTHON={sys.executable}", *args], capture_output=True, text=True)
    assert ret.returncode == 0, ret.stderr
    return ret.stdout


@pytest.mark.parametrize("args", [("PYINC=/nowhere",), ("PYTHON=/nowhere/python",)])
def test_library_and_program_need_no_python_headers(args):
    out = commands(*args)
    assert "sgemm_runner.cpp" in out and "generator_runner.cpp" in out and "sgemm_py.cpp" not in out


def test_binding_is_built_where_the_headers_are(tmp_path):
    (tmp_path / "Python.h").write_text("")
    assert "sgemm_py.cpp" in commands(f"PYINC={tmp_path}")


def test_a_missing_binding_is_built_only_where_it_can_be(monkeypatch, tmp_path):
    calls = []
    monkeypatch.setattr(api.subprocess, "run", lambda *a, **k: calls.append(a))
    present = tmp_path / "present"
    present.write_text("")
    monkeypatch.setattr(api, "LIB_PATH", present)
    monkeypatch.setattr(api, "RUNNER_PATH", present)
    monkeypatch.setattr(api, "NATIVE_PATH", tmp_path / "absent")
    monkeypatch.setattr(api.sysconfig, "get_paths", lambda: {"include": str(tmp_path)})
    api.build_library()
    assert not calls
    (tmp_path / "Python.h").write_text("")
    api.build_library()
    assert len(calls) == 1


def test_the_bindings_name_carries_the_interpreters_tag():
    """A module built for one Python must not be loaded by another: its file is named as import names extension modules."""
    suffix = api.sysconfig.get_config_var("EXT_SUFFIX")
    if not (Path(api.sysconfig.get_paths()["include"]) / "Python.h").exists():
        pytest.skip("Python's headers are not here")
    assert suffix != ".so" and api.NATIVE_PATH.name == "_sgemm_native" + suffix
    assert f"-o ../build/_sgemm_native{suffix} " in commands()
