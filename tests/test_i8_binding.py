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
    module.setup(api._type_code)
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


def norm(seam, r, x=A, g=A, res=None, total=None, x_type=None):
    return seam.i8_rmsnorm(r, 0, -1, x, g, A, A, 32, 4, res, total, 1e-6, 0, 0, 0, 0, x_type, 0)


def test_a_given_type_holds_for_every_operand_of_that_type(seam, r):
    """x_type beside tensors: gamma, the residual and the sum must have it, or be storage of another kind; so C and dw_type."""
    f, h, raw = torch.zeros(4, 32), torch.zeros(4, 32, dtype=torch.bfloat16), torch.zeros(4, 32, dtype=torch.int16)
    assert norm(seam, r, g=f[0], res=f, total=f, x_type=0) == 0 and norm(seam, r, h, h[0], h, h, x_type=2) == 0
    assert norm(seam, r, raw, raw[0], raw, raw, x_type=2) == 0 and norm(seam, r, h, raw[0], raw, h, x_type=2) == 0
    for code in (0, 1):
        for bad in (dict(x=h), dict(g=h[0]), dict(res=h), dict(total=h)):
            with pytest.raises(TypeError, match="element type"):
                norm(seam, r, **bad, x_type=code)
    for bad in (dict(g=h[0]), dict(res=h), dict(total=h)):       # without one: x's own
        with pytest.raises(TypeError):
            norm(seam, r, x=f, **bad)

    def wgrad(c, dw=A, dw_type=None):
        return seam.i8_wgrad(r, 0, -1, A, A, A, dw, 32, 4, 8, c, 1.0, 1.0, 0, 0, 0, 0, 2, dw_type, 0)

    assert wgrad(h, dw_type=2) == 0 and wgrad(h, h) == 0 and wgrad(raw, h, 2) == 0
    for code in (0, 1):
        with pytest.raises(TypeError, match="element type"):
            wgrad(h, dw_type=code)
    with pytest.raises(TypeError):
        wgrad(h, f)


@pytest.mark.parametrize("dtype, shape, code, ld", [
    (torch.uint8, (4, 16), 2, 8), (torch.uint8, (4, 40), 2, 20), (torch.uint8, (4, 32), 0, 8), (torch.int16, (4, 8), 1, 8), (torch.int16, (4, 24), 2, 24),
    (torch.int32, (4, 4), 2, 8), (torch.int32, (4, 12), 0, 12), (torch.int8, (4, 17), 2, None), (torch.uint8, (4, 34), 0, None), (torch.uint8, (4, 14), 2, None)])
def test_the_pitch_of_storage_of_another_kind_is_in_elements_of_the_given_type(seam, r, dtype, shape, code, ld):
    x = torch.zeros(shape, dtype=dtype)
    calls = {"out": (lambda: seam.i8_restore(r, 0, -1, A, A, x, 8, 4, 0, 0, code, 0), 1),
             "x": (lambda: seam.i8_quantize(r, 0, -1, x, A, A, 8, 4, False, 0, 0, code, 0), 0),
             "y": (lambda: seam.i8_linear(r, 0, -1, A, A, A, A, x, 8, 4, 16, None, 0, 0, 0, code, 0), 2),
             "sum": (lambda: seam.i8_rmsnorm(r, 0, -1, A, A, A, A, 8, 4, None, x, 1e-6, 0, 0, 0, 0, code, 0), 3),
             "residual": (lambda: seam.i8_rmsnorm(r, 0, -1, A, A, A, A, 8, 4, x, None, 1e-6, 0, 0, 0, 0, code, 0), 1),
             "dw": (lambda: seam.i8_wgrad(r, 0, -1, A, A, A, x, 8, 4, 16, None, 1.0, 0.0, 0, 0, 0, 0, 2, code, 0), 3),
             "c": (lambda: seam.i8_wgrad(r, 0, -1, A, A, A, A, 8, 4, 16, x, 1.0, 1.0, 0, 0, 0, 0, 2, code, 0), 2)}
    if code:
        calls["dy"] = (lambda: seam.i8_wgrad(r, 0, -1, A, A, x, A, 16, 8, 4, None, 1.0, 0.0, 0, 0, 0, 0, code, 0, 0), 1)
    for what, (call, at) in calls.items():
        if ld is None:
            with pytest.raises(ValueError, match="apart"):
                call()
        else:
            assert call() == 0 and (ctypes.c_uint32 * 4).in_dll(seam.state, "seam_ld")[at] == ld, what


class ByName:
    """A tensor of a type without DLPack's table: it is asked by method and attribute names."""

    def __init__(self, tensor):
        self._t = tensor
        for name in ("data_ptr", "get_device", "is_contiguous", "stride", "element_size"):
            setattr(self, name, getattr(tensor, name))
        self.dtype, self.shape = tensor.dtype, tensor.shape


def test_tensors_are_read_alike_by_dlpack_and_by_name(seam, r):
    """Shapes, strides, types and the refusals that follow from them, through both ways of asking; Parameters and views among them."""
    def outcome(x, type_code=None, k=8):
        try:
            seam.i8_restore(r, 0, -1, A, A, x, k, 4, 0, 0, type_code, 0)
            return (ctypes.c_uint32 * 4).in_dll(seam.state, "seam_ld")[1]
        except (TypeError, ValueError) as e:
            return type(e).__name__

    base = torch.zeros(6, 40)
    views = [base, base[:4, :8], base[::2, 3:11], base[:, :8].t(), base.view(3, 2, 40)[:, :, :8], base.view(2, 3, 40)[:, :2, :8], base[0], base[:1, :8],
             base[:1].expand(4, 40), base.double(), base.half(), base.bfloat16()[:, ::2], base.int(), torch.nn.Parameter(base), torch.zeros(4, 1, 8),
             torch.zeros(1, 4, 8).transpose(0, 1), torch.zeros(1, 1, 1, 40), base.to(torch.int8), torch.zeros(5, 1, 8, 1)[..., 0], base.requires_grad_()[1:]]
    seen = set()
    for x in views:
        for code in (None, 0, 1, 2):
            got = outcome(x, code)
            assert got == outcome(ByName(x), code), (tuple(x.shape), x.stride(), x.dtype, code)
            seen.add(got)
    assert {"TypeError", "ValueError", 8, 40, 80} <= seen


def shapes(**kw):
    """The operands of one call each as (shape, dtype), all exactly as large as the call needs; `kw` replaces some."""
    i8, f32, bf16 = torch.int8, torch.float32, torch.bfloat16
    t = {"w": ((16, 32), i8), "w_scale": ((16,), f32), "x": ((4, 32), i8), "x_scale": ((4,), f32), "y": ((4, 16), bf16), "bias": ((16,), f32),
         "a": ((4, 32), bf16), "gamma": ((32,), bf16), "q": ((4, 32), i8), "scale": ((4,), f32), "residual": ((4, 32), bf16), "total": ((4, 32), bf16),
         "dy": ((4, 16), bf16), "dw": ((16, 32), f32), "c": ((16, 32), f32)}
    return {k: kw[k] if k in kw else torch.zeros(v[0], dtype=v[1]) for k, v in t.items()}


RUN = {
    "i8_linear": (("w", "w_scale", "x", "x_scale", "y", "bias"), lambda s, r, t, m=16, n=4, k=32: s.i8_linear(
        r, 0, -1, t["w"], t["w_scale"], t["x"], t["x_scale"], t["y"], m, n, k, t["bias"], 0, 0, 0, None, 0)),
    "i8_quantize": (("a", "q", "scale"), lambda s, r, t, k=32, n=4: s.i8_quantize(r, 0, -1, t["a"], t["q"], t["scale"], k, n, False, 0, 0, None, 0)),
    "i8_restore": (("q", "scale", "a"), lambda s, r, t, k=32, n=4: s.i8_restore(r, 0, -1, t["q"], t["scale"], t["a"], k, n, 0, 0, None, 0)),
    "i8_rmsnorm": (("a", "gamma", "q", "scale", "residual", "total"), lambda s, r, t, k=32, n=4: s.i8_rmsnorm(
        r, 0, -1, t["a"], t["gamma"], t["q"], t["scale"], k, n, t["residual"], t["total"], 1e-6, 0, 0, 0, 0, None, 0)),
    "i8_wgrad": (("q", "scale", "dy", "dw", "c"), lambda s, r, t, m=32, n=16, tokens=4, beta=1.0: s.i8_wgrad(
        r, 0, -1, t["q"], t["scale"], t["dy"], t["dw"], m, n, tokens, t["c"], 1.0, beta, 0, 0, 0, 0, None, None, 0)),
}


@pytest.mark.parametrize("form", [lambda x: x, ByName], ids=["dlpack", "by_name"])
@pytest.mark.parametrize("name, operand", [(n, o) for n, (operands, _) in RUN.items() for o in operands])
def test_a_tensor_that_ends_before_the_call_does_is_refused(seam, r, name, operand, form):
    """One element less, or one row less, than the call reads or writes; more than that, and the same rows inside a wider tensor, are served."""
    run = RUN[name][1]
    full = shapes()[operand]
    assert run(seam, r, shapes()) == 0
    short = [full.reshape(-1)[:-1]] if full.dim() == 1 else [full[:-1], full.reshape(-1)[:-1], torch.zeros(4 * full.shape[0], 2 * full.shape[1], dtype=full.dtype)[:full.shape[0] - 1, :full.shape[1]],
                                                              torch.zeros(full.shape[0], full.shape[1] + 8, dtype=full.dtype)[:, :full.shape[1] - 1]]
    calls = value(seam, "seam_calls")
    for x in short:
        with pytest.raises(ValueError, match=r"elements, the call reaches over \d+"):
            run(seam, r, shapes(**{operand: form(x)}))
    assert value(seam, "seam_calls") == calls
    if full.dim() == 1:
        enough = [torch.zeros(full.shape[0] + 3, dtype=full.dtype), full[None], full[:, None]]
    else:
        enough = [torch.zeros(full.shape[0] + 1, full.shape[1], dtype=full.dtype), full.reshape(-1), full[None], full[:, None], full.reshape(2, -1, full.shape[1]),
                  torch.zeros(full.shape[0], full.shape[1] + 8, dtype=full.dtype)[:, :full.shape[1]], torch.zeros(full.shape[0], full.shape[1] + 8, dtype=full.dtype)]
    for x in enough:
        assert run(seam, r, shapes(**{operand: form(x)})) == 0
    if operand not in ("y", "a", "dy", "dw"):        # (an address comes with its type)
        assert run(seam, r, shapes(**{operand: A})) == 0


def test_extents_of_given_leading_dimensions_and_of_storage_of_another_kind(seam, r):
    flat = torch.zeros(3 * 40 + 32, dtype=torch.int8)

    def restore(q, ldq, out=A, ldo=0, code=0):
        return seam.i8_restore(r, 0, -1, q, A, out, 32, 4, ldq, ldo, code, 0)

    assert restore(flat, 40) == 0 and restore(flat.reshape(8, 19), 40) == 0
    for q, ldq in ((flat, 41), (flat[1:], 40), (flat[:32].expand(4, 32), 32), (flat[:32].expand(4, 32), 40)):
        with pytest.raises(ValueError, match="reaches over"):
            restore(q, ldq)
    raw = torch.zeros(4 * 64, dtype=torch.uint8)                  # 32 BF16 elements of 4 rows, or 16 FP32 ones
    assert restore(A, 0, raw, 0, 2) == 0 and restore(A, 0, raw.view(4, 64), 0, 2) == 0
    with pytest.raises(ValueError, match="reaches over"):
        restore(A, 0, raw, 0, 0)
    with pytest.raises(ValueError, match="reaches over"):
        restore(A, 0, raw[:-1], 0, 2)


def test_what_a_call_does_not_read_may_be_missing_or_empty(seam, r):
    """No tokens, no channels, no features; C beside beta 0; and what the C call refuses by itself reaches it."""
    none = {k: v.reshape(-1)[:0] for k, v in shapes().items()}
    linear, quantize, restore, rms, wgrad = (RUN[n][1] for n in ("i8_linear", "i8_quantize", "i8_restore", "i8_rmsnorm", "i8_wgrad"))
    assert linear(seam, r, none, n=0) == 0 and linear(seam, r, none, m=0) == 0
    assert quantize(seam, r, none, n=0) == 0 and restore(seam, r, none, n=0) == 0 and restore(seam, r, none, k=0) == 0 and rms(seam, r, none, n=0) == 0
    assert wgrad(seam, r, none, n=0) == 0 and wgrad(seam, r, none, m=0) == 0
    t = shapes(q=none["q"], scale=none["scale"], dy=none["dy"])
    assert wgrad(seam, r, t, tokens=0) == 0
    assert wgrad(seam, r, shapes(c=none["c"]), beta=0.0) == 0
    assert quantize(seam, r, shapes(q=none["q"], a=none["a"]), k=0) == 0
    with pytest.raises(ValueError, match="scale holds 0"):
        quantize(seam, r, none, k=0)                       # scales of empty rows are written
    with pytest.raises(ValueError, match="w_scale holds 0"):
        linear(seam, r, shapes(w_scale=none["w_scale"]), k=0)
    assert linear(seam, r, shapes(w=none["w"], x=none["x"]), k=0) == 0
    t = shapes()
    assert seam.i8_linear(r, 0, -1, t["w"], t["w_scale"], t["x"], t["x_scale"], t["y"], 16, 4, 131072, None, 131072, 131072, 0, None, 0) == 0
    assert seam.i8_linear(r, 0, -1, t["w"], t["w_scale"], t["x"], t["x_scale"], t["y"], 16, 4, 32, None, 31, 0, 0, None, 0) == 0


class Shell(torch.Tensor):
    """A tensor without storage of its own, as wrapper subclasses are."""

    @staticmethod
    def __new__(cls, inner):
        return torch.Tensor._make_wrapper_subclass(cls, inner.shape, dtype=inner.dtype, strides=inner.stride(), device=inner.device)

    @classmethod
    def __torch_dispatch__(cls, func, types, args=(), kwargs=None):
        raise NotImplementedError(str(func))


@pytest.mark.parametrize("name, operand", [("i8_linear", "bias"), ("i8_rmsnorm", "residual"), ("i8_rmsnorm", "total"), ("i8_linear", "w"), ("i8_wgrad", "c")])
def test_a_tensor_without_storage_is_not_taken_for_an_absent_one(seam, r, name, operand):
    calls = value(seam, "seam_calls")
    with pytest.raises((RuntimeError, TypeError, ValueError, NotImplementedError)):
        RUN[name][1](seam, r, shapes(**{operand: Shell(shapes()[operand])}))
    assert value(seam, "seam_calls") == calls


def test_an_object_that_tells_its_strides_only_by_name_keeps_its_pitch(seam, r):
    x = ByName(torch.zeros(4, 40)[:, :8])
    del x.element_size
    assert seam.i8_restore(r, 0, -1, A, A, x, 8, 4, 0, 0, None, 0) == 0
    assert (ctypes.c_uint32 * 4).in_dll(seam.state, "seam_ld")[1] == 40
    with pytest.raises(ValueError, match="reaches over"):
        seam.i8_restore(r, 0, -1, A, A, x, 8, 5, 0, 0, None, 0)
