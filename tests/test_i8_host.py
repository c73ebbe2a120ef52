"""Argument checks and launch plans of the 8-bit entry points, without a GPU: sgemm_i8.cpp is compiled against a stand-in for the runner
(tests/i8_host_seam.cpp) that records the launches instead of making them."""
import ctypes
import subprocess
from pathlib import Path

import pytest

from runner import api

ROOT = Path(__file__).resolve().parent.parent
CSRC = ROOT / "amdgpu-arch-gemm_b200" / "csrc"
A = 1 << 20          # an address aligned to everything; nothing is dereferenced
u32 = ctypes.c_uint32


class Launch(ctypes.Structure):
    _fields_ = [("count", u32), ("function", ctypes.c_int32), ("grid", u32), ("threads", u32), ("smem", u32), ("cluster", u32),
                ("maps", u32), ("box", u32 * 4), ("dims", ctypes.c_uint64 * 4), ("variant", ctypes.c_int32), ("parts", u32),
                ("tile_n", u32), ("tpr", u32)]


@pytest.fixture(scope="module")
def lib(tmp_path_factory):
    out = tmp_path_factory.mktemp("i8") / "seam.so"
    subprocess.run(["g++", "-O1", "-std=c++17", "-fPIC", "-shared", "-Wall", "-Wextra", f"-I{ROOT / 'include'}", f"-I{CSRC}",
                    "-o", str(out), str(Path(__file__).parent / "i8_host_seam.cpp"), str(CSRC / "sgemm_i8.cpp")], check=True)
    L = ctypes.CDLL(str(out))
    for name in ("sgemm_i8_linear", "sgemm_i8_quantize", "sgemm_i8_restore", "sgemm_i8_rmsnorm", "sgemm_i8_wgrad"):
        getattr(L, name).restype, getattr(L, name).argtypes = api.ABI[name]
    L.seam_handle.restype = ctypes.c_void_p
    L.seam_handle.argtypes = [ctypes.c_int, ctypes.c_int64, ctypes.c_int64]
    L.seam_error.restype = ctypes.c_char_p
    L.seam_name.restype = ctypes.c_char_p
    L.seam_name.argtypes = [ctypes.c_int]
    L.seam_last.argtypes = [ctypes.POINTER(Launch)]
    return L


def last(L):
    rec = Launch()
    L.seam_last(ctypes.byref(rec))
    return rec


def linear(L, h, m=256, n=256, k=256, ldw=None, ldx=None, ldy=None, y_type=2, w=A, sw=A, x=A, sx=A, bias=None, y=A):
    up = max(16, (k + 15) // 16 * 16)
    return L.sgemm_i8_linear(h, w, sw, x, sx, bias, y, y_type, m, n, k, up if ldw is None else ldw, up if ldx is None else ldx,
                             max(m, 1) if ldy is None else ldy, None)


def quantize(L, h, k=64, n=8, ldx=None, ldq=None, x_type=2, pow2=0, x=A, q=A, s=A):
    return L.sgemm_i8_quantize(h, x, x_type, q, s, k, n, k if ldx is None else ldx, k if ldq is None else ldq, pow2, None)


def restore(L, h, k=64, n=8, ldq=None, ldo=None, out_type=2, q=A, s=A, out=A):
    return L.sgemm_i8_restore(h, q, s, out, out_type, k, n, k if ldq is None else ldq, k if ldo is None else ldo, None)


def rmsnorm(L, h, k=64, n=8, x=A, r=None, g=A, x_type=2, eps=1e-6, q=A, s=A, total=None, ldx=None, ldr=None, ldq=None, lds=None):
    up = lambda v: k if v is None else v   # noqa: E731
    return L.sgemm_i8_rmsnorm(h, x, r, g, x_type, eps, q, s, total, k, n, up(ldx), up(ldr), up(ldq), up(lds), None)


def wgrad(L, h, m=256, n=256, t=256, q=A, s=A, g=A, g_type=2, c=None, d=A, d_type=0, alpha=1.0, beta=0.0, ldq=None, ldg=None, ldc=None, ldd=None):
    return L.sgemm_i8_wgrad(h, q, s, g, g_type, c, d, d_type, alpha, beta, m, n, t, (m + 15) // 16 * 16 if ldq is None else ldq,
                            (n + 7) // 8 * 8 if ldg is None else ldg, m if ldc is None else ldc, m if ldd is None else ldd, None)


REFUSED = [
    (linear, dict(y_type=3)), (linear, dict(y_type=-1)), (linear, dict(k=131072)), (linear, dict(ldw=255)), (linear, dict(ldx=255)),
    (linear, dict(ldy=255)), (linear, dict(w=None)), (linear, dict(sw=None)), (linear, dict(x=None)), (linear, dict(sx=None)),
    (linear, dict(y=None)), (linear, dict(y=A + 1)), (linear, dict(y=A + 2, y_type=0)), (linear, dict(sx=A + 2)), (linear, dict(bias=A + 1)),
    (linear, dict(m=0xFFFFFFFF, ldy=0xFFFFFFFF)), (linear, dict(n=0xFFFFFFFF)),
    (quantize, dict(x_type=3)), (quantize, dict(pow2=2)), (quantize, dict(ldx=63)), (quantize, dict(ldq=63)), (quantize, dict(x=None)),
    (quantize, dict(q=None)), (quantize, dict(s=None)), (quantize, dict(x=A + 1)), (quantize, dict(x=A + 2, x_type=0)), (quantize, dict(s=A + 1)),
    (quantize, dict(k=0xFFFFFFFF)), (quantize, dict(n=0xFFFFFFFF)),
    (restore, dict(out_type=4)), (restore, dict(ldq=63)), (restore, dict(ldo=63)), (restore, dict(q=None)), (restore, dict(s=None)),
    (restore, dict(out=None)), (restore, dict(out=A + 1)), (restore, dict(s=A + 2)),
    (rmsnorm, dict(x_type=3)), (rmsnorm, dict(eps=-1.0)), (rmsnorm, dict(eps=float("nan"))), (rmsnorm, dict(eps=float("inf"))), (rmsnorm, dict(k=0)),
    (rmsnorm, dict(ldx=63)), (rmsnorm, dict(ldq=63)), (rmsnorm, dict(r=A, ldr=63)), (rmsnorm, dict(total=A, lds=63)), (rmsnorm, dict(x=None)),
    (rmsnorm, dict(g=None)), (rmsnorm, dict(q=None)), (rmsnorm, dict(s=None)), (rmsnorm, dict(x=A + 1)), (rmsnorm, dict(g=A + 1)),
    (rmsnorm, dict(r=A + 1)), (rmsnorm, dict(total=A + 1)), (rmsnorm, dict(total=A, lds=80)), (rmsnorm, dict(x=2 * A, r=A, total=A, lds=80)),
    (wgrad, dict(g_type=0)), (wgrad, dict(g_type=3)), (wgrad, dict(d_type=3)), (wgrad, dict(ldq=255)), (wgrad, dict(ldg=255)), (wgrad, dict(ldd=255)),
    (wgrad, dict(c=A, beta=1.0, ldc=255)), (wgrad, dict(q=None)), (wgrad, dict(s=None)), (wgrad, dict(g=None)), (wgrad, dict(d=None)),
    (wgrad, dict(beta=1.0)), (wgrad, dict(d=A, c=A, beta=1.0, ldc=300)), (wgrad, dict(g=A + 1)), (wgrad, dict(d=A + 2)), (wgrad, dict(s=A + 1)),
    (wgrad, dict(c=A + 2, beta=1.0)), (wgrad, dict(t=0xFFFFFFFF)),
]


@pytest.mark.parametrize("call,kwargs", REFUSED, ids=[f"{c.__name__}-{'-'.join(k)}-{i}" for i, (c, k) in enumerate(REFUSED)])
def test_bad_arguments_are_refused_before_anything_is_launched(lib, call, kwargs):
    h = lib.seam_handle(1, 0, 0)
    assert call(lib, h) == 0 and last(lib).count == 1          # the same call without the mistake is served
    before = last(lib).count
    assert call(lib, h, **kwargs) == -1
    assert last(lib).count == before and lib.seam_error() != b""
    assert call(lib, None, **kwargs) == -1


@pytest.mark.parametrize("call", [linear, quantize, restore, rmsnorm, wgrad])
def test_handles_of_other_cubins_are_refused(lib, call):
    h = lib.seam_handle(0, 0, 0)
    assert call(lib, h) == -6 and last(lib).count == 0 and b"INT8" in lib.seam_error()


def test_forced_tensor_kernels_refuse_what_they_cannot_serve(lib):
    for force in (1, 3, 4):
        h = lib.seam_handle(1, force, 0)
        assert linear(lib, h, ldw=257) == -6 and linear(lib, h, x=A + 1) == -6 and linear(lib, h, k=0, ldw=16, ldx=16) == -6
        assert wgrad(lib, h, ldg=260) == -6 and wgrad(lib, h, q=A + 8) == -6 and wgrad(lib, h, t=0) == -6
        assert last(lib).count == 0


def test_empty_problems_launch_nothing(lib):
    h = lib.seam_handle(1, 0, 0)
    assert linear(lib, h, m=0, ldy=1, w=None, x=None, y=None, sw=None, sx=None) == 0 and linear(lib, h, n=0) == 0
    assert quantize(lib, h, n=0, x=None, q=None, s=None) == 0 and restore(lib, h, n=0) == 0 and restore(lib, h, k=0, ldq=1, ldo=1) == 0
    assert rmsnorm(lib, h, n=0) == 0 and wgrad(lib, h, m=0, ldq=16, ldc=1, ldd=1) == 0 and wgrad(lib, h, n=0, ldg=8) == 0
    assert last(lib).count == 0
    assert quantize(lib, h, k=0, ldx=1, ldq=1, x=None, q=None) == 0 and last(lib).count == 1    # zero scales are written
    assert wgrad(lib, h, t=0, q=None, s=None, g=None) == 0 and last(lib).count == 2             # beta * C is written


def test_linear_plans_cover_the_output(lib):
    """The kernel chosen, its grid and boxes: every tile once, K's parts a power of two up to 8, boxes as the kernels expect."""
    for m in (1, 100, 128, 1000, 4096, 8192, 50000):
        for n in (1, 16, 17, 64, 100, 128, 129, 509, 2000, 8192):
            for k in (1, 100, 128, 1024, 4096, 16384):
                for ld_odd in (False, True):
                    h = lib.seam_handle(1, 0, 0)
                    assert linear(lib, h, m=m, n=n, k=k, ldw=(k + 15) // 16 * 16 + ld_odd) == 0
                    rec = last(lib)
                    name = lib.seam_name(rec.function).decode()
                    if ld_odd:
                        assert name == "generated_gemm_simt" and rec.grid == -(-m // 64) * -(-n // 64) and rec.variant == 2
                        continue
                    assert rec.maps == 2 and list(rec.dims) == [k, m, k, n] and list(rec.box)[:3] == [128, 128, 128]
                    if name in ("generated_gemm", "i8_linear_half"):
                        tile = 256 if name == "generated_gemm" else 128
                        tiles = -(-m // 256) * -(-n // tile)
                        assert rec.grid == 2 * min(tiles, 74) and rec.box[3] == tile // 2 and rec.threads == 384 and rec.smem <= 232448
                        assert rec.variant == (1 if tile == 256 else 4)
                    else:
                        tile = int(name.rsplit("_", 1)[1])
                        assert rec.parts in (1, 2, 4, 8) and rec.cluster == rec.parts and rec.box[3] == tile and rec.variant == 3
                        assert rec.grid == -(-m // 128) * rec.parts and rec.threads == 128 and rec.smem <= 232448
                        assert tile == next(t for t in (16, 32, 64, 128) if n <= t) and -(-k // 128) >= (2 * rec.parts if rec.parts > 1 else 1)


def test_linear_plans_follow_the_measured_crossings(lib):
    name = lambda n, m, k: (linear(lib, lib.seam_handle(1, 0, 0), m=m, n=n, k=k), lib.seam_name(last(lib).function).decode())[1]   # noqa: E731
    assert name(8192, 8192, 8192) == "generated_gemm" and name(1024, 4096, 4096) == "generated_gemm"
    assert name(509, 4096, 4096) == "i8_linear_half" and name(200, 8192, 8192) == "i8_linear_half"
    assert name(1, 4096, 4096) == "i8_linear_few_16" and name(23, 8200, 8190) == "i8_linear_few_32" and name(64, 4096, 4096) == "i8_linear_few_64"


def test_row_plans_hold_the_row(lib):
    per, most = {"v1": 8, "v2": 16, "v4": 32, "u4": 32, "s4": 32}, {"v1": 1024, "v2": 512, "v4": 256, "u4": 256, "s4": 256}
    for x_type in (0, 1, 2):
        for k in (1, 7, 64, 250, 1000, 4096, 8192, 16384, 100000):
            for n in (1, 5, 100, 8192):
                for ldx in ((k + 15) // 16 * 16, (k + 15) // 16 * 16 + 1):
                    h = lib.seam_handle(1, 0, 0)
                    assert quantize(lib, h, k=k, n=n, ldx=ldx, ldq=(k + 15) // 16 * 16, x_type=x_type) == 0
                    rec = last(lib)
                    name = lib.seam_name(rec.function).decode()
                    form = name[-2:]
                    assert name.startswith("i8_quantize_" + ("fp32", "fp16", "bf16")[x_type])
                    assert (form[0] == "v") == (ldx % 16 == 0)
                    assert rec.tpr in (32, 64, 128, 256, 512, 1024) and rec.threads == max(256, rec.tpr)
                    assert rec.tpr <= most[form]                       # the block the kernel was compiled for
                    assert rec.grid == -(-n // (rec.threads // rec.tpr))
                    assert rec.tpr * per[form] >= min(k + 7 * (form == "u4"), 8192)         # one pass, up to 8192 elements


def test_wgrad_plans_cover_the_gradient(lib):
    for m in (1, 256, 1000, 1024, 4096):
        for n in (1, 256, 1000, 11001):
            for t in (1, 64, 100, 1000, 16384):
                h = lib.seam_handle(1, 0, 0)
                assert wgrad(lib, h, m=m, n=n, t=t) == 0
                rec = last(lib)
                tiles = -(-m // 256) * -(-n // 256)
                assert lib.seam_name(rec.function) == b"i8_wgrad" and rec.parts in (1, 2, 3, 4) and rec.cluster == 2 * rec.parts
                assert rec.grid == (tiles * 2 * rec.parts if rec.parts > 1 else 2 * min(tiles, 74))
                assert rec.parts == 1 or (tiles <= (74, 33, 22, 15)[rec.parts - 1] and -(-t // 64) >= rec.parts)
                assert list(rec.dims) == [m, t, n, t] and list(rec.box) == [128, 64, 64, 64] and rec.smem <= 232448


def test_row_forms_follow_alignment(lib):
    h = lib.seam_handle(1, 0, 0)
    form = lambda: lib.seam_name(last(lib).function).decode()[-2:]   # noqa: E731
    assert rmsnorm(lib, h) == 0 and form()[0] == "v"
    for kwargs in (dict(x=A + 2), dict(g=A + 8), dict(ldx=65), dict(ldq=65), dict(q=A + 4), dict(x=A + 2, r=A + 18, total=3 * A + 2, ldx=65, ldr=65, lds=73)):
        assert rmsnorm(lib, h, **kwargs) == 0 and form() == "u4", kwargs      # every matrix at the same offset into a vector
    for kwargs in (dict(r=A + 4), dict(total=A + 2), dict(r=A, ldr=66), dict(x=A + 2, r=A), dict(ldx=65, total=2 * A)):
        assert rmsnorm(lib, h, **kwargs) == 0 and form() == "s4", kwargs
    assert restore(lib, h) == 0 and form() == "_v"
    for kwargs in (dict(q=A + 8), dict(ldq=72), dict(out=A + 8), dict(ldo=65)):
        assert restore(lib, h, **kwargs) == 0 and form() == "_u", kwargs


def test_register_hand_over_is_checked_for_the_kernel_that_does_it(lib):
    lib.seam_registers.argtypes = [ctypes.c_int]
    names = [lib.seam_name(i).decode() for i in range(lib.seam_count())]
    assert len(set(names)) == len(names) and {n: lib.seam_registers(i) for i, n in enumerate(names) if lib.seam_registers(i)} == {"i8_wgrad": 72}
