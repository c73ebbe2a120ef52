"""ctypes binding of libsgemm_runner.so (the C ABI declared in include/sgemm_runner.h).

This is the Python face of the runner: the calls the reference makes inside its C++ runner program
(runner/generator_runner.cpp:69-190 — load the code object, read the TOML, pack arguments, launch) are
reachable from Python here, so tests and the benchmark drive exactly the path a C caller would.

There is no CPU implementation behind this module: when the shared library has not been built, or no
CUDA driver / device is present, the calls raise ``SgemmError``.
"""
from __future__ import annotations

import ctypes
import importlib.util
import os
import subprocess
import sys
import sysconfig
from pathlib import Path
from typing import Optional, Tuple

PKG_DIR = Path(__file__).resolve().parent.parent
LIB_PATH = PKG_DIR / "build" / "libsgemm_runner.so"
RUNNER_PATH = PKG_DIR / "build" / "GeneratorRunner"
NATIVE_PATH = PKG_DIR / "build" / ("_sgemm_native" + (sysconfig.get_config_var("EXT_SUFFIX") or ".so"))

_f32p = ctypes.POINTER(ctypes.c_float)
_u32 = ctypes.c_uint32
_u64 = ctypes.c_uint64
_vp = ctypes.c_void_p


class SgemmConfig(ctypes.Structure):
    """Mirror of ``struct sgemm_config``."""
    _fields_ = [
        ("a_type", ctypes.c_int32), ("b_type", ctypes.c_int32), ("cd_type", ctypes.c_int32), ("scalar_type", ctypes.c_int32),
        ("mfma", ctypes.c_int32 * 4), ("wave_group", ctypes.c_int32 * 2), ("wave_tiling", ctypes.c_int32 * 2),
        ("depth_k", ctypes.c_int32), ("vmem_stage", ctypes.c_int32), ("wavefront_size", ctypes.c_int32),
        ("lds_usage_bytes", ctypes.c_int32), ("trans_a", ctypes.c_int32), ("trans_b", ctypes.c_int32),
        ("variant", ctypes.c_int32), ("num_threads", ctypes.c_int32), ("dynamic_smem_bytes", ctypes.c_int32),
        ("stages", ctypes.c_int32), ("a_kmajor", ctypes.c_int32), ("split_inkernel", ctypes.c_int32),
        ("fallback_tile", ctypes.c_int32 * 3),
        ("fallback_threads", ctypes.c_int32), ("entry", ctypes.c_char * 64), ("fallback_entry", ctypes.c_char * 64),
        ("skinny_tile", ctypes.c_int32 * 3), ("skinny_threads", ctypes.c_int32), ("skinny_smem_bytes", ctypes.c_int32),
        ("skinny_entry", ctypes.c_char * 64), ("acc_chain", ctypes.c_int32), ("skinny_acc_chain", ctypes.c_int32),
        ("wholek_entry", ctypes.c_char * 64),
        ("thin_tile", ctypes.c_int32 * 3), ("thin_threads", ctypes.c_int32), ("thin_smem_bytes", ctypes.c_int32),
        ("thin_acc_chain", ctypes.c_int32), ("thin_entry", ctypes.c_char * 64),
        ("feed_tma", ctypes.c_int32),
    ]


class SgemmError(RuntimeError):
    def __init__(self, code: int, what: str, detail: str):
        super().__init__(f"{what}: {detail} [code {code}]")
        self.code = code


# every symbol include/sgemm_runner.h declares: name -> (restype, argtypes)
_GEMM_ARGS = [_vp, _vp, _vp, _vp, _vp, ctypes.c_float, ctypes.c_float, _u32, _u32, _u32, _u32, _u32, _u32, _u32]
ABI = {
    "sgemm_config_parse": (ctypes.c_int, [ctypes.c_char_p, ctypes.POINTER(SgemmConfig)]),
    "sgemm_config_tile": (ctypes.c_int, [ctypes.POINTER(SgemmConfig), ctypes.POINTER(_u32), ctypes.POINTER(_u32)]),
    "sgemm_open": (ctypes.c_int, [ctypes.c_char_p, ctypes.c_char_p, ctypes.c_int, ctypes.POINTER(_vp)]),
    "sgemm_close": (ctypes.c_int, [_vp]),
    "sgemm_launch": (ctypes.c_int, _GEMM_ARGS + [_vp]),
    "sgemm_launch_noalloc": (ctypes.c_int, _GEMM_ARGS + [_vp]),
    "sgemm_noalloc_scratch_bytes": (ctypes.c_size_t, []),
    "sgemm_run_host": (ctypes.c_int, _GEMM_ARGS),
    "sgemm_run_host_sharded": (ctypes.c_int, _GEMM_ARGS),
    "sgemm_shard_columns": (ctypes.c_int, [_u32, _u32, _u32, _u32, ctypes.POINTER(_u32), ctypes.POINTER(_u32)]),
    "sgemm_comm_unique_id": (ctypes.c_int, [ctypes.c_char_p]),
    "sgemm_comm_init": (ctypes.c_int, [_vp, ctypes.c_char_p, ctypes.c_int, ctypes.c_int]),
    "sgemm_comm_init_all": (ctypes.c_int, [ctypes.POINTER(_vp), ctypes.c_int]),
    "sgemm_comm_destroy": (ctypes.c_int, [_vp]),
    "sgemm_allgather_columns": (ctypes.c_int, [_vp, _vp, _u32, _u32, _u32, _u32, _vp]),
    "sgemm_bench": (ctypes.c_int, _GEMM_ARGS + [_u32, _u32, _vp, ctypes.POINTER(ctypes.c_float)]),
    "sgemm_last_status": (ctypes.c_int, [_vp, ctypes.POINTER(_u32 * 8)]),
    "sgemm_wait_selftest": (ctypes.c_int, [_vp, _u32, _u32]),
    "sgemm_set_option": (ctypes.c_int, [_vp, ctypes.c_char_p, ctypes.c_int64]),
    "sgemm_get_info": (ctypes.c_int, [_vp, ctypes.c_char_p, ctypes.POINTER(ctypes.c_int64)]),
    "sgemm_workspace_bytes": (ctypes.c_int, [_vp, _u32, _u32, _u32, _u32, _u32, ctypes.POINTER(ctypes.c_size_t)]),
    "sgemm_workspace_bytes_for": (ctypes.c_int, [_vp, _vp, _vp, _u32, _u32, _u32, _u32, _u32, ctypes.POINTER(ctypes.c_size_t)]),
    "sgemm_set_workspace": (ctypes.c_int, [_vp, _vp, ctypes.c_size_t]),
    "sgemm_fill_uniform": (ctypes.c_int, [_vp, _vp, _u64, _u64, _u64, _vp]),
    "sgemm_narrow16": (ctypes.c_int, [_vp, _vp, _vp, _u64, _vp]),
    "sgemm_i8_linear": (ctypes.c_int, [_vp] * 7 + [ctypes.c_int] + [_u32] * 6 + [_vp]),
    "sgemm_i8_quantize": (ctypes.c_int, [_vp, _vp, ctypes.c_int, _vp, _vp, _u32, _u32, _u32, _u32, ctypes.c_int, _vp]),
    "sgemm_i8_restore": (ctypes.c_int, [_vp, _vp, _vp, _vp, ctypes.c_int, _u32, _u32, _u32, _u32, _vp]),
    "sgemm_i8_rmsnorm": (ctypes.c_int, [_vp] * 4 + [ctypes.c_int, ctypes.c_float, _vp, _vp, _vp] + [_u32] * 6 + [_vp]),
    "sgemm_i8_wgrad": (ctypes.c_int, [_vp] * 4 + [ctypes.c_int, _vp, _vp, ctypes.c_int, ctypes.c_float, ctypes.c_float] + [_u32] * 7 + [_vp]),
    "sgemm_tile_map": (ctypes.c_int, [_vp, ctypes.POINTER(ctypes.c_int32), _u32, _u32]),
    "sgemm_dev_alloc": (ctypes.c_int, [_vp, ctypes.c_size_t, ctypes.POINTER(_vp)]),
    "sgemm_dev_free": (ctypes.c_int, [_vp, _vp]),
    "sgemm_dev_upload": (ctypes.c_int, [_vp, _vp, _vp, ctypes.c_size_t]),
    "sgemm_dev_download": (ctypes.c_int, [_vp, _vp, _vp, ctypes.c_size_t]),
    "sgemm_dev_memset": (ctypes.c_int, [_vp, _vp, ctypes.c_int, ctypes.c_size_t]),
    "sgemm_dev_sync": (ctypes.c_int, [_vp]),
    "sgemm_strerror": (ctypes.c_char_p, [ctypes.c_int]),
    "sgemm_last_error": (ctypes.c_char_p, [_vp]),
    "sgemm_device_count": (ctypes.c_int, []),
}

_lib: Optional[ctypes.CDLL] = None


def build_library(force: bool = False) -> Path:
    """Run the Makefile beside this file (g++ and nvcc; needs the CUDA toolkit headers, not a GPU).  The binding of the ``i8_*``
    methods is built too where Python's headers are."""
    headers = (Path(sysconfig.get_paths()["include"]) / "Python.h").exists()
    if force or not LIB_PATH.exists() or not RUNNER_PATH.exists() or (headers and not NATIVE_PATH.exists()):
        env = dict(os.environ, PYTHON=sys.executable)
        env.pop("CXX", None)
        subprocess.run(["make", "-C", str(Path(__file__).resolve().parent), "-s"] + (["-B"] if force else []),
                       check=True, env=env)
    return LIB_PATH


def lib() -> ctypes.CDLL:
    global _lib
    if _lib is None:
        if not LIB_PATH.exists():
            raise SgemmError(-5, "libsgemm_runner.so", f"{LIB_PATH} is not built; run __graft_entry__.build() "
                                                        f"or make -C {PKG_DIR / 'runner'}")
        L = ctypes.CDLL(str(LIB_PATH))
        for name, (res, args) in ABI.items():
            fn = getattr(L, name)
            fn.restype = res
            fn.argtypes = args
        _lib = L
    return _lib


_native_module = None


def _native():
    """The extension module behind the ``i8_*`` methods (csrc/sgemm_py.cpp)."""
    global _native_module
    if _native_module is None:
        lib()
        if not NATIVE_PATH.exists():
            raise SgemmError(-5, "_sgemm_native", f"{NATIVE_PATH} is not built; run __graft_entry__.build() or make -C {PKG_DIR / 'runner'} "
                                                 f"(needs Python's headers)")
        spec = importlib.util.spec_from_file_location("_sgemm_native", NATIVE_PATH)
        module = importlib.util.module_from_spec(spec)
        spec.loader.exec_module(module)
        module.setup(_type_code)
        _native_module = module
    return _native_module


def parse_config(toml_path: str) -> SgemmConfig:
    cfg = SgemmConfig()
    rc = lib().sgemm_config_parse(str(toml_path).encode(), ctypes.byref(cfg))
    if rc:
        raise SgemmError(rc, "sgemm_config_parse", lib().sgemm_last_error(None).decode())
    return cfg


def config_tile(cfg: SgemmConfig) -> Tuple[int, int]:
    tm, tn = _u32(), _u32()
    lib().sgemm_config_tile(ctypes.byref(cfg), ctypes.byref(tm), ctypes.byref(tn))
    return tm.value, tn.value


def _ptr(x) -> int:
    """Device/host address of a torch tensor, a NumPy array, an int, or None."""
    if x is None:
        return 0
    if isinstance(x, int):
        return x
    if hasattr(x, "data_ptr"):
        return x.data_ptr()
    if hasattr(x, "ctypes"):
        return x.ctypes.data
    raise TypeError(f"cannot take the address of {type(x)}")


_TYPE_CODES = {"float32": 0, "float16": 1, "bfloat16": 2, "int8": 3}
_VECTORS = {"w_scale", "x_scale", "scale", "bias", "gamma"}
_type_codes: dict = {}   # dtype object -> code, filled as dtypes are met


def _dtype_code(dtype) -> int:
    """Element type as the C ABI and the generator number it (0 FP32, 1 FP16, 2 BF16, 3 INT8), -1 for any other."""
    code = _type_codes.get(dtype)
    if code is None:
        code = _type_codes[dtype] = _TYPE_CODES.get(str(dtype).replace("torch.", ""), -1)
    return code


def _type_code(x, given: Optional[int]) -> int:
    """Element type of a matrix: the one given, which must be a tensor's own where that is one of FP32, FP16 and BF16, else the tensor's."""
    code = _dtype_code(getattr(x, "dtype", None))
    if given is not None:
        if 0 <= code <= 2 and code != int(given):
            raise TypeError(f"a tensor of {x.dtype} with the element type {given}")
        return int(given)
    if not 0 <= code <= 2:
        raise TypeError(f"element type of {type(x).__name__} {getattr(x, 'dtype', '')}: pass a FP32, FP16 or BF16 tensor, or the "
                        f"type with an address")
    return code


class SgemmRunner:
    """One loaded kernel on one device (wraps ``sgemm_handle``)."""

    AUTO, TENSOR, SIMT, TENSOR_SKINNY = 0, 1, 2, 3

    def __init__(self, cubin_path: str, toml_path: str, device: int = 0):
        self._L = lib()
        self._h = _vp()
        rc = self._L.sgemm_open(str(cubin_path).encode(), str(toml_path).encode(), device, ctypes.byref(self._h))
        if rc:
            self._h = None
            raise SgemmError(rc, "sgemm_open", self._L.sgemm_last_error(None).decode())
        self.device = device
        self._native = None

    # ---------------------------------------------------------------------------------- plumbing
    def _check(self, rc: int, what: str):
        if rc:
            raise SgemmError(rc, what, self._L.sgemm_last_error(self._h).decode())

    def close(self):
        if self._h:
            self._L.sgemm_close(self._h)
            self._h = None

    def __enter__(self):
        return self

    def __exit__(self, *exc):
        self.close()

    def __del__(self):
        try:
            self.close()
        except Exception:
            pass

    @staticmethod
    def _lds(m, n, k, lda, ldb, ldc, ldd):
        return (lda or max(m, 1), ldb or max(k, 1), ldc or max(m, 1), ldd or max(m, 1))

    # ----------------------------------------------------------------------------------- compute
    def launch(self, a, b, c, d, m, n, k, alpha=1.0, beta=0.0, lda=0, ldb=0, ldc=0, ldd=0, stream=0):
        """Asynchronous D = alpha*A*B + beta*C on device buffers (tensors, arrays' addresses or ints)."""
        lda, ldb, ldc, ldd = self._lds(m, n, k, lda, ldb, ldc, ldd)
        self._check(self._L.sgemm_launch(self._h, _ptr(a), _ptr(b), _ptr(c), _ptr(d), alpha, beta, m, n, k,
                                         lda, ldb, ldc, ldd, stream), "sgemm_launch")

    def launch_noalloc(self, a, b, c, d, m, n, k, alpha=1.0, beta=0.0, lda=0, ldb=0, ldc=0, ldd=0, stream=0):
        """``launch`` for callers that must not allocate device memory: the scratch comes from the library's
        fixed array (``noalloc_scratch_bytes()``); larger problems raise ``SgemmError`` with code -9."""
        lda, ldb, ldc, ldd = self._lds(m, n, k, lda, ldb, ldc, ldd)
        self._check(self._L.sgemm_launch_noalloc(self._h, _ptr(a), _ptr(b), _ptr(c), _ptr(d), alpha, beta, m, n, k,
                                                 lda, ldb, ldc, ldd, stream), "sgemm_launch_noalloc")

    def run_host(self, a, b, c, d, m, n, k, alpha=1.0, beta=0.0, lda=0, ldb=0, ldc=0, ldd=0):
        """The same with HOST buffers (upload, launch, download, synchronise)."""
        lda, ldb, ldc, ldd = self._lds(m, n, k, lda, ldb, ldc, ldd)
        self._check(self._L.sgemm_run_host(self._h, _ptr(a), _ptr(b), _ptr(c), _ptr(d), alpha, beta, m, n, k,
                                           lda, ldb, ldc, ldd), "sgemm_run_host")

    def run_host_sharded(self, a, b, c, d, m, n_local, k, alpha=1.0, beta=0.0, lda=0, ldb=0, ldc=0, ldd=0):
        """``run_host`` for one rank of a column-sharded call: ``a`` is the whole replicated A in host memory (only this
        rank's slice is uploaded, the ranks complete each other's copies over NVLink), ``b``, ``c``, ``d`` are this
        rank's column shards.  Collective over the handle's communicator (``comm_init``)."""
        lda, ldb, ldc, ldd = self._lds(m, n_local, k, lda, ldb, ldc, ldd)
        self._check(self._L.sgemm_run_host_sharded(self._h, _ptr(a), _ptr(b), _ptr(c), _ptr(d), alpha, beta, m, n_local, k,
                                                   lda, ldb, ldc, ldd), "sgemm_run_host_sharded")

    # ------------------------------------------------- 8-bit operands (cubins generated for INT8)
    def _addr(self, x, name: str, code: int = -1) -> int:
        """Address of an operand of an 8-bit call.  A tensor must lie on the handle's GPU, have the element type the call takes
        (`code`, -1: any) and lie as the call reads it: a vector without gaps, a matrix with the elements of a row one after
        the other and, where it has more than two dimensions, its rows at one distance throughout."""
        if x is None or isinstance(x, int):
            return _ptr(x)
        if not hasattr(x, "data_ptr"):
            raise TypeError(f"{name} is a {type(x).__name__}: the call takes tensors on the handle's GPU or device addresses")
        if x.get_device() != self.device:
            raise ValueError(f"{name} lies on {x.device}, the handle on GPU {self.device}")
        if code >= 0 and _dtype_code(x.dtype) != code:
            raise TypeError(f"{name} is {x.dtype}, the call takes {[k for k, v in _TYPE_CODES.items() if v == code][0]}")
        if not x.is_contiguous():
            if name in _VECTORS:
                raise ValueError(f"{name}: the elements must be contiguous")
            if x.shape[-1] > 1 and x.stride(-1) != 1:
                raise ValueError(f"{name}: the elements of a row must be contiguous")
            # dimensions of one have no distance of their own; the others, from the rows outwards, must follow one another
            outer = [(n, d) for n, d in zip(x.shape[:-1], x.stride()[:-1]) if n > 1]
            if any(far != near * count for (_, far), (count, near) in zip(outer, outer[1:])):
                raise ValueError(f"{name}: its rows do not lie at one distance; pass one part at a time or a copy")
        return x.data_ptr()

    # Operands are tensors on the handle's GPU or addresses (their element type then goes with ..._type: 0 FP32, 1 FP16, 2 BF16).  A leading
    # dimension of 0 is the distance of a tensor's rows (of all its dimensions but the last), and for addresses the length of a row.  A tensor
    # that ends before the last element the call would touch is refused (ValueError).
    def _i8(self, name: str, *args):
        if not self._h:
            raise SgemmError(-1, "sgemm_" + name, "the handle is closed")
        native = self._native
        if native is None:
            native = self._native = _native()
        rc = getattr(native, name)(self, self._h.value, self.device, *args)
        if rc:
            self._check(rc, "sgemm_" + name)

    def i8_linear(self, w, w_scale, x, x_scale, y, m, n, k, bias=None, ldw=0, ldx=0, ldy=0, y_type=None, stream=0):
        """Y[i, j] = (sum_k W[k, i] X[k, j]) * x_scale[j] * w_scale[i] (+ bias[i]): ``m`` channels, ``n`` tokens, ``k``
        features; int8 W and X column-major K x M and K x N (a channel's weights, a token's features contiguous), Y
        column-major M x N in FP32, FP16 or BF16, scales and bias FP32."""
        self._i8("i8_linear", w, w_scale, x, x_scale, y, m, n, k, bias, ldw, ldx, ldy, y_type, stream)

    def i8_quantize(self, x, q, scale, k, n, pow2=False, ldx=0, ldq=0, x_type=None, stream=0):
        """8-bit columns of the K x N matrix X with one scale each (a token's features or a channel's weights per column):
        scale max|x|/127, or with ``pow2`` the least power of two that holds the column (activation checkpoints)."""
        self._i8("i8_quantize", x, q, scale, k, n, pow2, ldx, ldq, x_type, stream)

    def i8_restore(self, q, scale, out, k, n, ldq=0, ldo=0, out_type=None, stream=0):
        """The values ``scale[j] * q[:, j]``, rounded to the output's type."""
        self._i8("i8_restore", q, scale, out, k, n, ldq, ldo, out_type, stream)

    def i8_rmsnorm(self, x, gamma, q, scale, k, n, residual=None, sum_out=None, eps=1e-6, ldx=0, ldr=0, ldq=0, lds=0,
                   x_type=None, stream=0):
        """Root-mean-square norm of X (+ residual) times gamma, as 8-bit columns with one scale each; ``sum_out`` receives
        X + residual in X's type (it may be the residual or X itself)."""
        self._i8("i8_rmsnorm", x, gamma, q, scale, k, n, residual, sum_out, eps, ldx, ldr, ldq, lds, x_type, stream)

    def i8_wgrad(self, q, scale, dy, dw, m, n, tokens, c=None, alpha=1.0, beta=0.0, ldq=0, lddy=0, ldc=0, lddw=0,
                 dy_type=None, dw_type=None, stream=0):
        """Weight gradient from an 8-bit checkpoint: dW[i, j] = alpha * sum_t V(q[i, t], scale[t]) * dY[j, t] + beta * C[i, j] with
        ``m`` features, ``n`` channels; V is the value ``i8_restore`` gives in dY's type (FP16 or BF16); C and dW have one type."""
        self._i8("i8_wgrad", q, scale, dy, dw, m, n, tokens, c, alpha, beta, ldq, lddy, ldc, lddw, dy_type, dw_type, stream)

    # ------------------------------------------------------------------------------- multi-GPU
    def comm_init(self, comm_id: bytes, rank: int, world: int):
        """Join the communicator ``comm_id`` (from ``comm_unique_id()`` on one rank) as ``rank`` of ``world``."""
        self._check(self._L.sgemm_comm_init(self._h, comm_id, rank, world), "sgemm_comm_init")

    def comm_destroy(self):
        self._check(self._L.sgemm_comm_destroy(self._h), "sgemm_comm_destroy")

    def allgather_columns(self, d_full, m, n, ldd=0, tile_n=0, stream=0):
        """In-place all-gather of D's column shards (this rank's shard already lies at its place in ``d_full``)."""
        self._check(self._L.sgemm_allgather_columns(self._h, _ptr(d_full), m, n, ldd or max(m, 1), tile_n or self.info("tile_n"),
                                                    stream), "sgemm_allgather_columns")

    def bench(self, a, b, c, d, m, n, k, alpha=1.0, beta=0.0, warmup=5, runs=50, stream=0) -> float:
        """Mean milliseconds of ``runs`` back-to-back launches after ``warmup`` (CUDA events)."""
        ms = ctypes.c_float()
        lda, ldb, ldc, ldd = self._lds(m, n, k, 0, 0, 0, 0)
        self._check(self._L.sgemm_bench(self._h, _ptr(a), _ptr(b), _ptr(c), _ptr(d), alpha, beta, m, n, k,
                                        lda, ldb, ldc, ldd, warmup, runs, stream, ctypes.byref(ms)), "sgemm_bench")
        return ms.value

    def last_status(self):
        st = (_u32 * 8)()
        self._check(self._L.sgemm_last_status(self._h, ctypes.byref(st)), "sgemm_last_status")
        return list(st)

    def wait_selftest(self, timeout_ms: int = 20, tag: int = 0x7E57):
        """Launch the bounded-wait self-test kernel (see ``sgemm_wait_selftest``); read the outcome with ``last_status``."""
        self._check(self._L.sgemm_wait_selftest(self._h, timeout_ms, tag), "sgemm_wait_selftest")

    # ------------------------------------------------------------------------- options and facts
    def set_option(self, key: str, value: int):
        self._check(self._L.sgemm_set_option(self._h, key.encode(), value), "sgemm_set_option")

    def info(self, key: str) -> int:
        v = ctypes.c_int64()
        self._check(self._L.sgemm_get_info(self._h, key.encode(), ctypes.byref(v)), "sgemm_get_info")
        return v.value

    def workspace_bytes(self, m, n, k, lda=0, ldb=0, a=None, b=None) -> int:
        """Scratch bytes a launch of this problem needs; with `a` / `b` (device addresses) the need of these very
        operands, aligned copies of unaligned ones included."""
        out = ctypes.c_size_t()
        self._check(self._L.sgemm_workspace_bytes_for(self._h, _ptr(a), _ptr(b), m, n, k, lda or m, ldb or k,
                                                      ctypes.byref(out)), "sgemm_workspace_bytes_for")
        if a is None and b is None:
            plain = ctypes.c_size_t()
            self._check(self._L.sgemm_workspace_bytes(self._h, m, n, k, lda or m, ldb or k, ctypes.byref(plain)),
                        "sgemm_workspace_bytes")
            assert plain.value == out.value
        return out.value

    def set_workspace(self, dptr, nbytes: int):
        self._check(self._L.sgemm_set_workspace(self._h, _ptr(dptr), nbytes), "sgemm_set_workspace")

    # --------------------------------------------------------------------------------- utilities
    def fill_uniform(self, dptr, count: int, stream_id: int, first_index: int = 0, stream=0):
        self._check(self._L.sgemm_fill_uniform(self._h, _ptr(dptr), count, first_index, stream_id, stream),
                    "sgemm_fill_uniform")

    def narrow16(self, dsrc, ddst, count: int, stream=0):
        """FP32 -> the cubin's 16-bit operand type (FP16 / BF16), on the device."""
        self._check(self._L.sgemm_narrow16(self._h, _ptr(dsrc), _ptr(ddst), count, stream), "sgemm_narrow16")

    def tile_map(self, nx: int, ny: int):
        buf = (ctypes.c_int32 * (2 * nx * ny))()
        self._check(self._L.sgemm_tile_map(self._h, buf, nx, ny), "sgemm_tile_map")
        return [(buf[2 * i], buf[2 * i + 1]) for i in range(nx * ny)]

    def dev_alloc(self, nbytes: int) -> int:
        p = _vp()
        self._check(self._L.sgemm_dev_alloc(self._h, nbytes, ctypes.byref(p)), "sgemm_dev_alloc")
        return p.value or 0

    def dev_free(self, dptr: int):
        self._check(self._L.sgemm_dev_free(self._h, dptr), "sgemm_dev_free")

    def upload(self, dptr: int, host_array):
        self._check(self._L.sgemm_dev_upload(self._h, dptr, _ptr(host_array), host_array.nbytes), "sgemm_dev_upload")

    def download(self, host_array, dptr: int):
        self._check(self._L.sgemm_dev_download(self._h, _ptr(host_array), dptr, host_array.nbytes), "sgemm_dev_download")

    def memset(self, dptr: int, value: int, nbytes: int):
        self._check(self._L.sgemm_dev_memset(self._h, dptr, value, nbytes), "sgemm_dev_memset")

    def sync(self):
        self._check(self._L.sgemm_dev_sync(self._h), "sgemm_dev_sync")


def shard_columns(n: int, world: int, rank: int, tile_n: int = 1) -> Tuple[int, int]:
    """The library's column-shard rule (``sgemm_shard_columns``); ``runner.shard.shard_columns`` restates it in Python."""
    n0, n1 = _u32(), _u32()
    rc = lib().sgemm_shard_columns(n, world, rank, tile_n, ctypes.byref(n0), ctypes.byref(n1))
    if rc:
        raise SgemmError(rc, "sgemm_shard_columns", "bad shard request")
    return n0.value, n1.value


def comm_unique_id() -> bytes:
    """Id of a new communicator (128 bytes): one rank makes it, the host program hands it to all ranks."""
    buf = ctypes.create_string_buffer(128)
    rc = lib().sgemm_comm_unique_id(buf)
    if rc:
        raise SgemmError(rc, "sgemm_comm_unique_id", lib().sgemm_last_error(None).decode())
    return buf.raw


def comm_init_all(runners) -> None:
    """One process, several ``SgemmRunner`` on distinct GPUs: one communicator over them, runner i = rank i."""
    arr = (_vp * len(runners))(*[r._h for r in runners])
    rc = lib().sgemm_comm_init_all(arr, len(runners))
    if rc:
        raise SgemmError(rc, "sgemm_comm_init_all", lib().sgemm_last_error(runners[0]._h).decode())


def noalloc_scratch_bytes() -> int:
    return int(lib().sgemm_noalloc_scratch_bytes())


def device_count() -> int:
    return int(lib().sgemm_device_count())
