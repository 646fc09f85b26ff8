"""ctypes binding of libactcomp.so (the C ABI declared in include/actcomp.h).

The shared library is the only compute path: if it is missing, importing this
module raises, and every op raises ``RuntimeError`` on a non-zero status.  There
is no CPU fallback.
"""
from __future__ import annotations

import ctypes
import os
import threading

_HERE = os.path.dirname(os.path.abspath(__file__))
#: the in-tree build; ACTCOMP_LIBRARY names another build of the same sources instead
LIB_PATH = os.environ.get("ACTCOMP_LIBRARY") or os.path.join(_HERE, "libactcomp.so")

c_i64 = ctypes.c_int64
c_i32 = ctypes.c_int32
c_vp = ctypes.c_void_p

ABI_VERSION = 2  # ACTCOMP_ABI_VERSION in include/actcomp.h

ACT_OK = 0
ACT_E_INVALID = -1
ACT_E_UNSUPPORTED = -2
ACT_E_ALIGN = -3
ACT_E_CUDA = -4
ACT_E_NODEVICE = -5
ACT_E_WORKSPACE = -6
ACT_E_TIMEOUT = -7
ACT_E_BOUNDS = -8

ACT_OP_DECODE = 0
ACT_OP_MUL = 1
ACT_OP_SILU_BWD = 2
ACT_OP_GELU_BWD = 3

ACT_RC_TWIN_LOWRANK = 1
ACT_RC_HALF_EVEN = 2
ACT_RC_SCALE_BATCH = 4
ACT_RC_ROW_PACK = 8
ACT_RC_OUTLIER_BF16 = 16


MX4_LINEAR_TOKENS = 4  # ACTCOMP_MX4_LINEAR_TOKENS


class CgDesc(ctypes.Structure):
    _fields_ = [
        ("tokens", c_i64), ("channels", c_i64),
        ("bits", c_i32), ("group", c_i32), ("rank", c_i32), ("n_outlier", c_i32), ("wht", c_i32), ("batch", c_i32),
        ("codes", c_vp), ("scales", c_vp), ("lowrank", c_vp), ("outliers", c_vp), ("outlier_idx", c_vp),
        ("basis_t", c_vp), ("basis", c_vp), ("basis_tile", c_vp),
    ]


class RcArgs(ctypes.Structure):
    _fields_ = [
        ("B", c_i64), ("M", c_i64), ("N", c_i64),
        ("K", c_i32), ("bits", c_i32), ("flags", c_i32), ("outlier", ctypes.c_float),
        ("l", c_vp), ("r", c_vp), ("s", c_vp), ("s_rows", c_i64),
        ("x", c_vp), ("sxb", c_i64), ("sxm", c_i64),
        ("o", c_vp), ("q", c_vp), ("out", c_vp),
    ]


class EwArgs(ctypes.Structure):
    _fields_ = [
        ("B", c_i64), ("M", c_i64), ("N", c_i64),
        ("x", c_vp), ("sxb", c_i64), ("sxm", c_i64),
        ("g", c_vp), ("sgb", c_i64), ("sgm", c_i64),
        ("out", c_vp), ("sob", c_i64), ("som", c_i64),
    ]


class GemmArgs(ctypes.Structure):
    _fields_ = [
        ("M", c_i64), ("N", c_i64), ("K", c_i64),
        ("batch", c_i32), ("in_dtype", c_i32), ("c_dtype", c_i32), ("activation", c_i32),
        ("a_kmajor", c_i32), ("b_kmajor", c_i32),
        ("A", c_vp), ("lda", c_i64), ("sa_batch", c_i64),
        ("B", c_vp), ("ldb", c_i64), ("sb_batch", c_i64),
        ("C", c_vp), ("ldc", c_i64), ("sc_batch", c_i64),
        ("K2", c_i64), ("A2", c_vp), ("lda2", c_i64), ("B2", c_vp), ("ldb2", c_i64),
    ]


class DropArgs(ctypes.Structure):
    _fields_ = [
        ("rows", c_i64), ("cols", c_i64), ("x", c_vp), ("ldx", c_i64), ("y", c_vp), ("ldy", c_i64),
        ("dtype", c_i32), ("reserved", c_i32), ("p", ctypes.c_double), ("seed", ctypes.c_uint64),
        ("seed_ptr", c_vp), ("row_offset", ctypes.c_uint64),
    ]


class LnArgs(ctypes.Structure):
    _fields_ = [
        ("rows", c_i64), ("cols", c_i64), ("x", c_vp), ("ldx", c_i64), ("res", c_vp), ("ldr", c_i64),
        ("weight", c_vp), ("bias", c_vp), ("y", c_vp), ("ldy", c_i64), ("h", c_vp), ("ldh", c_i64),
        ("mean", c_vp), ("rstd", c_vp), ("dtype", c_i32), ("wdtype", c_i32), ("eps", ctypes.c_float),
        ("reserved", c_i32), ("p", ctypes.c_double), ("seed", ctypes.c_uint64), ("seed_ptr", c_vp),
        ("row_offset", ctypes.c_uint64),
    ]


class LnBwdArgs(ctypes.Structure):
    _fields_ = [
        ("rows", c_i64), ("cols", c_i64), ("dy", c_vp), ("lddy", c_i64), ("x", c_vp), ("ldx", c_i64),
        ("dh", c_vp), ("lddh", c_i64), ("weight", c_vp), ("mean", c_vp), ("rstd", c_vp), ("dx", c_vp), ("lddx", c_i64),
        ("dr", c_vp), ("lddr", c_i64), ("dweight", c_vp), ("dbias", c_vp), ("dtype", c_i32), ("wdtype", c_i32),
        ("p", ctypes.c_double), ("seed", ctypes.c_uint64), ("seed_ptr", c_vp), ("row_offset", ctypes.c_uint64),
    ]


class Mx4Desc(ctypes.Structure):
    _fields_ = [("rows", c_i64), ("cols", c_i64), ("codes", c_vp), ("scales", c_vp)]


#: entry point -> (restype, argtypes); mirrors include/actcomp.h
SIGNATURES = {
    "actcomp_strerror": (ctypes.c_char_p, [ctypes.c_int]),
    "actcomp_abi_version": (ctypes.c_int, []),
    "actcomp_last_device_error": (ctypes.c_int, [c_vp, ctypes.POINTER(ctypes.c_uint32)]),
    "actcomp_clear_device_error": (ctypes.c_int, [c_vp]),
    "actcomp_selftest_bounded_wait": (ctypes.c_int, [ctypes.c_uint32, c_i32, c_vp]),
    "actcomp_cg_basis_prepare": (ctypes.c_int, [c_vp, c_i64, c_i32, c_i32, c_vp, c_vp, c_vp, c_vp]),
    "actcomp_cg_encode": (ctypes.c_int, [ctypes.POINTER(CgDesc), c_vp, c_i64, c_vp]),
    "actcomp_cg_decode": (ctypes.c_int, [ctypes.POINTER(CgDesc), c_vp, c_i64, c_vp]),
    "actcomp_cg_consume": (ctypes.c_int, [ctypes.POINTER(CgDesc), c_i32, c_vp, c_i64, c_vp, c_i64, c_vp]),
    "actcomp_cg_softmax_workspace": (ctypes.c_size_t, [ctypes.POINTER(CgDesc)]),
    "actcomp_cg_softmax_bwd": (ctypes.c_int, [ctypes.POINTER(CgDesc), c_vp, c_vp, c_i64, c_i32, c_vp,
                                              ctypes.c_size_t, c_vp]),
    "actcomp_cg_dw_workspace": (ctypes.c_size_t, [ctypes.POINTER(CgDesc), c_i64]),
    "actcomp_cg_dw": (ctypes.c_int, [ctypes.POINTER(CgDesc), c_vp, c_i64, c_i64, c_vp, c_i32, c_i64, c_vp,
                                     ctypes.c_size_t, c_vp]),
    "actcomp_cg_dw_fused_workspace": (ctypes.c_size_t, [ctypes.POINTER(CgDesc), c_i64]),
    "actcomp_cg_dw_fused": (ctypes.c_int, [ctypes.POINTER(CgDesc), c_vp, c_i64, c_i64, c_vp, c_i32, c_i64, c_vp,
                                           ctypes.c_size_t, c_vp]),
    "actcomp_cg_dw_static": (ctypes.c_int, [ctypes.POINTER(CgDesc), c_vp, c_i64, c_i64, c_vp, c_i32, c_i64, c_vp]),
    "actcomp_cg_channel_topk": (ctypes.c_int, [c_vp, c_i64, c_i64, c_i64, c_i32, c_vp, c_vp, c_vp]),
    "actcomp_cg_copy": (ctypes.c_int, [ctypes.POINTER(CgDesc), ctypes.POINTER(CgDesc), c_vp]),
    "actcomp_rc_encode": (ctypes.c_int, [ctypes.POINTER(RcArgs), c_vp]),
    "actcomp_rc_decode": (ctypes.c_int, [ctypes.POINTER(RcArgs), c_i32, c_vp]),
    "actcomp_rc_lowrank_add": (ctypes.c_int, [ctypes.POINTER(RcArgs), c_vp]),
    "actcomp_elementwise": (ctypes.c_int, [ctypes.POINTER(EwArgs), c_i32, c_vp]),
    "actcomp_softmax_bwd": (ctypes.c_int, [c_vp, c_vp, c_vp, c_i64, c_i64, c_i64, c_vp]),
    "actcomp_extract_unstructured": (ctypes.c_int, [c_vp, c_i64, ctypes.c_float, c_vp, c_vp, c_vp]),
    "actcomp_extract_channel": (ctypes.c_int, [c_vp, c_i64, c_i64, c_i64, c_vp, c_i32, c_vp, c_vp]),
    "actcomp_gemm": (ctypes.c_int, [ctypes.POINTER(GemmArgs), c_vp]),
    "actcomp_error_stats": (ctypes.c_int, [c_vp, c_vp, c_i64, c_vp, c_vp]),
    "actcomp_nf4_dequant": (ctypes.c_int, [c_vp, c_i64, c_i64, c_vp, c_vp, c_vp, c_vp, c_vp, c_i64,
                                           c_vp, c_vp, c_vp]),
    "actcomp_dropout": (ctypes.c_int, [ctypes.POINTER(DropArgs), c_vp]),
    "actcomp_layer_norm": (ctypes.c_int, [ctypes.POINTER(LnArgs), c_vp]),
    "actcomp_layer_norm_bwd_workspace": (ctypes.c_size_t, [c_i64, c_i64]),
    "actcomp_layer_norm_bwd": (ctypes.c_int, [ctypes.POINTER(LnBwdArgs), c_vp, ctypes.c_size_t, c_vp]),
    "actcomp_selftest_row_waits": (ctypes.c_int, [c_vp, c_i32, c_i32, ctypes.c_uint32, c_vp, c_vp]),
    "actcomp_mx4_code_bytes": (ctypes.c_size_t, [c_i64, c_i64]),
    "actcomp_mx4_scale_bytes": (ctypes.c_size_t, [c_i64, c_i64]),
    "actcomp_mx4_quantize": (ctypes.c_int, [c_vp, c_i64, c_i64, c_i64, c_i32, ctypes.POINTER(Mx4Desc),
                                            ctypes.POINTER(Mx4Desc), c_vp]),
    "actcomp_mx4_dequantize": (ctypes.c_int, [ctypes.POINTER(Mx4Desc), c_vp, c_i64, c_i32, c_vp]),
    "actcomp_mx4_linear": (ctypes.c_int, [c_vp, c_i64, c_i64, c_i64, c_i32, ctypes.POINTER(Mx4Desc), c_vp, c_i64,
                                          c_i32, c_vp]),
    "actcomp_mx4_gemm": (ctypes.c_int, [ctypes.POINTER(Mx4Desc), ctypes.POINTER(Mx4Desc), c_vp, c_i64, c_i32, c_vp]),
}

#: entry points behind :class:`Host`, bound on its first use
_HOST_API = ("actcomp_dropout", "actcomp_layer_norm", "actcomp_mx4_")
#: what another build of the library may lack: the rest of the package does not need them
_OPTIONAL = _HOST_API + ("actcomp_selftest_row_waits",)

_lock = threading.Lock()
_lib = None


def load() -> ctypes.CDLL:
    """Load libactcomp.so (building it first only if ACTCOMP_AUTOBUILD=1)."""
    global _lib
    with _lock:
        if _lib is not None:
            return _lib
        if not os.path.exists(LIB_PATH):
            if os.environ.get("ACTCOMP_AUTOBUILD") == "1":
                from . import build
                build.build()
            else:
                raise ImportError(
                    f"{LIB_PATH} is missing: build it with `python triton-kernel-test_b200/actcomp/build.py` "
                    "(nvcc, sm_100a). actcomp has no CPU fallback.")
        lib = ctypes.CDLL(LIB_PATH)
        for name, (res, args) in SIGNATURES.items():
            if name.startswith(_OPTIONAL) and not hasattr(lib, name):
                continue
            fn = getattr(lib, name)
            fn.restype = res
            fn.argtypes = args
        if lib.actcomp_abi_version() != ABI_VERSION:
            raise ImportError(f"{LIB_PATH}: ABI version {lib.actcomp_abi_version()} != {ABI_VERSION}")
        _lib = lib
        return lib


class ActcompError(RuntimeError):
    def __init__(self, fn: str, status: int):
        msg = load().actcomp_strerror(status).decode()
        super().__init__(f"{fn} failed: {msg} ({status})")
        self.status = status


def check(fn: str, status: int) -> None:
    if status != ACT_OK:
        raise ActcompError(fn, status)


class Host:
    """The extension module that runs the host side of :mod:`actcomp.norm` and
    :mod:`actcomp.mx4` (csrc/host.cpp), loaded and bound to the library by the
    first call of one of its functions: nothing else of the package needs it."""

    _guard = threading.Lock()

    def __getattr__(self, name):  # reached until _load has put the functions here
        with Host._guard:
            if "bind" not in self.__dict__:
                self._load()
        return object.__getattribute__(self, name)

    def _load(self) -> None:
        from importlib import util

        from . import build

        lib = load()
        path = build.host_path()
        if not os.path.exists(path):
            if os.environ.get("ACTCOMP_AUTOBUILD") != "1":
                raise ImportError(f"{path} is missing: build it with `python triton-kernel-test_b200/actcomp/build.py` "
                                  "(a module for another torch or Python does not serve)")
            build.build_host()
        names = [n for n in SIGNATURES if n.startswith(_HOST_API)]
        missing = [n for n in names if not hasattr(lib, n)]
        if missing:
            raise ImportError(f"{LIB_PATH} lacks {', '.join(missing)}")
        spec = util.spec_from_file_location(__package__ + "._host", path)
        module = util.module_from_spec(spec)
        spec.loader.exec_module(module)
        module.bind({n: ctypes.cast(getattr(lib, n), c_vp).value for n in names})
        self.__dict__.update({k: v for k, v in vars(module).items() if not k.startswith("__")})


host = Host()


def call(name: str, *args) -> None:
    check(name, getattr(load(), name)(*args))
