"""Binding of the block operators' C ABI (include/qmm_block.h).

The argument structs travel as packed bytes (struct.Struct in native layout):
one object per call instead of a ctypes structure, since a small operator's time
is the time of its call.
"""
from __future__ import annotations

import ctypes
import importlib.util
import struct
import warnings

import torch

from . import _lib
from . import build as _build
from ._lib import QmmError

ELEM_BF16, ELEM_F32, ELEM_F16 = 0, 1, 2
ELEMS = {torch.bfloat16: ELEM_BF16, torch.float32: ELEM_F32, torch.float16: ELEM_F16}

NORM_NONE, NORM_RMS, NORM_LAYER = 0, 1, 2
NORMS = {None: NORM_NONE, "none": NORM_NONE, "rms": NORM_RMS, "layer": NORM_LAYER}

# Every symbol include/qmm_block.h declares.
EXPORTED_SYMBOLS = (
    "qmm_mx4_code_bytes",
    "qmm_mx4_scale_bytes",
    "qmm_mx4_quantize",
    "qmm_mx4_dequantize",
    "qmm_mx4_tile_scales",
    "qmm_mx4_row_scales",
    "qmm_mx4_workspace_bytes",
    "qmm_mx4_linear_workspace_bytes",
    "qmm_mx4_linear",
    "qmm_qk_norm_rotary",
    "qmm_gated_residual_norm",
)

MX4 = struct.Struct("PPqq")                       # qmm_mx4
LINEAR = struct.Struct("PPqqqPqPPPPPPPQii")       # qmm_mx4_linear_args
ROTARY = struct.Struct("8PPqq12qq8if4x")          # qmm_rotary_args
NORM = struct.Struct("11P10q5iff4x")              # qmm_gated_norm_args

_lib_block = None
_host_module = None


def load() -> ctypes.CDLL:
    """libqmm.so with the block operators' prototypes."""
    global _lib_block
    if _lib_block is None:
        lib = _lib.load()
        vp, i64, i32, args = ctypes.c_void_p, ctypes.c_int64, ctypes.c_int32, ctypes.c_char_p
        for name, restype, argtypes in (
                ("qmm_mx4_code_bytes", ctypes.c_uint64, [i64, i64]),
                ("qmm_mx4_scale_bytes", ctypes.c_uint64, [i64, i64]),
                ("qmm_mx4_workspace_bytes", ctypes.c_uint64, [i64, i64]),
                ("qmm_mx4_linear_workspace_bytes", ctypes.c_uint64, [i64, i64, i64]),
                ("qmm_mx4_quantize", i32, [vp, i32, i64, i64, i64, vp, vp, vp]),
                ("qmm_mx4_dequantize", i32, [args, vp, i32, vp]),
                ("qmm_mx4_tile_scales", i32, [vp, i64, i64, vp, vp]),
                ("qmm_mx4_row_scales", i32, [vp, i64, i64, vp, vp]),
                ("qmm_mx4_linear", i32, [args, vp]),
                ("qmm_qk_norm_rotary", i32, [args, vp]),
                ("qmm_gated_residual_norm", i32, [args, vp])):
            fn = getattr(lib, name)
            fn.restype, fn.argtypes = restype, argtypes
        _lib_block = lib
    return _lib_block


class _General:
    """Stands in for the extension where it cannot be had: every call goes its general way."""

    mx_quantize = mx_dequantize = mx_linear = qk_norm_rotary = gated_norm = staticmethod(lambda *args: None)


def host():
    """The extension with the operators' ordinary calls (csrc/host/block_host.cpp),
    built first when stale: a small operator's time is the time of its call
    (B200, one-token linear: 14 us through the checks here and ctypes).  It only saves
    time: where it cannot be built, a warning says so and the operators run without."""
    global _host_module
    if _host_module is None:
        lib = load()
        try:
            if _build.host_is_stale():  # (never loaded stale: it fills the structs of the headers that it was built from)
                _build.build_host()
            spec = importlib.util.spec_from_file_location("_qmm_host", _build.HOST)
            module = importlib.util.module_from_spec(spec)
            spec.loader.exec_module(module)
        except Exception as exc:
            warnings.warn(f"_qmm_host.so cannot be used, calls of the block operators take longer: {exc}", RuntimeWarning, stacklevel=3)
            _host_module = _General
            return _host_module
        module.bind(*(ctypes.cast(getattr(lib, name), ctypes.c_void_p).value for name in (
            "qmm_mx4_linear", "qmm_mx4_linear_workspace_bytes", "qmm_mx4_quantize", "qmm_mx4_dequantize", "qmm_qk_norm_rotary",
            "qmm_gated_residual_norm")))
        _host_module = module
    return _host_module


def run(name: str, device: torch.device, *args) -> None:
    """Calls entry point `name` on `device` and its current stream."""
    fn = getattr(_lib_block or load(), name)
    index = device.index
    if index == torch._C._cuda_getDevice():
        status = fn(*args, torch._C._cuda_getCurrentRawStream(index))
    else:
        with torch.cuda.device(index):
            status = fn(*args, torch._C._cuda_getCurrentRawStream(index))
    if status:
        _lib.check(status)


def checked(result):
    """What a call of the extension made, or its status raised."""
    if result.__class__ is int:
        _lib.check(result)
    return result


def bad_argument(message: str) -> QmmError:
    return QmmError(_lib.QMM_ERR_INVALID_ARGUMENT, message)


def bad_shape(message: str) -> QmmError:
    return QmmError(_lib.QMM_ERR_BAD_SHAPE, message)


def require_cuda(t: torch.Tensor, what: str) -> torch.device:
    if not t.is_cuda:
        raise QmmError(_lib.QMM_ERR_CUDA, f"{what} is on {t.device}; the operator runs on CUDA only")
    return t.device


def elem_of(t: torch.Tensor, what: str) -> int:
    e = ELEMS.get(t.dtype)
    if e is None:
        raise bad_argument(f"{what} is {t.dtype}; bfloat16, float16 or float32 is needed")
    return e


def rows_of(t: torch.Tensor, cols: int) -> torch.Tensor:
    """t [..., cols] as [rows, cols] with consecutive columns, rows that do not overlap: a view
    where the strides allow, else (columns apart, one row expanded, a sliding window) a copy."""
    if t.dim() != 2:
        t = t.reshape(-1, cols)
    if (t.stride(1) != 1 and cols != 1) or (t.stride(0) < cols and t.shape[0] > 1):
        return t.contiguous()
    return t
