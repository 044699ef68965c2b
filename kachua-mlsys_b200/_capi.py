"""ctypes view of the C ABI in include/gdn_b200.h.

This is the thin host binding that replaces the reference's
``solution/cuda/binding.py`` (a torch cpp_extension JIT load, binding.py:20-31):
it loads the prebuilt ``lib/libgdn_b200.so`` and passes plain device pointers,
sizes and the current torch stream.  There is no CPU fallback: if the library
cannot be loaded the call raises.
"""
from __future__ import annotations

import ctypes
import struct
import threading

from . import _build

GDN_OK = 0
GDN_SEQLENS_INT32 = 0
GDN_SEQLENS_INT64 = 1
GDN_ERR_OVERLAP = 8
GDN_ERR_DEVICE_BAD_SEQLENS = 16
GDN_ERR_DEVICE_TIMEOUT = 32

# Every symbol include/gdn_b200.h declares.
EXPORTED_SYMBOLS = (
    "gdn_decode_launch",
    "gdn_prefill_workspace_size",
    "gdn_prefill_launch",
    "gdn_status_string",
    "gdn_read_device_status",
    "gdn_abi_version",
    "gdn_mma_selftest",
    "gdn_prefill_launch_noalloc",
    "gdn_decode_launch_host_staged",
    "gdn_decode_launch_tokens",
    "gdn_decode_launch_bf16_state",
    "gdn_decode_launch_heads",
    "gdn_prefill_launch_heads",
    "gdn_prefill_workspace_size_heads",
    "gdn_prefill_cp_workspace_size",
    "gdn_prefill_cp_summary_offset",
    "gdn_prefill_cp_launch",
    "gdn_scan_launch",
    "gdn_scan_checkpoint_rows",
    "gdn_scan_backward_launch",
    "gdn_scan_step_launch",
    "gdn_add_norm_launch",
    "gdn_add_norm_backward_workspace_size",
    "gdn_add_norm_backward_launch",
    "gdn_gated_norm_launch",
    "gdn_gated_norm_check",
    "gdn_gated_norm_backward_workspace_size",
    "gdn_gated_norm_backward_launch",
)
ABI_VERSION = 11
DTYPE_BF16, DTYPE_F16, DTYPE_F32 = 0, 1, 2
QUANT_NONE, QUANT_ROW, QUANT_GROUP = 0, 1, 2
PATH_AUTO, PATH_RECURRENT, PATH_CHUNKED, PATH_SEGMENTED = 0, 1, 2, 3
MMA_KIND_BF16, MMA_KIND_TF32, MMA_KIND_F16 = 1, 2, 3
MMA_A_MN, MMA_B_MN, MMA_D_LANE16, MMA_A_TMEM, MMA_NO_COMPLETION = 1, 2, 4, 8, 16


class GdnDecodeArgs(ctypes.Structure):
    _fields_ = [
        ("q", ctypes.c_void_p),
        ("k", ctypes.c_void_p),
        ("v", ctypes.c_void_p),
        ("state", ctypes.c_void_p),
        ("A_log", ctypes.c_void_p),
        ("a", ctypes.c_void_p),
        ("dt_bias", ctypes.c_void_p),
        ("b", ctypes.c_void_p),
        ("output", ctypes.c_void_p),
        ("new_state", ctypes.c_void_p),
        ("batch", ctypes.c_int64),
        ("scale", ctypes.c_float),
    ]


class GdnPrefillArgs(ctypes.Structure):
    _fields_ = [
        ("q", ctypes.c_void_p),
        ("k", ctypes.c_void_p),
        ("v", ctypes.c_void_p),
        ("state", ctypes.c_void_p),
        ("A_log", ctypes.c_void_p),
        ("a", ctypes.c_void_p),
        ("dt_bias", ctypes.c_void_p),
        ("b", ctypes.c_void_p),
        ("cu_seqlens", ctypes.c_void_p),
        ("cu_seqlens_dtype", ctypes.c_int32),
        ("path", ctypes.c_int32),
        ("total_tokens", ctypes.c_int64),
        ("num_seqs", ctypes.c_int64),
        ("scale", ctypes.c_float),
        ("output", ctypes.c_void_p),
        ("new_state", ctypes.c_void_p),
    ]


class GdnScanArgs(ctypes.Structure):
    _fields_ = [
        ("x", ctypes.c_void_p),
        ("a", ctypes.c_void_p),
        ("b", ctypes.c_void_p),
        ("x_stride", ctypes.c_int64),
        ("a_stride", ctypes.c_int64),
        ("b_stride", ctypes.c_int64),
        ("A_log", ctypes.c_void_p),
        ("dt_bias", ctypes.c_void_p),
        ("state", ctypes.c_void_p),
        ("cu_seqlens", ctypes.c_void_p),
        ("cu_seqlens_dtype", ctypes.c_int32),
        ("dtype", ctypes.c_int32),
        ("total_tokens", ctypes.c_int64),
        ("num_seqs", ctypes.c_int64),
        ("channels", ctypes.c_int64),
        ("output", ctypes.c_void_p),
        ("output_stride", ctypes.c_int64),
        ("new_state", ctypes.c_void_p),
        ("checkpoints", ctypes.c_void_p),
    ]


class GdnScanGradArgs(ctypes.Structure):
    _fields_ = [
        ("d_output", ctypes.c_void_p),
        ("d_output_stride", ctypes.c_int64),
        ("d_new_state", ctypes.c_void_p),
        ("dx", ctypes.c_void_p),
        ("da", ctypes.c_void_p),
        ("db", ctypes.c_void_p),
        ("dx_stride", ctypes.c_int64),
        ("da_stride", ctypes.c_int64),
        ("db_stride", ctypes.c_int64),
        ("dA_log", ctypes.c_void_p),
        ("d_dt_bias", ctypes.c_void_p),
        ("d_state", ctypes.c_void_p),
    ]


class GdnAddNormArgs(ctypes.Structure):
    _fields_ = [
        ("x", ctypes.c_void_p),
        ("residual", ctypes.c_void_p),
        ("x_stride", ctypes.c_int64),
        ("residual_stride", ctypes.c_int64),
        ("weight", ctypes.c_void_p),
        ("weight_dtype", ctypes.c_int32),
        ("dtype", ctypes.c_int32),
        ("quant", ctypes.c_int32),
        ("eps", ctypes.c_float),
        ("rows", ctypes.c_int64),
        ("width", ctypes.c_int64),
        ("output", ctypes.c_void_p),
        ("new_residual", ctypes.c_void_p),
        ("scale", ctypes.c_void_p),
    ]


class GdnGatedNormArgs(ctypes.Structure):
    _fields_ = [
        ("x", ctypes.c_void_p),
        ("z", ctypes.c_void_p),
        ("x_stride", ctypes.c_int64),
        ("z_stride", ctypes.c_int64),
        ("weight", ctypes.c_void_p),
        ("weight_dtype", ctypes.c_int32),
        ("dtype", ctypes.c_int32),
        ("quant", ctypes.c_int32),
        ("eps", ctypes.c_float),
        ("tokens", ctypes.c_int64),
        ("heads", ctypes.c_int32),
        ("head_dim", ctypes.c_int32),
        ("output", ctypes.c_void_p),
        ("scale", ctypes.c_void_p),
    ]


class GdnNormGradArgs(ctypes.Structure):
    _fields_ = [
        ("d_output", ctypes.c_void_p),
        ("d_output_stride", ctypes.c_int64),
        ("d_new_residual", ctypes.c_void_p),
        ("d_new_residual_stride", ctypes.c_int64),
        ("dx", ctypes.c_void_p),
        ("dz", ctypes.c_void_p),
        ("d_weight", ctypes.c_void_p),
    ]


def packer(struct_type):
    """``pack(*fields) -> bytes`` of a structure above, an integer for every
    pointer (0 for NULL): a third of what building the ctypes object costs."""
    codes = {ctypes.c_void_p: "Q", ctypes.c_int64: "q", ctypes.c_int32: "i", ctypes.c_float: "f"}
    pack = struct.Struct("@" + "".join(codes[t] for _, t in struct_type._fields_))
    tail = ctypes.sizeof(struct_type) - pack.size
    return pack.pack if not tail else struct.Struct(pack.format + f"{tail}x").pack


class GdnError(RuntimeError):
    """A gdn_status_t other than GDN_OK returned by the C ABI."""

    def __init__(self, status: int, what: str):
        self.status = status
        super().__init__(f"{what}: {status_string(status)} (status {status})")


class GdnArgumentError(GdnError, ValueError):
    """A status that says what is wrong with the call's arguments: nothing was launched."""


# NULL_POINTER, BAD_SIZE, MISALIGNED, WORKSPACE, BAD_DTYPE, OVERLAP
ARGUMENT_ERRORS = (1, 2, 3, 4, 6, GDN_ERR_OVERLAP)

_lib = None
_lock = threading.Lock()


def load(build_if_needed: bool = True) -> ctypes.CDLL:
    """Load (building first if needed) the C-ABI library and declare its signatures."""
    global _lib
    if _lib is not None:
        return _lib
    with _lock:
        if _lib is not None:
            return _lib
        if build_if_needed:
            _build.build()
        if not _build.LIB_PATH.exists():
            raise RuntimeError(f"{_build.LIB_PATH} is missing; run __graft_entry__.build()")
        lib = ctypes.CDLL(str(_build.LIB_PATH))
        P = ctypes.c_void_p
        lib.gdn_decode_launch.argtypes = [ctypes.POINTER(GdnDecodeArgs), P]
        lib.gdn_decode_launch.restype = ctypes.c_int
        lib.gdn_decode_launch_host_staged.argtypes = [ctypes.POINTER(GdnDecodeArgs), ctypes.POINTER(GdnDecodeArgs),
                                                      ctypes.c_int, P]
        lib.gdn_decode_launch_host_staged.restype = ctypes.c_int
        lib.gdn_decode_launch_tokens.argtypes = [ctypes.POINTER(GdnDecodeArgs), ctypes.c_int64, P]
        lib.gdn_decode_launch_tokens.restype = ctypes.c_int
        lib.gdn_decode_launch_bf16_state.argtypes = [ctypes.POINTER(GdnDecodeArgs), P]
        lib.gdn_decode_launch_bf16_state.restype = ctypes.c_int
        lib.gdn_decode_launch_heads.argtypes = [ctypes.POINTER(GdnDecodeArgs), ctypes.c_int32, ctypes.c_int32,
                                                ctypes.c_int64, ctypes.c_int32, P]
        lib.gdn_decode_launch_heads.restype = ctypes.c_int
        lib.gdn_prefill_launch_heads.argtypes = [ctypes.POINTER(GdnPrefillArgs), ctypes.c_int32, ctypes.c_int32, P,
                                                 ctypes.c_size_t, P]
        lib.gdn_prefill_launch_heads.restype = ctypes.c_int
        lib.gdn_prefill_workspace_size_heads.argtypes = [ctypes.c_int64, ctypes.c_int64, ctypes.c_int32]
        lib.gdn_prefill_workspace_size_heads.restype = ctypes.c_size_t
        lib.gdn_prefill_cp_workspace_size.argtypes = [ctypes.c_int64, ctypes.c_int64, ctypes.c_int32]
        lib.gdn_prefill_cp_workspace_size.restype = ctypes.c_size_t
        lib.gdn_prefill_cp_summary_offset.argtypes = [ctypes.c_int64, ctypes.c_int64]
        lib.gdn_prefill_cp_summary_offset.restype = ctypes.c_size_t
        lib.gdn_prefill_cp_launch.argtypes = [ctypes.POINTER(GdnPrefillArgs), P, ctypes.c_size_t, ctypes.c_int32,
                                              ctypes.c_int32, ctypes.c_int32, P]
        lib.gdn_prefill_cp_launch.restype = ctypes.c_int
        lib.gdn_prefill_workspace_size.argtypes = [ctypes.c_int64, ctypes.c_int64]
        lib.gdn_prefill_workspace_size.restype = ctypes.c_size_t
        lib.gdn_prefill_launch.argtypes = [ctypes.POINTER(GdnPrefillArgs), P, ctypes.c_size_t, P]
        lib.gdn_prefill_launch.restype = ctypes.c_int
        lib.gdn_status_string.argtypes = [ctypes.c_int]
        lib.gdn_status_string.restype = ctypes.c_char_p
        lib.gdn_read_device_status.argtypes = [ctypes.POINTER(ctypes.c_int), ctypes.c_int, P]
        lib.gdn_read_device_status.restype = ctypes.c_int
        lib.gdn_abi_version.argtypes = []
        lib.gdn_abi_version.restype = ctypes.c_int
        lib.gdn_mma_selftest.argtypes = [ctypes.c_int] * 5 + [P, P, P, P]
        lib.gdn_mma_selftest.restype = ctypes.c_int
        i64, size = ctypes.c_int64, ctypes.c_size_t
        scan = norm = gated = scan_grad = norm_grad = P  # byref() of a structure, or its packed bytes
        for name, restype, argtypes in (
                ("gdn_scan_launch", ctypes.c_int, [scan, P]),
                ("gdn_scan_checkpoint_rows", i64, [i64]),
                ("gdn_scan_backward_launch", ctypes.c_int, [scan, scan_grad, P]),
                ("gdn_scan_step_launch", ctypes.c_int, [scan, i64, P]),
                ("gdn_add_norm_launch", ctypes.c_int, [norm, P]),
                ("gdn_add_norm_backward_workspace_size", size, [i64, i64]),
                ("gdn_add_norm_backward_launch", ctypes.c_int, [norm, norm_grad, P, size, P]),
                ("gdn_gated_norm_launch", ctypes.c_int, [gated, P]),
                ("gdn_gated_norm_check", ctypes.c_int, [gated]),
                ("gdn_gated_norm_backward_workspace_size", size, [i64, ctypes.c_int32, ctypes.c_int32]),
                ("gdn_gated_norm_backward_launch", ctypes.c_int, [gated, norm_grad, P, size, P])):
            getattr(lib, name).restype = restype
            getattr(lib, name).argtypes = argtypes
        if lib.gdn_abi_version() != ABI_VERSION:
            raise RuntimeError("libgdn_b200.so ABI version mismatch; rebuild it")
        _lib = lib
        return lib


def status_string(status: int) -> str:
    try:
        return load(build_if_needed=False).gdn_status_string(int(status)).decode()
    except Exception:  # library not loadable: still give a readable message
        return f"status {status}"


def check(status: int, what: str) -> None:
    if status != GDN_OK:
        raise (GdnArgumentError if status in ARGUMENT_ERRORS else GdnError)(status, what)


def read_device_status(stream_handle: int, clear: bool = True) -> int:
    out = ctypes.c_int(0)
    check(load().gdn_read_device_status(ctypes.byref(out), int(clear), ctypes.c_void_p(stream_handle)),
          "gdn_read_device_status")
    return out.value
