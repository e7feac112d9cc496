"""ctypes binding of the C ABI in ``include/``.

The shared library must have been built (``diffuser_b200.build.build()``);
there is no fallback: loading fails loudly when it is missing.
"""
from __future__ import annotations

import ctypes
import os
import struct

from .build import LIB_PATH

_c_i64 = ctypes.c_int64
_c_p = ctypes.c_void_p
_c_sz = ctypes.c_size_t

# name -> (restype, argtypes); every symbol the header declares.
SIGNATURES = {
    "dq_version": (ctypes.c_char_p, []),
    "dq_abi_version": (ctypes.c_int, []),
    "dq_status_string": (ctypes.c_char_p, [ctypes.c_int]),
    "dq_quantize_nf4": (ctypes.c_int, [_c_p, ctypes.c_int, _c_i64, _c_p, _c_p, _c_p]),
    "dq_quantize_fp8": (ctypes.c_int, [_c_p, ctypes.c_int, _c_i64, _c_p, _c_p, _c_p]),
    "dq_dequant_nf4": (ctypes.c_int, [_c_p, _c_p, _c_i64, _c_p, _c_p]),
    "dq_dequant_fp8": (ctypes.c_int, [_c_p, ctypes.c_float, _c_i64, _c_p, _c_p]),
    "dq_workspace_size": (_c_sz, [_c_i64, _c_i64, _c_i64, ctypes.c_int]),
    "dq_linear_nf4": (ctypes.c_int, [_c_p, _c_i64, _c_i64, _c_p, _c_p, _c_p, _c_i64, _c_p,
                                     _c_p, _c_sz, _c_p]),
    "dq_linear_fp8": (ctypes.c_int, [_c_p, _c_i64, _c_i64, _c_p, ctypes.c_float, _c_p, _c_i64,
                                     _c_p, _c_p, _c_sz, _c_p]),
    "dq_linear_nf4_noalloc": (ctypes.c_int, [_c_p, _c_i64, _c_i64, _c_p, _c_p, _c_p, _c_i64,
                                             _c_p, _c_p]),
    "dq_device_error": (ctypes.c_int, [ctypes.POINTER(ctypes.c_int), _c_p]),
    "dq_set_tile_override": (ctypes.c_int, [ctypes.c_int, ctypes.c_int]),
    "dq_set_pair_mode": (ctypes.c_int, [ctypes.c_int]),
    "dq_tp_buffer_alloc": (ctypes.c_int, [ctypes.c_size_t, ctypes.POINTER(ctypes.c_void_p)]),
    "dq_tp_buffer_free": (ctypes.c_int, [ctypes.c_void_p]),
    "dq_ipc_handle": (ctypes.c_int, [ctypes.c_void_p, ctypes.c_void_p]),
    "dq_ipc_open": (ctypes.c_int, [ctypes.c_void_p, ctypes.POINTER(ctypes.c_void_p)]),
    "dq_ipc_close": (ctypes.c_int, [ctypes.c_void_p]),
    "dq_tp_linear_nf4": (ctypes.c_int, [ctypes.c_void_p, _c_i64, _c_i64, ctypes.c_void_p, ctypes.c_void_p,
                                        ctypes.c_void_p, _c_i64, ctypes.c_int, ctypes.c_int,
                                        ctypes.POINTER(ctypes.c_void_p), ctypes.POINTER(ctypes.c_void_p),
                                        ctypes.c_void_p, ctypes.c_uint, ctypes.c_void_p]),
    "dq_tp_linear_fp8": (ctypes.c_int, [ctypes.c_void_p, _c_i64, _c_i64, ctypes.c_void_p, ctypes.c_float,
                                        ctypes.c_void_p, _c_i64, ctypes.c_int, ctypes.c_int,
                                        ctypes.POINTER(ctypes.c_void_p), ctypes.POINTER(ctypes.c_void_p),
                                        ctypes.c_void_p, ctypes.c_uint, ctypes.c_void_p]),
    "dq_tp_linear_nf4_ws": (ctypes.c_int, [ctypes.c_void_p, _c_i64, _c_i64, ctypes.c_void_p, ctypes.c_void_p,
                                           ctypes.c_void_p, _c_i64, ctypes.c_int, ctypes.c_int,
                                           ctypes.POINTER(ctypes.c_void_p), ctypes.POINTER(ctypes.c_void_p),
                                           ctypes.c_void_p, ctypes.c_uint, ctypes.c_void_p, _c_sz,
                                           ctypes.c_void_p]),
    "dq_tp_linear_fp8_ws": (ctypes.c_int, [ctypes.c_void_p, _c_i64, _c_i64, ctypes.c_void_p, ctypes.c_float,
                                           ctypes.c_void_p, _c_i64, ctypes.c_int, ctypes.c_int,
                                           ctypes.POINTER(ctypes.c_void_p), ctypes.POINTER(ctypes.c_void_p),
                                           ctypes.c_void_p, ctypes.c_uint, ctypes.c_void_p, _c_sz,
                                           ctypes.c_void_p]),
    "dq_tp_linear_nf4_mc_ws": (ctypes.c_int, [ctypes.c_void_p, _c_i64, _c_i64, ctypes.c_void_p,
                                              ctypes.c_void_p, ctypes.c_void_p, _c_i64, ctypes.c_int,
                                              ctypes.c_int, ctypes.POINTER(ctypes.c_void_p), ctypes.c_void_p,
                                              ctypes.POINTER(ctypes.c_void_p), ctypes.c_void_p, ctypes.c_uint,
                                              ctypes.c_void_p, _c_sz, ctypes.c_void_p]),
    "dq_tp_linear_fp8_mc_ws": (ctypes.c_int, [ctypes.c_void_p, _c_i64, _c_i64, ctypes.c_void_p,
                                              ctypes.c_float, ctypes.c_void_p, _c_i64, ctypes.c_int,
                                              ctypes.c_int, ctypes.POINTER(ctypes.c_void_p), ctypes.c_void_p,
                                              ctypes.POINTER(ctypes.c_void_p), ctypes.c_void_p, ctypes.c_uint,
                                              ctypes.c_void_p, _c_sz, ctypes.c_void_p]),
    "dq_qk_norm_rope": (ctypes.c_int, [ctypes.c_void_p, _c_i64, ctypes.c_void_p, _c_i64, ctypes.c_int,
                                       ctypes.c_int, ctypes.c_int, ctypes.c_int, ctypes.c_int,
                                       ctypes.c_void_p, ctypes.c_void_p, ctypes.c_void_p, ctypes.c_void_p,
                                       ctypes.c_float, ctypes.c_void_p, ctypes.c_void_p]),
    "dq_qkv_norm_rope": (ctypes.c_int, [ctypes.c_int, ctypes.POINTER(ctypes.c_void_p),
                                        ctypes.POINTER(_c_i64), ctypes.POINTER(ctypes.c_void_p),
                                        ctypes.POINTER(_c_i64), ctypes.c_int, ctypes.c_int, ctypes.c_int,
                                        ctypes.c_int, ctypes.c_int, ctypes.POINTER(ctypes.c_void_p),
                                        ctypes.POINTER(ctypes.c_void_p), ctypes.POINTER(ctypes.c_int),
                                        ctypes.c_void_p, ctypes.c_void_p, ctypes.c_float,
                                        ctypes.POINTER(ctypes.c_void_p), ctypes.c_void_p]),
    "dq_heads_to_tokens": (ctypes.c_int, [ctypes.c_void_p, ctypes.c_int, ctypes.c_int, ctypes.c_int,
                                          ctypes.c_int, ctypes.c_int, ctypes.c_void_p, ctypes.c_void_p,
                                          ctypes.c_void_p]),
    "dq_linear_nf4_ld": (ctypes.c_int, [ctypes.c_void_p, _c_i64, _c_i64, ctypes.c_void_p, ctypes.c_void_p,
                                        ctypes.c_void_p, _c_i64, ctypes.c_int, ctypes.c_void_p, _c_i64,
                                        ctypes.c_void_p, _c_sz, ctypes.c_void_p]),
    "dq_linear_fp8_ld": (ctypes.c_int, [ctypes.c_void_p, _c_i64, _c_i64, ctypes.c_void_p, ctypes.c_float,
                                        ctypes.c_void_p, _c_i64, ctypes.c_int, ctypes.c_void_p, _c_i64,
                                        ctypes.c_void_p, _c_sz, ctypes.c_void_p]),
    "dq_heads_to_tokens_ld": (ctypes.c_int, [ctypes.c_void_p, ctypes.c_int, ctypes.c_int, ctypes.c_int,
                                             ctypes.c_int, ctypes.c_int, ctypes.c_void_p, _c_i64,
                                             ctypes.c_void_p, _c_i64, ctypes.c_void_p]),
    "dq_adaln_modulate": (ctypes.c_int, [ctypes.c_void_p, _c_i64, _c_i64, ctypes.c_int, ctypes.c_int,
                                         ctypes.c_void_p, ctypes.c_void_p, _c_i64, ctypes.c_float,
                                         ctypes.c_void_p, _c_i64, ctypes.c_void_p]),
    "dq_gated_residual": (ctypes.c_int, [ctypes.c_void_p, _c_i64, ctypes.c_void_p, _c_i64, ctypes.c_void_p,
                                         _c_i64, _c_i64, ctypes.c_int, ctypes.c_int, ctypes.c_void_p, _c_i64,
                                         ctypes.c_void_p]),
    "dq_linear_nf4_ex": (ctypes.c_int, [ctypes.c_void_p, _c_i64, _c_i64, ctypes.c_void_p, ctypes.c_void_p,
                                        ctypes.c_void_p, _c_i64, ctypes.c_int, ctypes.c_void_p,
                                        ctypes.c_void_p, _c_sz, ctypes.c_void_p]),
    "dq_linear_fp8_ex": (ctypes.c_int, [ctypes.c_void_p, _c_i64, _c_i64, ctypes.c_void_p, ctypes.c_float,
                                        ctypes.c_void_p, _c_i64, ctypes.c_int, ctypes.c_void_p,
                                        ctypes.c_void_p, _c_sz, ctypes.c_void_p]),
    "dq_linear_nf4_scaled": (ctypes.c_int, [ctypes.c_void_p, _c_i64, _c_i64, ctypes.c_void_p,
                                            ctypes.c_void_p, ctypes.c_int, ctypes.c_void_p, _c_i64,
                                            ctypes.c_int, ctypes.c_void_p, _c_i64, ctypes.c_void_p,
                                            _c_sz, ctypes.c_void_p]),
    "dq_dequant_nf4_scaled": (ctypes.c_int, [_c_p, _c_p, ctypes.c_int, _c_i64, _c_p, _c_p]),
    "dq_gated_norm": (ctypes.c_int, [_c_p, _c_i64, _c_p, _c_i64, _c_i64, ctypes.c_int, ctypes.c_int, _c_p, _c_i64,
                                     _c_p, _c_p, _c_i64, _c_p, _c_p, ctypes.c_int, ctypes.c_int, ctypes.c_float,
                                     ctypes.c_float, ctypes.c_int, _c_p, _c_i64, _c_p, _c_i64, _c_p]),
    "dq_gated_norm_backward_workspace": (_c_sz, [_c_i64, ctypes.c_int, ctypes.c_int]),
    "dq_gated_norm_backward": (ctypes.c_int, [_c_p, _c_i64, _c_p, _c_i64, _c_p, _c_i64, _c_p, _c_i64, _c_i64,
                                              ctypes.c_int, ctypes.c_int, _c_p, _c_i64, _c_p, _c_i64, _c_p, _c_p,
                                              ctypes.c_int, ctypes.c_int, ctypes.c_float, ctypes.c_float, _c_p,
                                              _c_i64, _c_p, _c_i64, _c_p, _c_p, _c_p, _c_p, _c_p, _c_p, _c_sz,
                                              _c_p]),
    "dq_adapter_plan_bytes": (_c_sz, [_c_i64, _c_i64, ctypes.c_int]),
    "dq_adapter_plan": (ctypes.c_int, [_c_p, _c_p, _c_i64, _c_i64, ctypes.c_int, _c_p, _c_sz, _c_p]),
    "dq_adapter_add_workspace": (_c_sz, [_c_i64, _c_i64, ctypes.c_int, ctypes.c_int]),
    "dq_adapter_add": (ctypes.c_int, [_c_p, _c_i64, _c_p, _c_i64, _c_i64, _c_i64, _c_i64, _c_i64, _c_p, _c_p, _c_p,
                                      ctypes.c_int, ctypes.c_int, _c_p, ctypes.c_int, _c_p, _c_i64, _c_p, _c_p,
                                      _c_sz, _c_p]),
    "dq_adapter_backward_workspace": (_c_sz, [_c_i64, _c_i64, _c_i64, _c_i64, ctypes.c_int, ctypes.c_int]),
    "dq_adapter_backward": (ctypes.c_int, [_c_p, _c_i64, _c_p, _c_i64, _c_p, _c_p, _c_i64, _c_i64, _c_i64, _c_i64,
                                           _c_p, _c_p, _c_p, ctypes.c_int, ctypes.c_int, _c_p, _c_p, _c_i64, _c_p,
                                           _c_i64, _c_p, _c_p, _c_p, _c_sz, _c_p]),
    "dq_checkpoint_pack": (ctypes.c_int, [_c_p, _c_i64, _c_i64, _c_i64, _c_p, _c_p, _c_p]),
    "dq_checkpoint_unpack": (ctypes.c_int, [_c_p, _c_p, _c_i64, _c_i64, _c_p, _c_i64, _c_p]),
    "dq_linear_dgrad_workspace": (_c_sz, [_c_i64, _c_i64]),
    "dq_linear_dgrad_workspace_for": (_c_sz, [_c_i64, _c_i64, _c_i64]),
    "dq_linear_nf4_dgrad": (ctypes.c_int, [_c_p, _c_i64, _c_i64, _c_p, _c_p, ctypes.c_int, _c_i64, _c_p, _c_p,
                                           _c_sz, _c_p]),
    "dq_linear_fp8_dgrad": (ctypes.c_int, [_c_p, _c_i64, _c_i64, _c_p, ctypes.c_float, _c_i64, _c_p, _c_p, _c_sz,
                                           _c_p]),
    "dq_plan_info": (ctypes.c_int, [_c_i64, _c_i64, _c_i64, ctypes.c_int] + [ctypes.POINTER(ctypes.c_int)] * 4),
}

# Entries that call() reaches through their packed form (include/dq_packed.h):
# one string of 8-byte words instead of an argument list, which ctypes converts
# one by one.
PACKED = ("dq_adapter_add", "dq_adapter_backward", "dq_checkpoint_pack", "dq_checkpoint_unpack",
          "dq_linear_nf4_dgrad", "dq_linear_fp8_dgrad", "dq_gated_norm", "dq_gated_norm_backward")
SIGNATURES.update({name + "_packed": (ctypes.c_int, [ctypes.c_char_p]) for name in PACKED})
_CALLS: dict = {}  # name -> (function, packer)

DQ_OK = 0
DQ_ERR_TIMEOUT = 5
DQ_ERR_SCRATCH_LIMIT = 9
DQ_ERR_INDEX = 10
DQ_NOALLOC_SCRATCH_BYTES = 8 << 20
DQ_IPC_HANDLE_BYTES = 64
DQ_ACT_NONE, DQ_ACT_GELU_TANH, DQ_ACT_SWIGLU, DQ_ACT_GEGLU_TANH = 0, 1, 2, 3
DQ_FMT_NF4, DQ_FMT_FP8 = 0, 1
DQ_DTYPE_F32, DQ_DTYPE_BF16 = 0, 1
DQ_NORM_NONE, DQ_NORM_RMS, DQ_NORM_LAYER = 0, 1, 2
DQ_ROUND_ONCE, DQ_ROUND_OPS = 0, 1

_LIB = None


class DqError(RuntimeError):
    """A non-zero dq_status returned by the engine."""

    def __init__(self, fn: str, status: int):
        self.status = status
        super().__init__(f"{fn} failed: status {status} ({status_string(status)})")


def lib() -> ctypes.CDLL:
    global _LIB
    if _LIB is None:
        if not os.path.exists(LIB_PATH):
            raise RuntimeError(
                f"engine library {LIB_PATH} is missing: build it with "
                "`python -m diffuser_b200.build` (no CPU fallback exists)")
        h = ctypes.CDLL(LIB_PATH)
        for name, (res, args) in SIGNATURES.items():
            fn = getattr(h, name)
            fn.restype = res
            fn.argtypes = args
        for name in PACKED:
            form = "=" + "".join("d" if t is ctypes.c_float else "q" for t in SIGNATURES[name][1])
            _CALLS[name] = getattr(h, name + "_packed"), struct.Struct(form).pack
        _LIB = h
    return _LIB


def status_string(status: int) -> str:
    return lib().dq_status_string(int(status)).decode()


def check(fn: str, status: int) -> None:
    if status != DQ_OK:
        raise DqError(fn, status)


def call(name: str, *args) -> None:
    """The entry `name` of PACKED with its arguments (0 for a null pointer)."""
    if _LIB is None:
        lib()
    fn, pack = _CALLS[name]
    status = fn(pack(*args))
    if status != DQ_OK:
        raise DqError(name, status)


def version() -> str:
    return lib().dq_version().decode()
