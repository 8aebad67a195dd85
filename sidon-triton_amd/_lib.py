"""ctypes binding of libsidon_flexrel.so (the C ABI in include/sidon_flexrel.h,
include/sidon_encoder.h and include/sidon_operators.h).

There is no fallback: if the library is missing or fails to load, every entry
point raises.  The library is built by ``build.py`` (or ``__graft_entry__.build()``).
"""

from __future__ import annotations

import ctypes
from pathlib import Path

import torch

LIB_PATH = Path(__file__).resolve().parent / "libsidon_flexrel.so"

SIDON_OK = 0
ERROR_NAMES = {
    -1: "SIDON_E_NULL",
    -2: "SIDON_E_SHAPE",
    -3: "SIDON_E_STRIDE",
    -4: "SIDON_E_ALIGN",
    -5: "SIDON_E_LAUNCH",
    -6: "SIDON_E_DEVICE",
    -7: "SIDON_E_CONFIG",
}

# Every symbol include/*.h declares, with its ctypes signature.
_I64P = ctypes.POINTER(ctypes.c_int64)
_IP = ctypes.POINTER(ctypes.c_int)
_VP = ctypes.c_void_p
SIGNATURES = {
    "sidon_flexrel_fwd": (ctypes.c_int, [_VP, _VP, _VP, _VP, _VP, _VP, ctypes.c_int, ctypes.c_int,
                                         ctypes.c_int, ctypes.c_int, _I64P, _I64P, _I64P, _I64P, _VP]),
    "sidon_flexrel_fwd_qkv": (ctypes.c_int, [_VP, _VP, _VP, _VP, ctypes.c_int, ctypes.c_int,
                                             ctypes.c_int, _VP]),
    "sidon_flexrel_launch_shape": (ctypes.c_int, [ctypes.c_int, ctypes.c_int, ctypes.c_int, _IP, _IP,
                                                  _IP, _IP]),
    "sidon_flexrel_debug_rerun_all": (None, [ctypes.c_int]),
    "sidon_res_norm": (ctypes.c_int, [_VP, _VP, _VP, _VP, _VP, ctypes.c_float, ctypes.c_int, _VP, _VP,
                                      ctypes.c_float, _VP, ctypes.c_int, ctypes.c_int, ctypes.c_int, _VP]),
    "sidon_res_norm_parts": (ctypes.c_int, [_VP, _VP, ctypes.c_int, _VP, _VP, _VP, ctypes.c_float, _VP, _VP,
                                            ctypes.c_float, _VP, ctypes.c_int, ctypes.c_int, _VP]),
    "sidon_glu": (ctypes.c_int, [_VP, _VP, ctypes.c_int, ctypes.c_int, _VP]),
    "sidon_silu": (ctypes.c_int, [_VP, ctypes.c_int64, _VP]),
    "sidon_gemm_bias_act_fits": (ctypes.c_int, [ctypes.c_int, ctypes.c_int, ctypes.c_int]),
    "sidon_gemm_bias_act_preferred": (ctypes.c_int, [ctypes.c_int, ctypes.c_int, ctypes.c_int]),
    "sidon_gemm_bias_act": (ctypes.c_int, [_VP, ctypes.c_int, _VP, ctypes.c_int, _VP, _VP, ctypes.c_int,
                                           ctypes.c_int, ctypes.c_int, ctypes.c_int, ctypes.c_int, _VP]),
    "sidon_gemm_lt_act": (ctypes.c_int, [_VP, ctypes.c_int, _VP, ctypes.c_int, _VP, _VP, ctypes.c_int,
                                         ctypes.c_int, ctypes.c_int, ctypes.c_int, ctypes.c_int, _VP]),
    "sidon_gemm_half_preferred": (ctypes.c_int, [ctypes.c_int, ctypes.c_int, ctypes.c_int]),
    "sidon_gemm_half_takes": (ctypes.c_int, [_VP, ctypes.c_int, _VP, ctypes.c_int, _VP, _VP, ctypes.c_int,
                                             ctypes.c_int, ctypes.c_int, ctypes.c_int]),
    "sidon_gemm_choice": (ctypes.c_int, [ctypes.c_int, ctypes.c_int, ctypes.c_int, ctypes.c_int, ctypes.c_int,
                                         ctypes.c_int, _IP, _IP]),
    "sidon_gemm_glu": (ctypes.c_int, [_VP, ctypes.c_int, _VP, ctypes.c_int, _VP, ctypes.c_int, ctypes.c_int,
                                      ctypes.c_int, ctypes.c_int, _VP]),
    "sidon_gemm_part_splits": (ctypes.c_int, [ctypes.c_int, ctypes.c_int, ctypes.c_int]),
    "sidon_gemm_part_rows": (ctypes.c_int64, [ctypes.c_int]),
    "sidon_gemm_part": (ctypes.c_int, [_VP, ctypes.c_int, _VP, ctypes.c_int, _VP, ctypes.c_int64, ctypes.c_int,
                                       ctypes.c_int, ctypes.c_int, _VP]),
    "sidon_gemm_res_fits": (ctypes.c_int, [ctypes.c_int, ctypes.c_int, ctypes.c_int]),
    "sidon_gemm_res_preferred": (ctypes.c_int, [ctypes.c_int, ctypes.c_int, ctypes.c_int]),
    "sidon_gemm_res": (ctypes.c_int, [_VP, ctypes.c_int, _VP, ctypes.c_int, _VP, ctypes.c_int, ctypes.c_int,
                                      ctypes.c_int, ctypes.c_int, _VP]),
    "sidon_gemm_nt": (ctypes.c_int, [_VP, ctypes.c_int, _VP, ctypes.c_int, _VP, ctypes.c_int, ctypes.c_int,
                                     ctypes.c_int, ctypes.c_int, ctypes.c_int, ctypes.c_float, _VP]),
    "sidon_gemm_nt_tune": (ctypes.c_int, [_VP, ctypes.c_int, _VP, ctypes.c_int, _VP, _VP, ctypes.c_int, ctypes.c_int,
                                          ctypes.c_int, ctypes.c_int, ctypes.c_int, ctypes.c_float, _VP,
                                          ctypes.POINTER(ctypes.c_int)]),
    "sidon_gemm_nt_pin": (ctypes.c_int, [ctypes.c_int] * 9),
    "sidon_causal_dw_norm": (ctypes.c_int, [_VP, ctypes.c_int, _VP, _VP, _VP, ctypes.c_float, _VP,
                                            ctypes.c_int, ctypes.c_int, ctypes.c_int, ctypes.c_int, _VP]),
    "sidon_fbank_frames": (ctypes.c_int, [_VP, _VP, ctypes.c_int, ctypes.c_int, _VP]),
    "sidon_fbank_logmel": (ctypes.c_int, [_VP, _VP, _VP, _VP, ctypes.c_int, _VP, ctypes.c_int, _VP]),
    "sidon_fbank_features": (ctypes.c_int, [_VP, _VP, _VP, _VP, _VP, _VP, _VP, ctypes.c_int, _VP, _VP,
                                            ctypes.c_size_t, _VP, ctypes.c_int, ctypes.c_int, _VP]),
    "sidon_fbank_workspace_bytes": (ctypes.c_size_t, [ctypes.c_int, ctypes.c_int]),
    "sidon_fbank_normalize": (ctypes.c_int, [_VP, _VP, _VP, ctypes.c_size_t, _VP, ctypes.c_int, ctypes.c_int, _VP]),
    "sidon_fbank_normalize_noalloc": (ctypes.c_int, [_VP, _VP, _VP, ctypes.c_int, ctypes.c_int, _VP]),
    "sidon_stage_items": (ctypes.c_int, [_VP, ctypes.c_int64, _VP, ctypes.c_int64, _I64P, _VP, _IP, _VP, _IP,
                                         ctypes.c_int, _VP]),
    "sidon_group_norm_workspace_bytes": (ctypes.c_size_t, [ctypes.c_int] * 5),
    "sidon_group_norm_passes": (ctypes.c_int, [*[ctypes.c_int] * 6, _IP, _IP, _IP]),
    "sidon_group_norm_act": (ctypes.c_int, [_VP, ctypes.c_int64, _VP, _VP, _VP, ctypes.c_float, _VP, ctypes.c_int64,
                                            _VP, ctypes.c_size_t, ctypes.c_int, ctypes.c_int, ctypes.c_int,
                                            ctypes.c_int, ctypes.c_int, ctypes.c_int, _VP]),
    "sidon_adapter_workspace_bytes": (ctypes.c_size_t, [ctypes.c_int] * 4),
    "sidon_adapter_linear": (ctypes.c_int, [_VP, ctypes.c_int, _VP, ctypes.c_int, _VP, _VP, _VP, _VP, _VP, _VP,
                                            ctypes.c_int, _VP, ctypes.c_size_t, *[ctypes.c_int] * 8, _VP]),
    "sidon_adapter_residual": (ctypes.c_int, [_VP, ctypes.c_int, _VP, ctypes.c_int, _VP, _VP, _VP, _VP, _VP,
                                              ctypes.c_int, _VP, ctypes.c_int, _VP, ctypes.c_size_t,
                                              *[ctypes.c_int] * 7, _VP]),
    "sidon_diff_attention_workspace_bytes": (ctypes.c_size_t, [ctypes.c_int] * 6),
    "sidon_diff_attention": (ctypes.c_int, [_VP, _VP, _VP, _VP, ctypes.c_int, ctypes.c_float, _VP, _VP, ctypes.c_float,
                                            _VP, _VP, ctypes.c_size_t, *[ctypes.c_int] * 8, _I64P, _I64P, _I64P, _I64P,
                                            _VP]),
    "sidon_last_error": (ctypes.c_char_p, []),
    "sidon_version": (ctypes.c_char_p, []),
}

# Element type and activation codes of include/sidon_operators.h.
DTYPES = {torch.float32: 0, torch.float16: 1, torch.bfloat16: 2}
ACTIVATIONS = {None: 0, "silu": 1, "gelu": 2, "relu": 3}

_lib = None


class Layouts(dict):
    """What a call's checks found for operands of one layout (their shapes,
    strides, types and devices, which the key holds all of, and nothing of what
    they contain): the next call of the same layout skips them, half of a small
    call's time on the host.  Emptied when full."""

    MOST = 1024

    def keep(self, key: tuple, found: tuple) -> tuple:
        if len(self) >= self.MOST:
            self.clear()
        self[key] = found
        return found


class SidonError(RuntimeError):
    """A nonzero return code of the C ABI."""

    def __init__(self, func: str, code: int, message: str):
        super().__init__(f"{func} failed with {ERROR_NAMES.get(code, code)}: {message}")
        self.code = code


def load() -> ctypes.CDLL:
    """Load the HIP library once (raises if it has not been built)."""
    global _lib
    if _lib is None:
        if not LIB_PATH.exists():
            raise RuntimeError(
                f"{LIB_PATH} is missing: build the HIP extension first "
                "(python -c 'import __graft_entry__ as g; g.build()')")
        lib = ctypes.CDLL(str(LIB_PATH))
        for name, (restype, argtypes) in SIGNATURES.items():
            fn = getattr(lib, name)
            fn.restype = restype
            fn.argtypes = argtypes
        _lib = lib
    return _lib


def check(func: str, code: int) -> None:
    if code != SIDON_OK:
        msg = load().sidon_last_error().decode(errors="replace")
        raise SidonError(func, code, msg)


INT_MAX = 2 ** 31 - 1


def ints(**values: int) -> None:
    """Refuses what a C int does not hold (ctypes would pass its low 32 bits)."""
    for name, value in values.items():
        if not -INT_MAX <= value <= INT_MAX:
            raise ValueError(f"{name.replace('_', ' ')} {value} must fit 32 bits")


def strides3(st) -> ctypes.Array:
    return (ctypes.c_int64 * 3)(*[int(x) for x in st])


def launch_shape(batch: int, heads: int, length: int) -> dict:
    """(queries per workgroup, key splits, workgroups, threads) the library uses."""
    lib = load()
    vals = [ctypes.c_int() for _ in range(4)]
    check("sidon_flexrel_launch_shape",
          lib.sidon_flexrel_launch_shape(batch, heads, length, *[ctypes.byref(x) for x in vals]))
    keys = ("queries_per_block", "key_splits", "workgroups", "threads_per_block")
    return {k: v.value for k, v in zip(keys, vals)}


def version() -> str:
    return load().sidon_version().decode()
