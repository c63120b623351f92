"""ctypes binding of libflashmlp.so (the C ABI declared in include/flashmlp.h).

The library is loaded lazily, once. If it has not been built, every call raises: there
is no fallback path.
"""
from __future__ import annotations

import ctypes
import threading
from pathlib import Path

LIB_PATH = Path(__file__).resolve().with_name("libflashmlp.so")

FMLP_OK = 0
FMLP_DTYPE_F16 = 0
FMLP_DTYPE_BF16 = 1
FMLP_DTYPE_F32 = 2
# OR-ed into the dtype code: outputs are fp32 arrays holding the unrounded fp32 sums
FMLP_OUT_F32 = 0x100
# OR-ed into the backward's dtype code: dW products with hi/lo io-dtype terms of h and dZ
FMLP_DW_HILO = 0x200
# OR-ed into the backward's dtype code: the recompute-only form (no stored dZ in the workspace)
FMLP_BWD_RECOMPUTE = 0x400
# OR-ed into the backward's dtype code: the stored-dZ form whenever the workspace allows (tests)
FMLP_BWD_STORE_DZ = 0x800
# OR-ed into the backward's dtype code: no dx wanted (dx may be NULL) / no dw1, dw2 wanted
FMLP_BWD_NO_DX = 0x1000
FMLP_BWD_NO_DW = 0x2000
ACT_CODES = {"": 0, "silu": 1, "leaky_relu": 2, "sigmoid": 3}



class Join(ctypes.Structure):
    """fmlp_join of include/flashmlp.h"""
    _fields_ = ([(n, ctypes.c_void_p) for n in (
        "r", "o", "w_post", "gate", "w_pre", "r_out", "y", "rs_o", "rs_r", "dr_out", "dy", "dr", "d_o", "dw_post",
        "dgate", "dw_pre")]
        + [(n, ctypes.c_int64) for n in (
            "B", "H", "D", "groups", "r_stride", "o_head_stride", "o_row_stride", "y_head_stride", "y_row_stride",
            "dr_out_stride", "d_o_head_stride", "d_o_row_stride")]
        + [("scale", ctypes.c_float), ("eps", ctypes.c_float), ("dtype", ctypes.c_int), ("r_dtype", ctypes.c_int),
           ("post", ctypes.c_int)])


class MuonTensor(ctypes.Structure):
    """fmlp_muon_tensor of include/flashmlp.h"""
    _fields_ = ([(n, ctypes.c_void_p) for n in ("w", "g", "m")] + [(n, ctypes.c_int64) for n in ("H", "R", "C")]
                + [(n, ctypes.c_int) for n in ("w_dtype", "g_dtype", "m_dtype")] + [("scale", ctypes.c_float)])


# (name, restype, argtypes) for every symbol include/flashmlp.h declares
_i64 = ctypes.c_int64
_vp = ctypes.c_void_p
_i64p = ctypes.POINTER(ctypes.c_int64)
_vpp = ctypes.POINTER(_vp)
_intp = ctypes.POINTER(ctypes.c_int)
_f32p = ctypes.POINTER(ctypes.c_float)
SIGNATURES = {
    "fmlp_abi_version": (ctypes.c_int, []),
    "fmlp_status_string": (ctypes.c_char_p, [ctypes.c_int]),
    "fmlp_last_error": (ctypes.c_char_p, []),
    "fmlp_act_from_name": (ctypes.c_int, [ctypes.c_char_p]),
    "fmlp_shape_supported": (ctypes.c_int, [_i64, _i64, _i64, _i64, ctypes.c_int]),
    "fmlp_shape_tuned": (ctypes.c_int, [_i64, _i64, ctypes.c_int]),
    "fmlp_shape_dense": (ctypes.c_int, [_i64, _i64, ctypes.c_int]),
    "fmlp_fwd": (ctypes.c_int, [_vp, _vp, _vp, _vp, _i64, _i64, _i64, _i64, ctypes.c_int, ctypes.c_int, _vp]),
    "fmlp_fwd_strided": (ctypes.c_int, [_vp, _vp, _vp, _vp, _i64, _i64, _i64, _i64, _i64p, _i64p, _i64p,
                                        ctypes.c_int, ctypes.c_int, _vp]),
    "fmlp_fwd_strided_ws": (ctypes.c_int, [_vp, _vp, _vp, _vp, _i64, _i64, _i64, _i64, _i64p, _i64p, _i64p,
                                           ctypes.c_int, ctypes.c_int, _vp, ctypes.c_size_t, _vp]),
    "fmlp_fwd_workspace_bytes": (ctypes.c_size_t, [_i64, _i64, _i64, _i64, ctypes.c_int]),
    "fmlp_fwd_ws": (ctypes.c_int, [_vp, _vp, _vp, _vp, _i64, _i64, _i64, _i64, ctypes.c_int, ctypes.c_int, _vp,
                                   ctypes.c_size_t, _vp]),
    "fmlp_copy_dense": (ctypes.c_int, [ctypes.c_int, ctypes.POINTER(_vp), ctypes.POINTER(_vp), _i64p, _i64p, ctypes.c_int,
                                       _vp]),
    "fmlp_bwd_workspace_bytes": (ctypes.c_size_t, [_i64, _i64, _i64, _i64, ctypes.c_int]),
    "fmlp_bwd_stores_dz": (ctypes.c_int, [_i64, _i64, _i64, _i64, ctypes.c_int, ctypes.c_int]),
    "fmlp_bwd_plan": (ctypes.c_int, [_i64, _i64, _i64, _i64, ctypes.c_int, ctypes.c_int, _i64p, ctypes.c_int]),
    "fmlp_bwd": (ctypes.c_int, [_vp, _vp, _vp, _vp, _vp, _vp, _vp, _i64, _i64, _i64, _i64, ctypes.c_int,
                                ctypes.c_int, _vp, ctypes.c_size_t, _vp]),
    "fmlp_bwd_strided": (ctypes.c_int, [_vp, _vp, _vp, _vp, _vp, _vp, _vp, _i64, _i64, _i64, _i64, _i64p, _i64p,
                                        _i64p, _i64p, ctypes.c_int, ctypes.c_int, _vp, ctypes.c_size_t, _vp]),
    "fmlp_gated_min_workspace_bytes": (ctypes.c_size_t, [_i64, _i64, _i64, ctypes.c_int]),
    "fmlp_gated_fwd_workspace_bytes": (ctypes.c_size_t, [_i64, _i64, _i64, _i64, ctypes.c_int]),
    "fmlp_gated_fwd": (ctypes.c_int, [_vp] * 5 + [_i64] * 5 + [ctypes.c_int, ctypes.c_int, _vp, ctypes.c_size_t, _vp]),
    "fmlp_gated_bwd_workspace_bytes": (ctypes.c_size_t, [_i64, _i64, _i64, _i64, ctypes.c_int]),
    "fmlp_gated_bwd": (ctypes.c_int, [_vp] * 9 + [_i64] * 6 + [ctypes.c_int, ctypes.c_int, ctypes.c_float, _vp,
                                                               ctypes.c_size_t, _vp]),
    "fmlp_head_sum": (ctypes.c_int, [_vp, _vp, _i64, _i64, ctypes.c_float, ctypes.c_int, _vp]),
    "fmlp_join_fwd": (ctypes.c_int, [ctypes.POINTER(Join), _vp]),
    "fmlp_join_bwd_workspace_bytes": (ctypes.c_size_t, [ctypes.POINTER(Join)]),
    "fmlp_join_bwd": (ctypes.c_int, [ctypes.POINTER(Join), _vp, ctypes.c_size_t, _vp]),
    "fmlp_clip_workspace_bytes": (ctypes.c_size_t, [ctypes.c_int, _i64p]),
    "fmlp_grad_norm": (ctypes.c_int, [ctypes.c_int, _vpp, _i64p, _intp, _vp, _vp, ctypes.c_size_t, _vp]),
    "fmlp_clip_grads": (ctypes.c_int, [ctypes.c_int, _vpp, _vpp, _i64p, _intp, _intp, ctypes.c_float, _vp, _vp,
                                       ctypes.c_size_t, _vp]),
    "fmlp_route_fwd": (ctypes.c_int, [_vp] * 3 + [_i64] * 4 + [ctypes.c_int, ctypes.c_int, _vp]),
    "fmlp_route_bwd": (ctypes.c_int, [_vp] * 5 + [_i64] * 4 + [ctypes.c_int, ctypes.c_int, _vp]),
    "fmlp_expert_plan_workspace_bytes": (ctypes.c_size_t, [_i64] * 3),
    "fmlp_expert_plan": (ctypes.c_int, [_vp, ctypes.c_int, _vp, _vp] + [_i64] * 4 + [_vp, ctypes.c_size_t, _vp]),
    "fmlp_expert_scatter": (ctypes.c_int, [_vp, _i64] + [_vp] * 6 + [_i64] * 5 + [ctypes.c_int, _vp]),
    "fmlp_expert_gather": (ctypes.c_int, [_vp] * 4 + [_i64] * 5 + [ctypes.c_int, _vp]),
    "fmlp_orthogonalize_workspace_bytes": (ctypes.c_size_t, [_i64] * 3 + [ctypes.c_int, ctypes.c_int]),
    "fmlp_orthogonalize_workspace_bytes_for": (ctypes.c_size_t, [_i64] * 3 + [ctypes.c_int, ctypes.c_int, _f32p]),
    "fmlp_orthogonalize": (ctypes.c_int, [_vp, _vp] + [_i64] * 3 + [ctypes.c_int, ctypes.c_int, _f32p, ctypes.c_float, _vp,
                                                                    ctypes.c_size_t, _vp]),
    "fmlp_muon_workspace_bytes": (ctypes.c_size_t, [ctypes.c_int, ctypes.POINTER(MuonTensor), ctypes.c_int]),
    "fmlp_muon_workspace_bytes_for": (ctypes.c_size_t, [ctypes.c_int, ctypes.POINTER(MuonTensor), ctypes.c_int, _f32p]),
    "fmlp_muon_step": (ctypes.c_int, [ctypes.c_int, ctypes.POINTER(MuonTensor), ctypes.c_double, ctypes.c_double,
                                      ctypes.c_int, ctypes.c_double, ctypes.c_int, _f32p, ctypes.c_float, _vp,
                                      ctypes.c_size_t, _vp]),
    "fmlp_bwd_noalloc": (ctypes.c_int, [_vp, _vp, _vp, _vp, _vp, _vp, _vp, _i64, _i64, _i64, _i64, ctypes.c_int,
                                        ctypes.c_int, _vp]),
}
FMLP_SCRATCH_MAX_BYTES = 64 << 20
ABI_VERSION = 4  # FMLP_ABI_VERSION of include/flashmlp.h

_lock = threading.Lock()
_lib = None


class FlashMLPLibraryError(RuntimeError):
    """libflashmlp.so is missing or does not match this package."""


def lib() -> ctypes.CDLL:
    global _lib
    if _lib is not None:
        return _lib
    with _lock:
        if _lib is None:
            if not LIB_PATH.exists():
                raise FlashMLPLibraryError(
                    f"{LIB_PATH} is not built; run `python -m flashmlp_amd.build` (hipcc, gfx950)")
            handle = ctypes.CDLL(str(LIB_PATH))
            for name, (res, args) in SIGNATURES.items():
                fn = getattr(handle, name, None)
                if fn is None:  # entry points were added within an ABI version
                    raise FlashMLPLibraryError(f"{LIB_PATH} has no {name}: rebuild it (`python -m flashmlp_amd.build`)")
                fn.restype = res
                fn.argtypes = args
            if handle.fmlp_abi_version() != ABI_VERSION:
                raise FlashMLPLibraryError("libflashmlp.so ABI version mismatch; rebuild it")
            _lib = handle
    return _lib


def strides(t) -> "ctypes.Array":
    """The three element strides of a 3-D tensor as an int64_t[3] for the *_strided calls."""
    return (ctypes.c_int64 * 3)(*t.stride())


def check(status: int, what: str) -> None:
    if status != FMLP_OK:
        L = lib()
        msg = L.fmlp_status_string(status).decode()
        detail = L.fmlp_last_error().decode()
        raise RuntimeError(f"flashmlp {what} failed: {msg}: {detail}")
