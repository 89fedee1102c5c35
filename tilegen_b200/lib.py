"""ctypes binding of libtilegen_b200.so (declarations in include/tilegen_b200.h).

The library is looked up in ``$TILEGEN_B200_LIB`` or next to this file (built in-tree
by ``python -m tilegen_b200.build``).  There is no fallback: if the library cannot be
loaded every entry point raises :class:`LibraryError`.
"""

from __future__ import annotations

import ctypes
import os
import re
from typing import List, Optional

PKG_DIR = os.path.dirname(os.path.abspath(__file__))
REPO_DIR = os.path.dirname(PKG_DIR)
HEADER = os.path.join(REPO_DIR, "include", "tilegen_b200.h")
HEADER_PAGED = os.path.join(REPO_DIR, "include", "tilegen_b200_paged.h")

TG_OK = 0
TG_EINVAL = -1
TG_ECUDA = -2
TG_ENOMEM = -3
TG_EUNSUPPORTED = -4
TG_ETIMEDOUT = -5
TG_EBOUNDS = -6

TG_SPLIT_ROWWISE = 0
TG_SPLIT_MERGE = 1
TG_SPLIT_AUTO = 2
TG_SPLIT_STREAM = 3
TG_SPLIT_BLOCK = 4

TG_FLAG_BOUNDS_CHECK = 1
TG_FLAG_INJECT_BUG = 2
TG_FLAG_REUSE_PLAN = 4
TG_FLAG_INDEX32 = 8
TG_FLAG_CAUSAL = 16
TG_FLAG_ROPE_INVERSE = 32

TG_ROPE_HALF = 0
TG_ROPE_INTERLEAVED = 1

STATUS_NAMES = {
    TG_OK: "TG_OK",
    TG_EINVAL: "TG_EINVAL",
    TG_ECUDA: "TG_ECUDA",
    TG_ENOMEM: "TG_ENOMEM",
    TG_EUNSUPPORTED: "TG_EUNSUPPORTED",
    TG_ETIMEDOUT: "TG_ETIMEDOUT",
    TG_EBOUNDS: "TG_EBOUNDS",
}


class LibraryError(RuntimeError):
    """libtilegen_b200.so is missing or failed to load."""


class TgError(RuntimeError):
    """A tg_* call returned a negative status."""

    def __init__(self, status: int, what: str, message: str):
        self.status = status
        super().__init__("%s failed: %s (%s)" % (what, STATUS_NAMES.get(status, status), message))


class TgSched(ctypes.Structure):
    _fields_ = [
        ("tile", ctypes.c_int32),
        ("threads_per_row", ctypes.c_int32),
        ("unroll", ctypes.c_int32),
        ("vector_width", ctypes.c_int32),
        ("block_size", ctypes.c_int32),
        ("split", ctypes.c_int32),
        ("chunk_nnz", ctypes.c_int32),
        ("flags", ctypes.c_uint32),
    ]

    def as_dict(self):
        return {name: getattr(self, name) for name, _ in self._fields_}


class TgCsr(ctypes.Structure):
    _fields_ = [
        ("rows", ctypes.c_int64),
        ("cols", ctypes.c_int64),
        ("nnz", ctypes.c_int64),
        ("indptr", ctypes.c_void_p),
        ("indices", ctypes.c_void_p),
        ("data", ctypes.c_void_p),
    ]


class TgRope(ctypes.Structure):
    _fields_ = [
        ("freq", ctypes.c_void_p),
        ("rot_dim", ctypes.c_int32),
        ("layout", ctypes.c_int32),
        ("scale", ctypes.c_double),
    ]


class TgRows(ctypes.Structure):
    _fields_ = [
        ("data", ctypes.c_void_p),
        ("token_stride", ctypes.c_int64),
        ("head_stride", ctypes.c_int64),
    ]


class TgPagedKV(ctypes.Structure):
    _fields_ = [
        ("k", ctypes.c_void_p),
        ("v", ctypes.c_void_p),
        ("pages", ctypes.c_int64),
        ("page_size", ctypes.c_int64),
        ("heads", ctypes.c_int32),
        ("dim", ctypes.c_int32),
        ("k_page_stride", ctypes.c_int64),
        ("k_slot_stride", ctypes.c_int64),
        ("k_head_stride", ctypes.c_int64),
        ("v_page_stride", ctypes.c_int64),
        ("v_slot_stride", ctypes.c_int64),
        ("v_head_stride", ctypes.c_int64),
    ]


class TgKvAppendArgs(ctypes.Structure):
    _fields_ = [
        ("cache", ctypes.c_void_p),  # TgPagedKV
        ("pages", ctypes.c_void_p),  # TgCsr
        ("seq_len", ctypes.c_void_p),
        ("tokens", ctypes.c_int64),
        ("q_indptr", ctypes.c_void_p),
        ("k", TgRows),
        ("v", TgRows),
        ("rope", ctypes.c_void_p),  # TgRope
        ("q", ctypes.c_void_p),  # TgRows
        ("q_out", ctypes.c_void_p),  # TgRows
        ("q_heads", ctypes.c_int32),
        ("position_base", ctypes.c_int64),
        ("positions", ctypes.c_void_p),
        ("flags", ctypes.c_uint32),
    ]


class TgHeadNorm(ctypes.Structure):
    _fields_ = [
        ("weight", ctypes.c_void_p),
        ("weight_f32", ctypes.c_int32),
        ("eps", ctypes.c_double),
        ("offset", ctypes.c_double),
    ]


class TgNormRopeArgs(ctypes.Structure):
    _fields_ = [
        ("tokens", ctypes.c_int64),
        ("dim", ctypes.c_int32),
        ("q_heads", ctypes.c_int32),
        ("k_heads", ctypes.c_int32),
        ("q", TgRows),
        ("k", TgRows),
        ("q_out", TgRows),
        ("k_out", TgRows),
        ("q_norm", ctypes.c_void_p),  # TgHeadNorm
        ("k_norm", ctypes.c_void_p),  # TgHeadNorm
        ("rope", ctypes.c_void_p),  # TgRope
        ("positions", ctypes.c_void_p),
        ("flags", ctypes.c_uint32),
    ]


class TgNormRopeGradArgs(ctypes.Structure):
    _fields_ = [
        ("tokens", ctypes.c_int64),
        ("dim", ctypes.c_int32),
        ("q_heads", ctypes.c_int32),
        ("k_heads", ctypes.c_int32),
        ("q", TgRows),
        ("k", TgRows),
        ("dq_out", TgRows),
        ("dk_out", TgRows),
        ("dq", TgRows),
        ("dk", TgRows),
        ("q_norm", ctypes.c_void_p),  # TgHeadNorm
        ("k_norm", ctypes.c_void_p),  # TgHeadNorm
        ("dq_weight", ctypes.c_void_p),
        ("dk_weight", ctypes.c_void_p),
        ("rope", ctypes.c_void_p),  # TgRope
        ("positions", ctypes.c_void_p),
        ("flags", ctypes.c_uint32),
    ]


class TgPrefixAttentionArgs(ctypes.Structure):
    _fields_ = [
        ("cache", ctypes.c_void_p),  # TgPagedKV
        ("pages", ctypes.c_void_p),  # TgCsr
        ("seq_len", ctypes.c_void_p),
        ("max_seq_len", ctypes.c_int64),
        ("prefix_pages", ctypes.c_void_p),
        ("n_prefix_pages", ctypes.c_int64),
        ("prefix_len", ctypes.c_int64),
        ("tokens", ctypes.c_int64),
        ("q_indptr", ctypes.c_void_p),
        ("max_q_len", ctypes.c_int64),
        ("q_heads", ctypes.c_int32),
        ("q", TgRows),
        ("out", TgRows),
        ("lse", ctypes.c_void_p),
        ("scale", ctypes.c_double),
        ("flags", ctypes.c_uint32),
    ]


class TgPagedMass(ctypes.Structure):
    _fields_ = [
        ("data", ctypes.c_void_p),
        ("page_stride", ctypes.c_int64),
        ("slot_stride", ctypes.c_int64),
        ("head_stride", ctypes.c_int64),
    ]


class TgAttentionMassArgs(ctypes.Structure):
    _fields_ = [
        ("cache", ctypes.c_void_p),  # TgPagedKV
        ("pages", ctypes.c_void_p),  # TgCsr
        ("seq_len", ctypes.c_void_p),
        ("max_seq_len", ctypes.c_int64),
        ("tokens", ctypes.c_int64),
        ("q_indptr", ctypes.c_void_p),
        ("max_q_len", ctypes.c_int64),
        ("q_heads", ctypes.c_int32),
        ("q", TgRows),
        ("lse", ctypes.c_void_p),
        ("scale", ctypes.c_double),
        ("mass", TgPagedMass),
        ("decay", ctypes.c_double),
        ("flags", ctypes.c_uint32),
    ]


class TgKvEvictArgs(ctypes.Structure):
    _fields_ = [
        ("cache", ctypes.c_void_p),  # TgPagedKV
        ("pages", ctypes.c_void_p),  # TgCsr
        ("seq_len", ctypes.c_void_p),
        ("max_seq_len", ctypes.c_int64),
        ("budget", ctypes.c_int64),
        ("first", ctypes.c_int64),
        ("recent", ctypes.c_int64),
        ("mass", TgPagedMass),
        ("mass_out", TgPagedMass),
        ("seq_len_out", ctypes.c_void_p),
        ("kept", ctypes.c_void_p),
        ("kept_width", ctypes.c_int64),
        ("flags", ctypes.c_uint32),
    ]


_I64 = ctypes.c_int64
_P = ctypes.c_void_p
_F64 = ctypes.c_double
_SZ = ctypes.c_size_t
_SP = ctypes.POINTER(TgSched)
_CP = ctypes.POINTER(TgCsr)

# name -> (restype, argtypes); every symbol declared in include/tilegen_b200.h
SIGNATURES = {
    "tg_version": (ctypes.c_char_p, []),
    "tg_last_error_string": (ctypes.c_char_p, []),
    "tg_last_status": (ctypes.c_int, []),
    "tg_launch_count": (ctypes.c_uint64, []),
    "tg_dist_init": (ctypes.c_int, [ctypes.c_int32, ctypes.POINTER(ctypes.c_int32), ctypes.POINTER(ctypes.c_void_p)]),
    "tg_dist_finalize": (ctypes.c_int, [ctypes.c_void_p]),
    "tg_dist_spmv_power": (ctypes.c_int, [ctypes.c_void_p, _CP, ctypes.c_void_p, ctypes.c_int32, _SP, ctypes.c_void_p,
                                          ctypes.c_void_p, ctypes.c_double]),
    "tg_dist_spmm_f32": (ctypes.c_int, [ctypes.c_void_p, _CP, ctypes.c_void_p, ctypes.c_int64, ctypes.c_void_p, _SP,
                                        ctypes.c_double]),
    "tg_dist_sddmm_f32": (ctypes.c_int, [ctypes.c_void_p, _CP, ctypes.c_void_p, ctypes.c_void_p, ctypes.c_int64,
                                         ctypes.c_void_p, _SP, ctypes.c_double]),
    "tg_renumber_columns": (ctypes.c_int, [ctypes.c_void_p, ctypes.c_void_p, ctypes.c_int64, ctypes.c_void_p,
                                           ctypes.c_int32, ctypes.c_int64, ctypes.c_void_p]),
    "tg_renumber_columns_i32": (ctypes.c_int, [ctypes.c_void_p, ctypes.c_void_p, ctypes.c_int64, ctypes.c_void_p,
                                               ctypes.c_int32, ctypes.c_int64, ctypes.c_void_p]),
    "tg_default_schedule": (None, [_SP]),
    "tg_validate_schedule": (ctypes.c_int, [_SP]),
    "tg_set_schedule": (ctypes.c_int, [_SP]),
    "tg_get_schedule": (ctypes.c_int, [_SP]),
    "tg_spmv_workspace_bytes": (_SZ, [_I64, _I64, _SP]),
    "tg_spmm_workspace_bytes": (_SZ, [_I64, _I64, _I64, _SP]),
    "tg_sddmm_workspace_bytes": (_SZ, [_I64, _I64, _I64, _SP]),
    "tg_spmv_f64": (ctypes.c_int, [_CP, _P, _P, _SP, _P, _SZ, _P]),
    "tg_spmv_f32": (ctypes.c_int, [_CP, _P, _P, _SP, _P, _SZ, _P]),
    "tg_fused_spmv_axpy_f64": (ctypes.c_int, [_CP, _P, _P, _P, _F64, _F64, _SP, _P, _SZ, _P]),
    "tg_fused_spmv_axpy_f32": (ctypes.c_int, [_CP, _P, _P, _P, ctypes.c_float, ctypes.c_float, _SP, _P, _SZ, _P]),
    "tg_spmm_f32": (ctypes.c_int, [_CP, _P, _P, _I64, _SP, _P, _SZ, _P]),
    "tg_spmm_f64": (ctypes.c_int, [_CP, _P, _P, _I64, _SP, _P, _SZ, _P]),
    "tg_sddmm_f32": (ctypes.c_int, [_CP, _P, _P, _P, _I64, _SP, _P, _SZ, _P]),
    "tg_sddmm_f64": (ctypes.c_int, [_CP, _P, _P, _P, _I64, _SP, _P, _SZ, _P]),
    "tg_axpy_f64": (ctypes.c_int, [_P, _P, _P, _F64, _F64, _I64, _SP, _P]),
    "tg_axpy_f32": (ctypes.c_int, [_P, _P, _P, ctypes.c_float, ctypes.c_float, _I64, _SP, _P]),
    "tg_power_workspace_bytes": (_SZ, [_I64, _SP]),
    "tg_power_step_f64": (ctypes.c_int, [_CP, _P, ctypes.c_int32, _I64, _P, _SP, _P, _SZ, _P]),
    "tg_shard_norm2_f64": (ctypes.c_int, [_P, _I64, _I64, _P, _SZ, _P]),
    "tg_power_finalize_f64": (ctypes.c_int, [_P, ctypes.c_int32, _I64, ctypes.c_int32, _I64, _P, _P, _P]),
    "tg_power_step_p2p_f64": (ctypes.c_int, [_CP, _P, ctypes.c_int32, ctypes.c_int32, _I64, _P, _P,
                                             ctypes.c_uint64, _SP, _P, _SZ, _P]),
    "tg_p2p_wait": (ctypes.c_int, [_P, ctypes.c_int32, ctypes.c_uint64, _P, _SZ, _P]),
    "tg_power_error": (ctypes.c_int, [_P, ctypes.POINTER(ctypes.c_uint32), _P]),
    "tg_power_clear_error": (ctypes.c_int, [_P, _P]),
    "tg_power_step_ce_f64": (ctypes.c_int, [_CP, _P, ctypes.c_int32, ctypes.c_int32, _I64, _P, _P, ctypes.c_uint64,
                                            ctypes.c_int32, _SP, _P, _SZ, _P]),
    "tg_peer_buffer_alloc": (ctypes.c_int, [_SZ, ctypes.POINTER(ctypes.c_void_p)]),
    "tg_peer_buffer_free": (ctypes.c_int, [_P]),
    "tg_ipc_get_handle": (ctypes.c_int, [_P, ctypes.c_char_p]),
    "tg_ipc_open": (ctypes.c_int, [ctypes.c_char_p, ctypes.POINTER(ctypes.c_void_p)]),
    "tg_ipc_close": (ctypes.c_int, [_P]),
    "tg_spmv_f64_noalloc": (ctypes.c_int, [_CP, _P, _P, _SP, _P]),
    "tg_rcm_order": (ctypes.c_int, [_I64, _P, _P, _P]),
    "launch_spmv": (None, [_P, _P, _P, _P, _P, _I64, _I64, _I64]),
    "launch_spmm": (None, [_P, _P, _P, _P, _P, _I64, _I64, _I64, _I64]),
    "launch_sddmm": (None, [_P, _P, _P, _P, _P, _P, _I64, _I64, _I64, _I64]),
    "launch_fused_spmv_axpy": (None, [_P, _P, _P, _P, _P, _P, _F64, _F64, _I64, _I64, _I64]),
    "launch_axpy": (None, [_P, _P, _P, _F64, _F64, _I64]),
}

_ROPE = [ctypes.POINTER(TgRope), ctypes.POINTER(TgRows), ctypes.POINTER(TgRows), _I64, ctypes.c_int32,
         ctypes.c_int32, _P, ctypes.c_uint32, _P]

_TYPES = ("f32", "f16", "bf16")

# every symbol declared in include/tilegen_b200_paged.h
SIGNATURES_PAGED = {
    "tg_rope_f32": (ctypes.c_int, _ROPE),
    "tg_rope_f16": (ctypes.c_int, _ROPE),
    "tg_rope_bf16": (ctypes.c_int, _ROPE),
    "tg_kv_append_f32": (ctypes.c_int, [ctypes.POINTER(TgKvAppendArgs), _P]),
    "tg_kv_append_f16": (ctypes.c_int, [ctypes.POINTER(TgKvAppendArgs), _P]),
    "tg_kv_append_bf16": (ctypes.c_int, [ctypes.POINTER(TgKvAppendArgs), _P]),
    **{"tg_norm_rope_" + t: (ctypes.c_int, [ctypes.POINTER(TgNormRopeArgs), _P]) for t in _TYPES},
    "tg_norm_rope_backward_workspace_bytes": (_SZ, [ctypes.POINTER(TgNormRopeGradArgs)]),
    **{"tg_norm_rope_backward_" + t: (ctypes.c_int, [ctypes.POINTER(TgNormRopeGradArgs), _P, _SZ, _P]) for t in _TYPES},
    **{"tg_kv_append_normed_" + t: (ctypes.c_int, [ctypes.POINTER(TgKvAppendArgs), ctypes.POINTER(TgHeadNorm),
                                                   ctypes.POINTER(TgHeadNorm), _P]) for t in _TYPES},
    "tg_prefix_attention_workspace_bytes": (_SZ, [ctypes.POINTER(TgPrefixAttentionArgs)]),
    "tg_prefix_attention_needed_bytes": (_SZ, [ctypes.POINTER(TgPrefixAttentionArgs)]),
    "tg_prefix_attention_f16": (ctypes.c_int, [ctypes.POINTER(TgPrefixAttentionArgs), _P, _SZ, _P]),
    "tg_prefix_attention_bf16": (ctypes.c_int, [ctypes.POINTER(TgPrefixAttentionArgs), _P, _SZ, _P]),
    "tg_attention_mass_workspace_bytes": (_SZ, [ctypes.POINTER(TgAttentionMassArgs)]),
    "tg_attention_mass_needed_bytes": (_SZ, [ctypes.POINTER(TgAttentionMassArgs)]),
    "tg_attention_mass_f16": (ctypes.c_int, [ctypes.POINTER(TgAttentionMassArgs), _P, _SZ, _P]),
    "tg_attention_mass_bf16": (ctypes.c_int, [ctypes.POINTER(TgAttentionMassArgs), _P, _SZ, _P]),
    "tg_kv_evict_workspace_bytes": (_SZ, [ctypes.POINTER(TgKvEvictArgs)]),
    **{"tg_kv_evict_" + t: (ctypes.c_int, [ctypes.POINTER(TgKvEvictArgs), _P, _SZ, _P]) for t in _TYPES},
}

_lib: Optional[ctypes.CDLL] = None


def lib_path() -> str:
    env = os.environ.get("TILEGEN_B200_LIB")
    if env:
        return env
    return os.path.join(PKG_DIR, "libtilegen_b200.so")


def load() -> ctypes.CDLL:
    """Load (once) and type the library; raises LibraryError when it is absent."""
    global _lib
    if _lib is not None:
        return _lib
    path = lib_path()
    if not os.path.exists(path):
        raise LibraryError("libtilegen_b200.so not found at %s; build it with `python -m tilegen_b200.build` "
                           "(there is no CPU fallback)" % path)
    try:
        L = ctypes.CDLL(path)
    except OSError as exc:
        raise LibraryError("cannot load %s: %s" % (path, exc)) from exc
    for name, (res, args) in {**SIGNATURES, **SIGNATURES_PAGED}.items():
        fn = getattr(L, name)
        fn.restype = res
        fn.argtypes = args
    _lib = L
    return L


def header_symbols(path: str = HEADER) -> List[str]:
    """Function names declared in include/tilegen_b200.h."""
    text = open(path).read()
    return re.findall(r"^TG_API\s+[\w\s\*]+?\b(\w+)\s*\(", text, flags=re.M)


def last_error() -> str:
    msg = load().tg_last_error_string()
    return msg.decode("utf-8", "replace") if msg else ""


def check(status: int, what: str) -> None:
    if status != TG_OK:
        raise TgError(status, what, last_error())


def version() -> str:
    return load().tg_version().decode()


def default_schedule() -> TgSched:
    s = TgSched()
    load().tg_default_schedule(ctypes.byref(s))
    return s


def validate_schedule(s: TgSched) -> None:
    check(load().tg_validate_schedule(ctypes.byref(s)), "tg_validate_schedule")


def set_schedule(s: TgSched) -> None:
    check(load().tg_set_schedule(ctypes.byref(s)), "tg_set_schedule")


def get_schedule() -> TgSched:
    s = TgSched()
    check(load().tg_get_schedule(ctypes.byref(s)), "tg_get_schedule")
    return s
