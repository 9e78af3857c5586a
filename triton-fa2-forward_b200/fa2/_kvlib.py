"""ctypes binding of the C ABI in include/fa2_kvcache_sm100.h (libfa2_kvcache_sm100.so, built
in-tree): rotary positions, the 8-bit paged K/V cache, attention over it. As in `_lib`, the library
is required; there is no CPU or library fallback.
"""

import ctypes
import os

from ._lib import Fa2Error, strerror  # noqa: F401  (statuses are shared with the attention library)

LIB_NAME = "libfa2_kvcache_sm100.so"
LIB_PATH = os.path.join(os.path.dirname(os.path.abspath(__file__)), LIB_NAME)

ABI_VERSION = 1

# Every symbol the header declares (the ABI test checks the library exports all of them).
EXPORTED = (
    "fa2_rotary_sm100_check",
    "fa2_rotary_sm100",
    "fa2_kv8_append_sm100_check",
    "fa2_kv8_append_sm100",
    "fa2_kv8_read_sm100_check",
    "fa2_kv8_read_sm100",
    "fa2_kv8_attn_sm100_check",
    "fa2_kv8_attn_sm100_workspace_bytes",
    "fa2_kv8_attn_sm100",
    "fa2_kvcache_sm100_abi_version",
    "fa2_kvcache_sm100_params_size",
)

_p, _i32, _i64 = ctypes.c_void_p, ctypes.c_int32, ctypes.c_int64


class Kv8Cache(ctypes.Structure):
    """Mirror of `Fa2Kv8Cache`."""

    _fields_ = [("k", _p), ("v", _p), ("k_scale", _p), ("v_scale", _p),
                ("k_stride", _i64 * 3), ("v_stride", _i64 * 3), ("ks_stride", _i64 * 3), ("vs_stride", _i64 * 3),
                ("num_pages", _i32), ("page_size", _i32), ("heads_kv", _i32), ("head_dim", _i32)]


class RotaryParams(ctypes.Structure):
    """Mirror of `Fa2RotaryParams`."""

    _fields_ = [("q", _p), ("k", _p), ("q_out", _p), ("k_out", _p),
                ("q_stride", _i64 * 4), ("k_stride", _i64 * 4), ("q_out_stride", _i64 * 4), ("k_out_stride", _i64 * 4),
                ("positions", _p), ("pos_stride", _i64 * 2), ("inv_freq", _p),
                ("pos_is_64", _i32), ("batch", _i32), ("seqlen", _i32), ("heads_q", _i32), ("heads_kv", _i32),
                ("head_dim", _i32), ("rotary_dim", _i32), ("dtype", _i32), ("interleaved", _i32), ("inverse", _i32),
                ("magnitude", ctypes.c_float), ("reserved", _i32)]


class AppendParams(ctypes.Structure):
    """Mirror of `Fa2Kv8AppendParams`."""

    _fields_ = [("cache", Kv8Cache), ("k", _p), ("v", _p), ("k_in_stride", _i64 * 4), ("v_in_stride", _i64 * 4),
                ("block_table", _p), ("cache_seqlens", _p), ("cu_seqlens", _p), ("err_flag", _p),
                ("block_table_stride", _i64), ("pages_per_seq", _i32), ("batch", _i32), ("seqlen", _i32),
                ("dtype", _i32)]


class ReadParams(ctypes.Structure):
    """Mirror of `Fa2Kv8ReadParams`."""

    _fields_ = [("cache", Kv8Cache), ("k_out", _p), ("v_out", _p), ("block_table", _p), ("cu_seqlens", _p),
                ("err_flag", _p), ("block_table_stride", _i64), ("pages_per_seq", _i32), ("batch", _i32),
                ("total", _i32), ("dtype", _i32)]


class AttnParams(ctypes.Structure):
    """Mirror of `Fa2Kv8AttnParams`."""

    _fields_ = [("cache", Kv8Cache), ("q", _p), ("o", _p), ("q_stride", _i64 * 4), ("o_stride", _i64 * 4),
                ("block_table", _p), ("cache_seqlens", _p), ("cu_seqlens_q", _p), ("err_flag", _p),
                ("workspace", _p), ("workspace_bytes", _i64), ("block_table_stride", _i64), ("timeout_cycles", _i64),
                ("pages_per_seq", _i32), ("batch", _i32), ("heads_q", _i32), ("seqlen_q", _i32), ("total_q", _i32),
                ("max_seqlen_k", _i32), ("dtype", _i32), ("causal", _i32), ("causal_align", _i32),
                ("num_splits", _i32), ("qk_scale", ctypes.c_float), ("reserved", _i32)]


STRUCTS = (RotaryParams, AppendParams, ReadParams, AttnParams)
_lib = None


def lib():
    """Load (once) and return the native library, checking its ABI version and struct sizes."""
    global _lib
    if _lib is not None:
        return _lib
    if not os.path.exists(LIB_PATH):
        raise ImportError(f"{LIB_PATH} is missing: build it with `python triton-fa2-forward_b200/build.py`")
    L = ctypes.CDLL(LIB_PATH)
    L.fa2_kvcache_sm100_abi_version.argtypes = []
    L.fa2_kvcache_sm100_abi_version.restype = ctypes.c_int
    L.fa2_kvcache_sm100_params_size.argtypes = [_i32]
    L.fa2_kvcache_sm100_params_size.restype = _i64
    for name, struct in (("fa2_rotary_sm100", RotaryParams), ("fa2_kv8_append_sm100", AppendParams),
                         ("fa2_kv8_read_sm100", ReadParams), ("fa2_kv8_attn_sm100", AttnParams)):
        f, check = getattr(L, name), getattr(L, name + "_check")
        f.argtypes, f.restype = [ctypes.POINTER(struct), _p], ctypes.c_int
        check.argtypes, check.restype = [ctypes.POINTER(struct)], ctypes.c_int
    L.fa2_kv8_attn_sm100_workspace_bytes.argtypes = [ctypes.POINTER(AttnParams)]
    L.fa2_kv8_attn_sm100_workspace_bytes.restype = _i64
    if L.fa2_kvcache_sm100_abi_version() != ABI_VERSION:
        raise ImportError(f"{LIB_PATH}: ABI version {L.fa2_kvcache_sm100_abi_version()} != {ABI_VERSION}")
    for i, struct in enumerate(STRUCTS):
        if L.fa2_kvcache_sm100_params_size(i) != ctypes.sizeof(struct):
            raise ImportError(f"{LIB_PATH}: size of {struct.__name__} {L.fa2_kvcache_sm100_params_size(i)} != "
                              f"ctypes mirror {ctypes.sizeof(struct)}")
    _lib = L
    return L


def launch(name, params, stream_handle):
    """Runs one entry point; raises Fa2Error for a status other than OK."""
    rc = getattr(lib(), name)(ctypes.byref(params), _p(stream_handle or None))
    if rc != 0:
        raise Fa2Error(rc, strerror(rc))
