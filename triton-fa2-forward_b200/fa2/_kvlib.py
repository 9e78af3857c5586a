"""ctypes binding of the C ABI in include/fa2_kvcache_sm100.h (libfa2_kvcache_sm100.so, built
in-tree): rotary positions, the 8-bit paged K/V cache, attention over it. As in `_lib`, the library
is required; there is no CPU or library fallback.
"""

import ctypes
import os
import struct

import torch

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


class Layout:
    """A parameter struct: its fields' names in order, and the packing of their values (arrays flat).
    Packed at once into bytes, which costs a call a third of what setting ctypes fields does."""

    def __init__(self, *fields):
        self.fields = [(name, code) for name, code in fields]
        self.packer = struct.Struct("@" + "".join(code for _, code in fields))
        self.pack, self.size = self.packer.pack, self.packer.size


# Native alignment and sizes, as the C compiler lays the structs out. CACHE is the head of three.
CACHE = (("k", "P"), ("v", "P"), ("k_scale", "P"), ("v_scale", "P"), ("k_stride", "3q"), ("v_stride", "3q"),
         ("ks_stride", "3q"), ("vs_stride", "3q"), ("num_pages", "i"), ("page_size", "i"), ("heads_kv", "i"),
         ("head_dim", "i"))
ROTARY = Layout(("q", "P"), ("k", "P"), ("q_out", "P"), ("k_out", "P"), ("q_stride", "4q"), ("k_stride", "4q"),
                ("q_out_stride", "4q"), ("k_out_stride", "4q"), ("positions", "P"), ("pos_stride", "2q"),
                ("inv_freq", "P"), ("pos_is_64", "i"), ("batch", "i"), ("seqlen", "i"), ("heads_q", "i"),
                ("heads_kv", "i"), ("head_dim", "i"), ("rotary_dim", "i"), ("dtype", "i"), ("interleaved", "i"),
                ("inverse", "i"), ("magnitude", "f"), ("reserved", "i"))
APPEND = Layout(*CACHE, ("k_in", "P"), ("v_in", "P"), ("k_in_stride", "4q"), ("v_in_stride", "4q"),
                ("block_table", "P"), ("cache_seqlens", "P"), ("cu_seqlens", "P"), ("err_flag", "P"),
                ("block_table_stride", "q"), ("pages_per_seq", "i"), ("batch", "i"), ("seqlen", "i"), ("dtype", "i"))
READ = Layout(*CACHE, ("k_out", "P"), ("v_out", "P"), ("block_table", "P"), ("cu_seqlens", "P"), ("err_flag", "P"),
              ("block_table_stride", "q"), ("pages_per_seq", "i"), ("batch", "i"), ("total", "i"), ("dtype", "i"))
ATTN = Layout(*CACHE, ("q", "P"), ("o", "P"), ("q_stride", "4q"), ("o_stride", "4q"), ("block_table", "P"),
              ("cache_seqlens", "P"), ("cu_seqlens_q", "P"), ("err_flag", "P"), ("workspace", "P"),
              ("workspace_bytes", "q"), ("block_table_stride", "q"), ("timeout_cycles", "q"), ("pages_per_seq", "i"),
              ("batch", "i"), ("heads_q", "i"), ("seqlen_q", "i"), ("total_q", "i"), ("max_seqlen_k", "i"),
              ("dtype", "i"), ("causal", "i"), ("causal_align", "i"), ("num_splits", "i"), ("qk_scale", "f"),
              ("reserved", "i"))

STRUCTS = (ROTARY, APPEND, READ, ATTN)  # the order of fa2_kvcache_sm100_params_size
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
    for name in ("fa2_rotary_sm100", "fa2_kv8_append_sm100", "fa2_kv8_read_sm100", "fa2_kv8_attn_sm100"):
        f, check = getattr(L, name), getattr(L, name + "_check")
        f.argtypes, f.restype = [ctypes.c_char_p, _p], ctypes.c_int  # the packed struct, read only
        check.argtypes, check.restype = [ctypes.c_char_p], ctypes.c_int
    L.fa2_kv8_attn_sm100_workspace_bytes.argtypes = [ctypes.c_char_p]
    L.fa2_kv8_attn_sm100_workspace_bytes.restype = _i64
    if L.fa2_kvcache_sm100_abi_version() != ABI_VERSION:
        raise ImportError(f"{LIB_PATH}: ABI version {L.fa2_kvcache_sm100_abi_version()} != {ABI_VERSION}")
    for i, layout in enumerate(STRUCTS):
        if L.fa2_kvcache_sm100_params_size(i) != layout.size:
            raise ImportError(f"{LIB_PATH}: size of struct {i} {L.fa2_kvcache_sm100_params_size(i)} != {layout.size} packed")
    _lib = L
    return L


def launch(entry, packed, index):
    """Runs one entry point of lib() on torch's current stream of CUDA device `index`; raises
    Fa2Error for a status other than OK."""
    if index == torch.cuda.current_device():
        rc = entry(packed, torch._C._cuda_getCurrentRawStream(index))
    else:
        with torch.cuda.device(index):
            rc = entry(packed, torch._C._cuda_getCurrentRawStream(index))
    if rc != 0:
        raise Fa2Error(rc, strerror(rc))
