"""ctypes mirrors of the parameter blocks of include/fa_kv.h and include/fa_rope.h (libfa_kv.so): the same boundary that
csrc/fa_kv_aten.cpp binds, for hosts that come through ctypes."""
from __future__ import annotations

import ctypes
import os

_HERE = os.path.dirname(os.path.abspath(__file__))
LIB_PATH = os.path.join(_HERE, "lib", "libfa_kv.so")

FA_KV_ABI_VERSION = 1
FA_KV_E4M3, FA_KV_INT8 = 0, 1
FA_KV_MAX_BATCH = 8192
FA_DTYPE_FP32 = 2
FA_ROPE_MAX_AXES = 8

# every symbol the two headers declare
EXPORTED_SYMBOLS = (
    "fa_kv_version", "fa_kv_error_string", "fa_kv_plan_validate", "fa_kv_plan_launch", "fa_kv_write_validate", "fa_kv_write_launch",
    "fa_kv_attn_validate", "fa_kv_attn_workspace_bytes", "fa_kv_attn_launch", "fa_rope_validate", "fa_rope_launch",
)


def _ptrs(*names):
    return [(n, ctypes.c_void_p) for n in names]


def _longs(*names):
    return [(n, ctypes.c_int64) for n in names]


def _ints(*names):
    return [(n, ctypes.c_int32) for n in names]


def _strides(prefix, dims):
    return _longs(*(f"{prefix}_stride_{d}" for d in dims))


class FaKvPlanParams(ctypes.Structure):
    """Mirror of `struct fa_kv_plan_params`."""

    _fields_ = (_ptrs("cached", "new_tokens", "block_table", "free_pages", "free_count", "cu_seqlens", "seqused", "positions", "slots",
                      "admitted", "free_left")
                + _longs("block_table_stride")
                + _ints("batch", "table_pages", "page_size", "max_tokens", "free_capacity", "reserved"))


class FaKvWriteParams(ctypes.Structure):
    """Mirror of `struct fa_kv_write_params`."""

    _fields_ = (_ptrs("key", "value", "key_pages", "value_pages", "key_scales", "value_scales", "slots")
                + _strides("key", "th") + _strides("value", "th") + _strides("kp", "psh") + _strides("vp", "psh")
                + _strides("ks", "pbh") + _strides("vs", "pbh")
                + _ints("tokens", "heads", "head_dim", "num_pages", "page_size", "scale_block", "dtype", "format"))


class FaKvAttnParams(ctypes.Structure):
    """Mirror of `struct fa_kv_attn_params`."""

    _fields_ = (_ptrs("q", "key_pages", "value_pages", "key_scales", "value_scales", "out", "lse", "block_table", "seqused_k", "cu_seqlens_q")
                + _strides("q", "bsh") + _strides("kp", "psh") + _strides("vp", "psh") + _strides("ks", "pbh") + _strides("vs", "pbh")
                + _strides("o", "bsh") + _strides("lse", "bhs") + _longs("block_table_stride")
                + _ints("batch", "heads_q", "heads_k", "seqlen_q", "total_q", "head_dim", "num_pages", "table_pages", "page_size", "scale_block")
                + [("scale", ctypes.c_float)] + _ints("dtype", "format", "is_causal", "num_splits", "reserved"))


class FaRopeParams(ctypes.Structure):
    """Mirror of `struct fa_rope_params`."""

    _fields_ = (_ptrs("q", "k", "q_out", "k_out", "positions", "inv_freq", "axes")
                + _strides("q", "bsh") + _strides("k", "bsh") + _strides("qo", "bsh") + _strides("ko", "bsh") + _strides("pos", "abs")
                + _ints("batch", "seqlen", "heads_q", "heads_k", "head_dim", "pairs", "num_axes", "dtype", "positions_64", "inv_freq_64",
                        "interleaved", "inverse"))


_lib = None


def lib() -> ctypes.CDLL:
    """Load libfa_kv.so (built in-tree by torch_mlu_amd._build); raises if it is missing."""
    global _lib
    if _lib is None:
        if not os.path.exists(LIB_PATH):
            raise ImportError(f"{LIB_PATH} is missing: build it with `python -c 'import __graft_entry__ as g; g.build()'`; there is no fallback path")
        L = ctypes.CDLL(LIB_PATH)
        L.fa_kv_version.restype, L.fa_kv_version.argtypes = ctypes.c_int, []
        L.fa_kv_error_string.restype, L.fa_kv_error_string.argtypes = ctypes.c_char_p, [ctypes.c_int]
        for name, struct in (("fa_kv_plan", FaKvPlanParams), ("fa_kv_write", FaKvWriteParams), ("fa_kv_attn", FaKvAttnParams), ("fa_rope", FaRopeParams)):
            ptr = ctypes.POINTER(struct)
            f = getattr(L, name + "_validate")
            f.restype, f.argtypes = ctypes.c_int, [ptr]
            f = getattr(L, name + "_launch")
            f.restype = ctypes.c_int
            f.argtypes = [ptr, ctypes.c_void_p, ctypes.c_size_t, ctypes.c_void_p] if name == "fa_kv_attn" else [ptr, ctypes.c_void_p]
        L.fa_kv_attn_workspace_bytes.restype, L.fa_kv_attn_workspace_bytes.argtypes = ctypes.c_size_t, [ctypes.POINTER(FaKvAttnParams)]
        _lib = L
    return _lib
