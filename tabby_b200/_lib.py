"""ctypes binding of libtabbysample.so (include/tabby_sample.h) and libtabbydecode.so
(include/tabby_decode.h).

The libraries are the product: there is no Python or CPU fallback. If a shared object is
missing or fails to load, ``lib()`` and ``decode_lib()`` raise.
"""
from __future__ import annotations

import ctypes
import os

import numpy as np

_PKG = os.path.dirname(os.path.abspath(__file__))
LIB_PATH = os.path.join(_PKG, "lib", "libtabbysample.so")

TABBY_OK = 0
TABBY_EINVAL = 1
TABBY_ECUDA = 2
TABBY_ENOMEM = 3
TABBY_EINPUT = 4
TABBY_ETIMEOUT = 5
TABBY_EEMPTY = 6
TABBY_MAX_TOP_K_LIMIT = 1024
TABBY_DEFAULT_MAX_TOP_K = 64
TABBY_SHARD_TOP_K = 64
TABBY_NOALLOC_MAX_TOP_K = 256
TABBY_EXCHANGE_MAX_WORLD = 16
TABBY_EXCHANGE_HANDLE_BYTES = 64
SHARD_BLOCK_WORDS = 2 + 2 * TABBY_SHARD_TOP_K

# tabby_sampling_params (24 bytes) and tabby_sample_outcome (48 bytes).
PARAMS_DTYPE = np.dtype(
    [("temperature", "<f8"), ("top_p", "<f8"), ("top_k", "<i4"), ("reserved", "<i4")]
)
OUTCOME_DTYPE = np.dtype(
    [
        ("id", "<i4"),
        ("considered_count", "<i4"),
        ("probability", "<f8"),
        ("pool_mass", "<f8"),
        ("pool_exhausted", "<i4"),
        ("pool_size", "<i4"),
        ("max_logit", "<f4"),
        ("sum_exp", "<f4"),
        ("status", "<i4"),
        ("reserved", "<i4"),
    ]
)
assert PARAMS_DTYPE.itemsize == 24 and OUTCOME_DTYPE.itemsize == 48


class SamplerConfig(ctypes.Structure):
    _fields_ = [
        ("device", ctypes.c_int32),
        ("max_top_k", ctypes.c_int32),
        ("max_rows", ctypes.c_int32),
        ("max_vocab", ctypes.c_int32),
    ]


# Every symbol include/tabby_sample.h declares, with its ctypes signature.
_P = ctypes.c_void_p
_I32 = ctypes.c_int32
_I64 = ctypes.c_int64
_F32 = ctypes.c_float
_F64 = ctypes.c_double
SIGNATURES = {
    "tabby_abi_version": ([], _I32),
    "tabby_last_error": ([], ctypes.c_char_p),
    "tabby_pool_size": ([_F64, _I32, _I32], _I32),
    "tabby_sampler_create": ([ctypes.POINTER(SamplerConfig), ctypes.POINTER(_P)], ctypes.c_int),
    "tabby_sampler_destroy": ([_P], ctypes.c_int),
    "tabby_sample_rows_async": (
        [_P, _P, _I64, _I32, _I32, _P, _P, _P, _P, _P, _I32, _P], ctypes.c_int),
    "tabby_softmax_rows_async": ([_P, _I32, _I32, _I32, _I32, _P], ctypes.c_int),
    "tabby_sample_rows_rng_async": (
        [_P, _P, _I64, _I32, _I32, _P, _P, _P, _P, _P, _I32, _P], ctypes.c_int),
    "tabby_sample_rows_debug_async": (
        [_P, _P, _I64, _I32, _I32, _P, _P, _P, ctypes.c_uint32, _I32, _P], ctypes.c_int),
    "tabby_lmhead_create": ([_I32, _I32, _I32, _I32, ctypes.POINTER(_P)], ctypes.c_int),
    "tabby_lmhead_destroy": ([_P], ctypes.c_int),
    "tabby_lmhead_sample_async": (
        [_P, _P, _P, _I32, _P, _P, _P, _P, _P, _I32, _P, _P], ctypes.c_int),
    "tabby_sample_rows": ([_P, _P, _I64, _I32, _I32, _P, _P, _P, _P, _P, _I32], ctypes.c_int),
    "tabby_topk_rows_async": ([_P, _P, _I64, _I32, _I32, _I32, _P, _I32, _P], ctypes.c_int),
    "tabby_shard_local_async": ([_P, _P, _I64, _I32, _I32, _I64, _P, _I32, _P], ctypes.c_int),
    "tabby_shard_merge_async": (
        [_P, _P, _I32, _I32, _I32, _P, _P, _P, _P, _P, _I32, _P], ctypes.c_int),
    "tabby_exchange_create": ([_I32, _I32, _I32, _I32, ctypes.POINTER(_P)], ctypes.c_int),
    "tabby_exchange_ipc_handle": ([_P, _P], ctypes.c_int),
    "tabby_exchange_open": ([_P, _P], ctypes.c_int),
    "tabby_exchange_blocks": ([_P, ctypes.POINTER(_P), ctypes.POINTER(_I32)], ctypes.c_int),
    "tabby_exchange_merge_async": ([_P, _I32, _P, _P, _P, _P], ctypes.c_int),
    "tabby_exchange_destroy": ([_P], ctypes.c_int),
    "tabby_sample_from_topk": ([_P, _P, _I32, _F32, _F32, _P, _F64, _P], ctypes.c_int),
    "tabby_sample_rows_noalloc": (
        [_P, _I64, _I32, _I32, _I32, _P, _P, _P, _P, _P, _I32, _P], ctypes.c_int),
}

TABBY_BEAM_MAX = 64
TABBY_BEAM_MAX_OUT = 128
TABBY_TREE_MAX_NODES = 64
TABBY_TREE_MAX_DIM = 128
TABBY_F32, TABBY_BF16, TABBY_F16 = 0, 1, 2
DECODE_LIB_PATH = os.path.join(_PKG, "lib", "libtabbydecode.so")
DECODE_TORCH_PATH = os.path.join(_PKG, "lib", "tabby_decode_torch.so")


class StateLayout(ctypes.Structure):
    _fields_ = [
        ("row_stride", _I64),
        ("segment_stride", _I64),
        ("entry_stride", _I64),
        ("entry_bytes", _I64),
        ("segments", _I32),
        ("entries", _I32),
    ]


class TreeAttentionArgs(ctypes.Structure):
    _fields_ = [
        *[(n, _P) for n in ("q", "k", "v", "out")],
        *[(f"{t}_{d}_stride", _I64) for t, ds in (("q", ("batch", "node", "head")),
                                                  ("k", ("batch", "head", "entry")),
                                                  ("v", ("batch", "head", "entry")),
                                                  ("out", ("batch", "node", "head")))
          for d in ds],
        ("lengths", _P),
        ("parents", _P),
        ("parents_stride", _I64),
        *[(n, _I32) for n in ("dtype", "batch", "nodes", "heads", "kv_heads", "dim", "entries")],
        ("scale", _F32),
        ("workspace", _P),
        ("workspace_bytes", ctypes.c_size_t),
    ]


# Every symbol include/tabby_decode.h declares, with its ctypes signature.
DECODE_SIGNATURES = {
    "tabby_decode_abi_version": ([], _I32),
    "tabby_decode_last_error": ([], ctypes.c_char_p),
    "tabby_beam_workspace_bytes": (
        [_I32, _I32, _I32, _I32, ctypes.POINTER(ctypes.c_size_t)], ctypes.c_int),
    "tabby_beam_step_async": (
        [_I32, _P, _I32, _I64, _I64, _I32, _I32, _I32, _P, _P, _I32, _I32, _P, _P, _P, _P, _P,
         _P, ctypes.c_size_t, _P], ctypes.c_int),
    "tabby_states_reorder_async": (
        [_I32, _P, _I32, ctypes.POINTER(StateLayout), _I32, _I32, _P, _P, _P], ctypes.c_int),
    "tabby_tree_workspace_bytes": (
        [_I32, _I32, _I32, _I32, _I32, ctypes.POINTER(ctypes.c_size_t)], ctypes.c_int),
    "tabby_tree_attention_async": (
        [_I32, ctypes.POINTER(TreeAttentionArgs), _P], ctypes.c_int),
    "tabby_tree_accept_async": (
        [_I32, _P, _I64, _I64, _P, _P, _I64, _I32, _I32, _P, _P, _P, _P, _P, _P, _I32,
         ctypes.POINTER(StateLayout), _P], ctypes.c_int),
}

_lib = None
_decode_lib = None


class TabbyError(RuntimeError):
    def __init__(self, status: int, message: str):
        super().__init__(f"[tabby status {status}] {message}")
        self.status = status


def _load(path: str, signatures: dict) -> ctypes.CDLL:
    if not os.path.exists(path):
        raise RuntimeError(f"{path} is missing; build it with `python -m tabby_b200.build`")
    l = ctypes.CDLL(path)
    for name, (args, res) in signatures.items():
        fn = getattr(l, name)
        fn.argtypes = args
        fn.restype = res
    return l


def lib() -> ctypes.CDLL:
    """Load the shared library (raises if it is missing: no fallback exists)."""
    global _lib
    if _lib is None:
        _lib = _load(LIB_PATH, SIGNATURES)
    return _lib


def decode_lib() -> ctypes.CDLL:
    """Load the decode operators' library (raises if it is missing: no fallback exists)."""
    global _decode_lib
    if _decode_lib is None:
        _decode_lib = _load(DECODE_LIB_PATH, DECODE_SIGNATURES)
    return _decode_lib


def check(status: int) -> None:
    if status != TABBY_OK:
        raise TabbyError(status, lib().tabby_last_error().decode(errors="replace"))
