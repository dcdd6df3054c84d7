"""ctypes binding of libmssample.so (the C ABI in include/mssample.h).

There is no fallback: if the library is missing or no CUDA device is
present, every sampling call raises.
"""
from __future__ import annotations

import ctypes
import os
import threading

HERE = os.path.dirname(os.path.abspath(__file__))
LIB_PATH = os.path.join(HERE, "libmssample.so")

MS_OK = 0
MS_E_TOO_LARGE = -5
MS_DTYPE_F32 = 0
MS_DTYPE_BF16 = 1
MS_DTYPE_F16 = 2
MS_ROW_OK = 0
MS_ROW_ALL_MASKED = 1
MS_ROW_BAD_TEMPERATURE = 2
MS_ROW_NONFINITE = 4
MS_ROW_UNSUPPORTED = 8
MS_ROW_PEER_TIMEOUT = 16
MS_ROW_BAD_SLOT = 32
MS_ROW_BAD_POSITION = 64
MS_ROW_BAD_LENGTH = 128
MS_ROW_BAD_PAGE = 256
MS_ROW_WAIT_TIMEOUT = 512

BINDING_PATH = os.path.join(HERE, "_binding.so")

_lock = threading.Lock()
_lib = None
_binding = None

_P = ctypes.c_void_p
_I64 = ctypes.c_int64
_I32 = ctypes.c_int32


class KvAppendArgs(ctypes.Structure):
    """ms_kv_append_args of include/mssample.h."""
    _fields_ = [("dtype", _I32), ("heads", _I32), ("kv_heads", _I32), ("head_dim", _I32), ("rotary", _I32),
                ("interleaved", _I32), ("tokens", _I64),
                ("q", _P), ("q_token", _I64), ("q_head", _I64), ("k", _P), ("k_token", _I64), ("k_head", _I64),
                ("v", _P), ("v_token", _I64), ("v_head", _I64), ("q_out", _P), ("q_out_token", _I64),
                ("q_out_head", _I64), ("cache_k", _P), ("ck_page", _I64), ("ck_token", _I64), ("ck_head", _I64),
                ("cache_v", _P), ("cv_page", _I64), ("cv_token", _I64), ("cv_head", _I64), ("pages", _I64),
                ("page_size", _I64), ("slots", _P), ("positions", _P), ("table", _P), ("table_rows", _I64),
                ("status", _P)]


class PrefixAttentionArgs(ctypes.Structure):
    """ms_prefix_attention_args of include/mssample.h."""
    _fields_ = [("dtype", _I32), ("heads", _I32), ("kv_heads", _I32), ("head_dim", _I32), ("rows", _I64),
                ("q", _P), ("q_row", _I64), ("q_head", _I64), ("cache_k", _P), ("ck_page", _I64), ("ck_token", _I64),
                ("ck_head", _I64), ("cache_v", _P), ("cv_page", _I64), ("cv_token", _I64), ("cv_head", _I64),
                ("pages", _I64), ("page_size", _I64), ("table", _P), ("table_width", _I64), ("table_row", _I64),
                ("lengths", _P), ("prefix_pages", _P), ("prefix_length", _I64), ("scale", ctypes.c_float),
                ("out", _P), ("out_row", _I64), ("out_head", _I64), ("lse", _P), ("status", _P), ("workspace", _P),
                ("workspace_bytes", _I64)]


# name -> (restype, argtypes); every function include/mssample.h declares
SIGNATURES = {
    "ms_sample": (ctypes.c_int, [_P, ctypes.c_int, _I64, _I64, _I64, _P, _P, _P, _P, _P, _I64,
                                 _P, _P, _P, _P]),
    "ms_sample_generic": (ctypes.c_int, [_P, ctypes.c_int, _I64, _I64, _I64, _P, _P, _P, _P, _P,
                                         _I64, _P, _P, _P, _P]),
    "ms_shard_candidates": (ctypes.c_int, [_P, ctypes.c_int, _I64, _I64, _I64, _I64, _I64, _P, _P, _P,
                                           _I64, ctypes.c_int32, _P, _P]),
    "ms_nucleus_hist_words": (_I64, []),
    "ms_nucleus_record_words": (_I64, []),
    "ms_nucleus_cut_words": (_I64, []),
    "ms_nucleus_segments": (_I64, []),
    "ms_nucleus_hist": (ctypes.c_int, [_P, ctypes.c_int, _I64, _I64, _P, _I64, _P, _I64, _I64, _I64, _P,
                                       ctypes.c_int32, ctypes.c_int32, _P, _P, _P, _P]),
    "ms_nucleus_bracket": (ctypes.c_int, [_P, _P, _I64, _I64, _P, _P, _P]),
    "ms_nucleus_classify": (ctypes.c_int, [_P, ctypes.c_int, _I64, _I64, _I64, _P, _I64, _P, _I64, _I64, _P,
                                           ctypes.c_int32, ctypes.c_int32, _P, _P, _P, _P, _P]),
    "ms_nucleus_cut": (ctypes.c_int, [_P, ctypes.c_int32, _P, _P, _P, _I64, _I64, _P, ctypes.c_int32, _P, _P, _P,
                                      _P, _P]),
    "ms_nucleus_draw": (ctypes.c_int, [_P, ctypes.c_int, _I64, _I64, _I64, _P, _I64, _P, _I64, _I64, _P,
                                       ctypes.c_int32, ctypes.c_int32, _P, _P, _P, _P, ctypes.c_int32, _P, _P]),
    "ms_build_json_mask_noalloc": (ctypes.c_int, [_P, _I64, _P, _P, _I64, _P, _I64, _P, _P]),
    "ms_mask_from_logits": (ctypes.c_int, [_P, ctypes.c_int, _I64, _I64, _I64, _P, _I64, _P]),
    "ms_shard_record_words": (_I64, [ctypes.c_int32]),
    "ms_shard_merge": (ctypes.c_int, [_P, ctypes.c_int32, _I64, ctypes.c_int32, _I64, _P, _P, _P, _P,
                                      _P, _P, _P, _P]),
    "ms_exchange_words": (_I64, [_I64, ctypes.c_int32, ctypes.c_int32]),
    "ms_exchange_records_offset": (_I64, [_I64, ctypes.c_int32, ctypes.c_int32, ctypes.c_uint32]),
    "ms_shard_exchange": (ctypes.c_int, [_P, ctypes.c_int, _I64, _I64, _I64, _I64, _I64, _P, _P, _P, _P, _P,
                                         _I64, ctypes.c_int32, _P, _P, ctypes.c_int32, ctypes.c_int32, _I64,
                                         ctypes.c_int32, ctypes.c_uint32, _P]),
    "ms_exchange_merge": (ctypes.c_int, [_P, _P, ctypes.c_int32, ctypes.c_int32, _I64, _I64, ctypes.c_int32,
                                         ctypes.c_int32, _I64, _P, _P, _P, _P, ctypes.c_uint32, _I64, _P, _P, _P,
                                         _P]),
    "ms_exchange_results": (ctypes.c_int, [_P, ctypes.c_int32, _I64, _I64, ctypes.c_int32, ctypes.c_uint32, _I64,
                                           _P, _P, _P, _P]),
    "ms_device_alloc": (ctypes.c_int, [_I64, ctypes.POINTER(ctypes.c_void_p)]),
    "ms_device_free": (ctypes.c_int, [_P]),
    "ms_ipc_handle": (ctypes.c_int, [_P, ctypes.c_char_p]),
    "ms_ipc_open": (ctypes.c_int, [ctypes.c_char_p, ctypes.POINTER(ctypes.c_void_p)]),
    "ms_ipc_close": (ctypes.c_int, [_P]),
    "ms_json_state_words": (_I64, []),
    "ms_json_init": (ctypes.c_int, [_P, _P, _I64, _P, _P]),
    "ms_json_advance": (ctypes.c_int, [_P, _I64, _P, _P, _I64, _P, _P]),
    "ms_build_json_mask": (ctypes.c_int, [_P, _I64, _P, _P, _I64, _P, _I64, _P, _P]),
    "ms_json_pack_vocab": (ctypes.c_int, [_P, _P, _I64, _P, _P, _P]),
    "ms_build_json_mask_packed": (ctypes.c_int, [_P, _I64, _P, _P, _P, _P, _I64, _P, _I64, _P, _P]),
    "ms_json_pack_vocab_ordered": (ctypes.c_int, [_P, _P, _I64, _P, _P, _P, _P]),
    "ms_build_json_mask_ordered": (ctypes.c_int, [_P, _I64, _P, _P, _P, _P, _P, _I64, _P, _I64, _P, _P]),
    "ms_kv_append": (ctypes.c_int, [ctypes.POINTER(KvAppendArgs), _P]),
    "ms_quantize_rows": (ctypes.c_int, [_P, ctypes.c_int, _I64, _I64, _I64, _P, _I64, _P, _P]),
    "ms_int8_matmul": (ctypes.c_int, [_P, _I64, _P, _I64, _P, _I64, _P, _I64, _I64, _P, _P, ctypes.c_int, _I64, _P]),
    "ms_int8_workspace": (_I64, [_I64, _I64]),
    "ms_int8_linear": (ctypes.c_int, [_P, ctypes.c_int, _I64, _I64, _P, _I64, _P, _I64, _I64, _P, _P, ctypes.c_int,
                                      _I64, _P, _P]),
    "ms_prefix_attention": (ctypes.c_int, [ctypes.POINTER(PrefixAttentionArgs), _P]),
    "ms_prefix_attention_workspace": (_I64, [_I64, _I32, _I32, _I32, _I64]),
    "ms_error_string": (ctypes.c_char_p, [ctypes.c_int]),
    "ms_last_cuda_error": (ctypes.c_int, []),
    "ms_version": (ctypes.c_int, []),
}


class SamplerLibraryError(RuntimeError):
    pass


def lib():
    """Load libmssample.so once; raise if it has not been built."""
    global _lib
    if _lib is not None:
        return _lib
    with _lock:
        if _lib is None:
            if not os.path.exists(LIB_PATH):
                raise SamplerLibraryError(
                    f"{LIB_PATH} is missing: build it with `python -m miniserve_b200.build` "
                    "(there is no CPU fallback)")
            handle = ctypes.CDLL(LIB_PATH)
            for name, (res, args) in SIGNATURES.items():
                fn = getattr(handle, name)
                fn.restype = res
                fn.argtypes = args
            _lib = handle
    return _lib


def binding():
    """Load _binding.so once, with the library's entry points; raise if it has
    not been built for this torch."""
    global _binding
    if _binding is not None:
        return _binding
    import importlib.machinery
    import importlib.util

    import torch
    handle = lib()
    with _lock:
        if _binding is None:
            if not os.path.exists(BINDING_PATH):
                raise SamplerLibraryError(
                    f"{BINDING_PATH} is missing: build it with `python -m miniserve_b200.build`")
            loader = importlib.machinery.ExtensionFileLoader("miniserve_b200._binding", BINDING_PATH)
            try:
                module = importlib.util.module_from_spec(
                    importlib.util.spec_from_file_location("miniserve_b200._binding", BINDING_PATH, loader=loader))
                loader.exec_module(module)
            except ImportError as e:  # another torch's symbols, before the version could be compared
                raise SamplerLibraryError(f"{BINDING_PATH} cannot be loaded with torch {torch.__version__}: build it "
                                          f"again with `python -m miniserve_b200.build` ({e})") from e
            if module.torch_version != torch.__version__.split("+")[0]:
                raise SamplerLibraryError(f"{BINDING_PATH} was built for torch {module.torch_version}, this is "
                                          f"{torch.__version__}: build it again")
            module.bind(*(ctypes.cast(getattr(handle, name), ctypes.c_void_p).value for name in (
                "ms_kv_append", "ms_prefix_attention", "ms_prefix_attention_workspace", "ms_int8_linear",
                "ms_int8_workspace")))
            _binding = module
    return _binding


def check(rc: int, what: str) -> None:
    if rc != MS_OK:
        L = lib()
        msg = L.ms_error_string(rc).decode()
        if rc == -3:
            msg += f" (cudaError {L.ms_last_cuda_error()})"
        raise SamplerLibraryError(f"{what} failed: {msg}")
