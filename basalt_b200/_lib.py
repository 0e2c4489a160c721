"""ctypes binding of libbasalt_cuda.so (include/basalt_cuda.h).

There is no CPU fallback: if the library is missing, loading raises. A missing GPU surfaces as a
``BasaltUnsupportedOperationException`` from the first engine call, never as a silent switch to
another implementation.
"""
from __future__ import annotations

import ctypes
import operator
from pathlib import Path

PACKAGE = Path(__file__).resolve().parent
LIBRARY = PACKAGE / "libbasalt_cuda.so"
HEADER = PACKAGE.parent / "include" / "basalt_cuda.h"

BST_OK = 0
BST_INVALID = -1
BST_SHAPE = -2
BST_UNKNOWN_HANDLE = -3
BST_CONTEXT = -4
BST_GRAPH = -5
BST_PANIC = -6
BST_OOM = -7
BST_UNSUPPORTED = -8

FAMILY_PADDED_DECODER = 1
FAMILY_DECODER = 2
FAMILY_CHAR_LM = 3
FAMILY_LAST_TOKEN = 4

DTYPE_F32 = 0
DTYPE_BF16 = 1
DTYPE_U4 = 2

KERNEL_CLASSES = 15


class ModelSpecStruct(ctypes.Structure):
    _fields_ = [("family", ctypes.c_int32), ("vocabulary", ctypes.c_int32),
                ("window", ctypes.c_int32), ("dimension", ctypes.c_int32),
                ("layers", ctypes.c_int32), ("heads", ctypes.c_int32),
                ("hidden", ctypes.c_int32), ("weight_dtype", ctypes.c_int32),
                ("kv_dtype", ctypes.c_int32), ("max_rows", ctypes.c_int32),
                ("attention_window", ctypes.c_int32), ("attention_sinks", ctypes.c_int32),
                ("reserved", ctypes.c_int32 * 4)]


class SequencesStruct(ctypes.Structure):
    _fields_ = [("count", ctypes.c_int32), ("tokens", ctypes.c_int32),
                ("rows", ctypes.c_void_p), ("starts", ctypes.c_void_p),
                ("lengths", ctypes.c_void_p)]


class KvCacheStruct(ctypes.Structure):
    _fields_ = [("storage", ctypes.c_int32), ("rows", ctypes.c_int32),
                ("kv_heads", ctypes.c_int32), ("slots", ctypes.c_int32),
                ("head_dim", ctypes.c_int32), ("reserved", ctypes.c_int32 * 3),
                ("k", ctypes.c_void_p), ("v", ctypes.c_void_p),
                ("k_scale", ctypes.c_void_p), ("v_scale", ctypes.c_void_p)]


class AttentionSpecStruct(ctypes.Structure):
    _fields_ = [("heads", ctypes.c_int32), ("kv_heads", ctypes.c_int32),
                ("head_dim", ctypes.c_int32), ("dtype", ctypes.c_int32),
                ("window", ctypes.c_int32), ("sinks", ctypes.c_int32),
                ("scale", ctypes.c_float), ("reserved", ctypes.c_int32)]


class SamplingStruct(ctypes.Structure):
    _fields_ = [("temperature", ctypes.c_float), ("top_p", ctypes.c_float),
                ("min_p", ctypes.c_float), ("top_k", ctypes.c_int32),
                ("temperatures", ctypes.c_void_p), ("top_ps", ctypes.c_void_p),
                ("min_ps", ctypes.c_void_p), ("top_ks", ctypes.c_void_p)]


def int32(value) -> int:
    """The nearest 32-bit whole number, for counts of which those beyond mean no more than it (ctypes
    would drop their upper bits)."""
    return max(-2 ** 31, min(2 ** 31 - 1, operator.index(value)))


TOKEN_SINK = ctypes.CFUNCTYPE(ctypes.c_int32, ctypes.c_void_p, ctypes.c_int32, ctypes.c_int32,
                              ctypes.c_int32)

_P = ctypes.POINTER
_i32p = _P(ctypes.c_int32)
_i64p = _P(ctypes.c_int64)
_f32p = _P(ctypes.c_float)
_f64p = _P(ctypes.c_double)
_u64 = ctypes.c_uint64

SIGNATURES = {
    "bst_abi_version": (ctypes.c_int32, []),
    "bst_device_count": (ctypes.c_int32, [_i32p]),
    "bst_engine_create": (ctypes.c_int32, [_P(ModelSpecStruct), ctypes.c_int32, _P(_u64)]),
    "bst_engine_destroy": (ctypes.c_int32, [_u64]),
    "bst_parameter_count": (ctypes.c_int32, [_u64, _i32p]),
    "bst_parameter_info": (ctypes.c_int32, [_u64, ctypes.c_int32, ctypes.c_char_p,
                                            ctypes.c_int32, _i64p]),
    "bst_set_parameter": (ctypes.c_int32, [_u64, ctypes.c_char_p, _f32p, ctypes.c_int64]),
    "bst_get_parameter": (ctypes.c_int32, [_u64, ctypes.c_char_p, _f32p, ctypes.c_int64]),
    "bst_save": (ctypes.c_int32, [_u64, ctypes.c_char_p]),
    "bst_load": (ctypes.c_int32, [_u64, ctypes.c_char_p]),
    "bst_scores": (ctypes.c_int32, [_u64, _i32p, ctypes.c_int32, ctypes.c_int32, _f64p]),
    "bst_generate": (ctypes.c_int32, [_u64, _i32p, ctypes.c_int32, ctypes.c_int32,
                                      ctypes.c_int32, _i32p, TOKEN_SINK, ctypes.c_void_p]),
    "bst_sample": (ctypes.c_int32, [_u64, _i32p, ctypes.c_int32, ctypes.c_int32,
                                    ctypes.c_int32, ctypes.c_float, ctypes.c_int32, _i32p,
                                    TOKEN_SINK, ctypes.c_void_p]),
    "bst_sample_filtered": (ctypes.c_int32, [_u64, _i32p, ctypes.c_int32, ctypes.c_int32,
                                             ctypes.c_int32, _P(SamplingStruct), _f64p, _i32p,
                                             TOKEN_SINK, ctypes.c_void_p]),
    "bst_sample_filtered_logits": (ctypes.c_int32, [_u64, _i32p, ctypes.c_int32, ctypes.c_int32,
                                                    ctypes.c_int32, _P(SamplingStruct), _f64p,
                                                    _i32p, _f32p]),
    "bst_generate_logits": (ctypes.c_int32, [_u64, _i32p, ctypes.c_int32, ctypes.c_int32,
                                             ctypes.c_int32, _i32p, _f32p]),
    "bst_sample_logits": (ctypes.c_int32, [_u64, _i32p, ctypes.c_int32, ctypes.c_int32,
                                           ctypes.c_int32, ctypes.c_float, ctypes.c_int32, _i32p,
                                           _f32p]),
    "bst_generate_logits_rows": (ctypes.c_int32, [_u64, _i32p, ctypes.c_int32, ctypes.c_int32,
                                                  ctypes.c_int32, _i32p, ctypes.c_int32, _i32p,
                                                  _f32p]),
    "bst_sample_logits_rows": (ctypes.c_int32, [_u64, _i32p, ctypes.c_int32, ctypes.c_int32,
                                                ctypes.c_int32, ctypes.c_float, ctypes.c_int32,
                                                _i32p, ctypes.c_int32, _i32p, _f32p]),
    "bst_generate_device": (ctypes.c_int32, [_u64, ctypes.c_void_p, ctypes.c_int32,
                                             ctypes.c_int32, ctypes.c_int32, ctypes.c_void_p]),
    "bst_sample_device": (ctypes.c_int32, [_u64, ctypes.c_void_p, ctypes.c_int32,
                                           ctypes.c_int32, ctypes.c_int32, ctypes.c_float,
                                           ctypes.c_int32, ctypes.c_void_p]),
    "bst_seed": (ctypes.c_int32, [_u64, ctypes.c_int64]),
    "bst_get_rng_state": (ctypes.c_int32, [_u64, _i64p]),
    "bst_set_rng_state": (ctypes.c_int32, [_u64, ctypes.c_int64]),
    "bst_begin_scope": (ctypes.c_int32, [_u64]),
    "bst_end_scope": (ctypes.c_int32, [_u64, _i32p]),
    "bst_scope_depth": (ctypes.c_int32, [_u64, _i32p]),
    "bst_engine_stats": (ctypes.c_int32, [_u64, _i64p]),
    "bst_engine_stream": (ctypes.c_int32, [_u64, _P(ctypes.c_void_p)]),
    "bst_profile_enable": (ctypes.c_int32, [_u64, ctypes.c_int32]),
    "bst_profile_reset": (ctypes.c_int32, [_u64]),
    "bst_profile_read": (ctypes.c_int32, [_u64, ctypes.c_int32, ctypes.c_char_p, ctypes.c_int32,
                                          _i64p, _f64p, _f64p, _f64p]),
    "bst_matmul": (ctypes.c_int32, [ctypes.c_int32, ctypes.c_void_p, ctypes.c_void_p,
                                    ctypes.c_void_p, ctypes.c_void_p, ctypes.c_int64,
                                    ctypes.c_int64, ctypes.c_int64]),
    "bst_matmul_static": (ctypes.c_int32, [ctypes.c_int32, ctypes.c_void_p, ctypes.c_void_p,
                                           ctypes.c_void_p, ctypes.c_void_p, ctypes.c_int64,
                                           ctypes.c_int64, ctypes.c_int64]),
    "bst_recognize_model": (ctypes.c_int32, [_P(ctypes.c_char_p), _i32p, _i64p, ctypes.c_int32,
                                             ctypes.c_int32, ctypes.c_int32, ctypes.c_int32,
                                             _P(ModelSpecStruct)]),
    "bst_engine_create_from_parameters": (ctypes.c_int32, [
        _P(ctypes.c_char_p), _i32p, _i64p, _P(_f32p), ctypes.c_int32, ctypes.c_int32,
        ctypes.c_int32, ctypes.c_int32, ctypes.c_int32, ctypes.c_int32, ctypes.c_int32,
        _P(_u64)]),
    "bst_context_create": (ctypes.c_int32, [ctypes.c_int32, _P(_u64)]),
    "bst_context_destroy": (ctypes.c_int32, [_u64]),
    "bst_tensor_create": (ctypes.c_int32, [_u64, ctypes.c_int32, _i64p, ctypes.c_int32, _f32p,
                                           _P(_u64)]),
    "bst_tensor_transfer": (ctypes.c_int32, [_u64, _u64, ctypes.c_int32, _P(_u64)]),
    "bst_tensor_read": (ctypes.c_int32, [_u64, _u64, _f32p, ctypes.c_int64]),
    "bst_tensor_write": (ctypes.c_int32, [_u64, _u64, _f32p, ctypes.c_int64]),
    "bst_tensor_info": (ctypes.c_int32, [_u64, _u64, _i32p, _i32p, _i64p, ctypes.c_int32]),
    "bst_tensor_release": (ctypes.c_int32, [_u64, _u64, _i32p]),
    "bst_execute_queue": (ctypes.c_int32, [_u64, ctypes.c_void_p, ctypes.c_int32]),
    "bst_context_stats": (ctypes.c_int32, [_u64, _i64p]),
    "bst_context_clear_graph": (ctypes.c_int32, [_u64]),
    "bst_kv_append": (ctypes.c_int32, [ctypes.c_int32, ctypes.c_void_p, _P(KvCacheStruct),
                                       _P(SequencesStruct), ctypes.c_void_p, ctypes.c_int64,
                                       ctypes.c_void_p, ctypes.c_int64, ctypes.c_int32]),
    "bst_kv_read": (ctypes.c_int32, [ctypes.c_int32, ctypes.c_void_p, _P(KvCacheStruct),
                                     _P(SequencesStruct), ctypes.c_void_p, ctypes.c_int64,
                                     ctypes.c_void_p, ctypes.c_int64, ctypes.c_int32]),
    "bst_attention_cached_workspace": (ctypes.c_int32, [_P(KvCacheStruct), _P(SequencesStruct),
                                                        _P(AttentionSpecStruct), _i64p]),
    "bst_attention_cached": (ctypes.c_int32, [ctypes.c_int32, ctypes.c_void_p, _P(KvCacheStruct),
                                              _P(SequencesStruct), _P(AttentionSpecStruct),
                                              ctypes.c_void_p, ctypes.c_int64, ctypes.c_void_p,
                                              ctypes.c_int64, ctypes.c_void_p, ctypes.c_int64]),
    "bst_attention_shared_workspace": (ctypes.c_int32, [
        _P(KvCacheStruct), _P(SequencesStruct), _P(AttentionSpecStruct), _P(KvCacheStruct), ctypes.c_int32,
        ctypes.c_int32, _i64p]),
    "bst_attention_shared": (ctypes.c_int32, [
        ctypes.c_int32, ctypes.c_void_p, _P(KvCacheStruct), _P(SequencesStruct), _P(AttentionSpecStruct),
        _P(KvCacheStruct), ctypes.c_int32, ctypes.c_int32, ctypes.c_void_p, ctypes.c_int64, ctypes.c_void_p,
        ctypes.c_int64, ctypes.c_void_p, ctypes.c_int64]),
    "bst_attention_weights_workspace": (ctypes.c_int32, [_P(KvCacheStruct), _P(SequencesStruct),
                                                         _P(AttentionSpecStruct), _i64p]),
    "bst_attention_weights": (ctypes.c_int32, [
        ctypes.c_int32, ctypes.c_void_p, _P(KvCacheStruct), _P(SequencesStruct), _P(AttentionSpecStruct),
        ctypes.c_void_p, ctypes.c_int64, ctypes.c_void_p, ctypes.c_int64, ctypes.c_void_p, ctypes.c_float,
        ctypes.c_void_p, ctypes.c_void_p, ctypes.c_int64]),
    "bst_kv_evict": (ctypes.c_int32, [
        ctypes.c_int32, ctypes.c_void_p, _P(KvCacheStruct), _P(SequencesStruct), ctypes.c_void_p,
        ctypes.c_int32, ctypes.c_int32, ctypes.c_int32, _P(KvCacheStruct), ctypes.c_void_p, ctypes.c_void_p,
        ctypes.c_void_p, ctypes.c_void_p]),
    "bst_attention_packed_workspace": (ctypes.c_int32, [_P(SequencesStruct),
                                                        _P(AttentionSpecStruct), _i64p]),
    "bst_attention_packed": (ctypes.c_int32, [ctypes.c_int32, ctypes.c_void_p,
                                              _P(SequencesStruct), _P(AttentionSpecStruct),
                                              ctypes.c_void_p, ctypes.c_int64, ctypes.c_void_p,
                                              ctypes.c_int64, ctypes.c_void_p, ctypes.c_int64,
                                              ctypes.c_void_p, ctypes.c_int64, ctypes.c_void_p,
                                              ctypes.c_int64]),
    "bst_sample_tokens": (ctypes.c_int32, [ctypes.c_int32, ctypes.c_void_p, ctypes.c_void_p,
                                           ctypes.c_int32, ctypes.c_int32, ctypes.c_int32,
                                           ctypes.c_int64, _P(SamplingStruct), ctypes.c_void_p,
                                           ctypes.c_void_p]),
    "bst_last_error": (ctypes.c_int32, [_u64, ctypes.c_char_p, ctypes.c_int32]),
    "bst_write_synthetic_weights": (ctypes.c_int32, [_P(ModelSpecStruct), ctypes.c_char_p,
                                                     ctypes.c_int64, ctypes.c_double]),
    "bst_synthetic_prompts": (ctypes.c_int32, [ctypes.c_int64, ctypes.c_int32, ctypes.c_int32,
                                               ctypes.c_int32, _i32p]),
}

_lib = None


def load() -> ctypes.CDLL:
    """Loads libbasalt_cuda.so; raises if it has not been built."""
    global _lib
    if _lib is None:
        if not LIBRARY.exists():
            raise ImportError(
                f"{LIBRARY} is missing: build it with `python -m basalt_b200.build` (nvcc, sm_100a)")
        lib = ctypes.CDLL(str(LIBRARY))
        for name, (res, args) in SIGNATURES.items():
            fn = getattr(lib, name)
            fn.restype = res
            fn.argtypes = args
        _lib = lib
    return _lib


def last_error(handle: int = 0) -> str:
    buf = ctypes.create_string_buffer(1024)
    load().bst_last_error(handle, buf, len(buf))
    return buf.value.decode(errors="replace")
