"""eakv_b200 - Python host binding of libeakv_b200.so.

The library is the product: a C-ABI shared library (include/eakv.h,
include/eakv_cuda.h) whose kernels are hand-written sm_100a CUDA. This module
is a thin ctypes layer over it that mirrors the reference's C API one for one
(petlukk/eakv include/eakv.h:25-83: same function names, same argument
meaning, same integer return codes), plus a small `Cache` convenience class.
There is no CPU implementation behind any of these calls: if the shared
library is missing or cannot be loaded, importing `lib()` raises.

Array arguments accept numpy float32 arrays (host pointers) or any object
exposing `data_ptr()` (torch CUDA tensors, device pointers) for the *_device
entry points.
"""
import ctypes
import os
import struct
from array import array

import numpy as np

EAKV_OK = 0
EAKV_ERR_IO = -1
EAKV_ERR_FORMAT = -2
EAKV_ERR_ALLOC = -3
EAKV_ERR_INVALID = -4

_HERE = os.path.dirname(os.path.abspath(__file__))
# EAKV_B200_LIB selects another build of the library (same ABI)
LIB_PATH = os.environ.get("EAKV_B200_LIB") or os.path.join(_HERE, "libeakv_b200.so")

_c = ctypes
_P = _c.c_void_p
_I = _c.c_int
_F = _c.c_float

# name -> (restype, argtypes); every symbol declared in the headers of
# include/.
SIGNATURES = {
    # eakv.h
    "eakv_cache_create": (_P, [_I, _I, _I, _I]),
    "eakv_cache_free": (None, [_P]),
    "eakv_cache_load_raw": (_I, [_P, _P, _I]),
    "eakv_cache_append": (_I, [_P, _P, _I, _I, _I]),
    "eakv_cache_advance": (_I, [_P, _I]),
    "eakv_cache_clear": (None, [_P]),
    "eakv_checkpoint": (_I, [_P]),
    "eakv_restore": (_I, [_P, _I]),
    "eakv_attention_scores": (None, [_P, _P, _I, _I, _I, _P]),
    "eakv_attention_output": (None, [_P, _P, _I, _I, _I, _P]),
    "eakv_cache_save": (_I, [_P, _c.c_char_p]),
    "eakv_cache_load": (_I, [_c.c_char_p, _c.POINTER(_P)]),
    "eakv_cache_seq_len": (_I, [_P]),
    "eakv_cache_n_layers": (_I, [_P]),
    "eakv_cache_n_heads": (_I, [_P]),
    "eakv_cache_head_dim": (_I, [_P]),
    "eakv_cache_max_seq_len": (_I, [_P]),
    "eakv_cache_compression_ratio": (_F, [_P]),
    # eakv_cuda.h
    "eakv_last_error": (_I, []),
    "eakv_last_error_string": (_c.c_char_p, []),
    "eakv_device_status": (_I, [_I, _I]),
    "eakv_set_device": (_I, [_I]),
    "eakv_cache_device": (_I, [_P]),
    "eakv_cache_device_bytes": (_c.c_size_t, [_P]),
    "eakv_cache_set_stream": (_I, [_P, _P]),
    "eakv_cache_stream": (_P, [_P]),
    "eakv_cache_synchronize": (_I, [_P]),
    "eakv_cache_load_raw_device": (_I, [_P, _P, _I]),
    "eakv_cache_append_device": (_I, [_P, _P, _I, _I, _I]),
    "eakv_cache_append_step_device": (_I, [_P, _P, _I]),
    "eakv_attention_scores_device": (_I, [_P, _P, _I, _I, _I, _P]),
    "eakv_attention_output_device": (_I, [_P, _P, _I, _I, _I, _P]),
    "eakv_attention_fused": (_I, [_P, _P, _I, _I, _I, _P]),
    "eakv_attention_fused_device": (_I, [_P, _P, _I, _I, _I, _P]),
    "eakv_decode_attention": (_I, [_P, _I, _P, _I, _P, _P]),
    "eakv_decode_attention_host": (_I, [_P, _I, _P, _I, _P, _P]),
    "eakv_decode_attention_noalloc": (_I, [_P, _I, _P, _I, _P, _P]),
    "eakv_decode_launches": (_I, [_P, _I, _I]),
    "eakv_decode_splits": (_I, [_P, _I, _I]),
    "eakv_decode_attention_partial": (_I, [_P, _I, _P, _I, _I, _I, _P, _P, _P]),
    "eakv_lse_combine": (_I, [_I, _I, _I, _P, _P, _P, _P, _P]),
    "eakv_test_force_splits": (_I, [_I]),
    "eakv_test_force_path": (_I, [_I]),
    "eakv_test_extend_registers": (_I, [_I]),
    "eakv_test_choose_splits": (_I, [_c.c_longlong, _I, _I, _I, _I, _I]),
    "eakv_test_stall": (_I, [_I, ctypes.c_uint]),
    "eakv_test_separate_merge": (_I, [_I]),
    "eakv_cache_validate": (_I, [_P, _P]),
    "eakv_cache_dequantize_device": (_I, [_P, _I, _I, _I, _I, _P, _P]),
    "eakv_cache_dequantize": (_I, [_P, _I, _I, _I, _I, _P]),
    "eakv_append_rotary": (_I, [_P, _I, _I, _P, _P, _P, _P, _P, _I, _P, _P]),
    "eakv_extend_attention": (_I, [_P, _I, _I, _P, _P, _P, _I, _F, _I, _P, _P, _P, _c.c_size_t, _P]),
    "eakv_extend_attention_depths": (_I, [_P, _I, _I, _P, _P, _P, _I, _F, _I, _P, _P, _P, _P, _c.c_size_t, _P]),
    "eakv_extend_workspace": (_I, [_P, _I, _P, _I, _I, _I, _I, _c.POINTER(_c.c_size_t)]),
    "eakv_cache_copy": (_I, [_P, _I, _I, _P, _I, _I, _P]),
    "eakv_cache_fork": (_I, [_P, _I, _I, _c.POINTER(_P)]),
    "eakv_cache_gather": (_I, [_P, _I, _P, _P, _c.c_int64, _c.c_int64, _I, _P]),
    "eakv_cache_compact": (_I, [_P, _I, _P, _c.c_int64, _c.c_int64, _I, _P]),
    "eakv_cache_read": (_I, [_P, _I, _I, _I, _P, _P, _P, _P, _c.c_int64, _P]),
    # eakv_nccl.h
    "eakv_nccl_version": (_I, []),
    "eakv_nccl_unique_id": (_I, [_P]),
    "eakv_nccl_comm_init": (_I, [_c.POINTER(_P), _I, _P, _I, _I]),
    "eakv_nccl_comm_destroy": (_I, [_P]),
    "eakv_nccl_comm_abort": (_I, [_P]),
    "eakv_decode_attention_split": (_I, [_P, _I, _P, _I, _I, _I, _P, _P, _P]),
    "eakv_decode_attention_split_host": (_I, [_P, _I, _P, _I, _P, _P, _P]),
    # eakv_ggml.h
    "eakv_quantize_row": (None, [_P, _P, _c.c_int64]),
    "eakv_dequantize_row": (None, [_P, _P, _c.c_int64]),
    "eakv_vec_dot_q4_f32": (None, [_I, _P, _c.c_size_t, _P, _c.c_size_t, _P, _c.c_size_t, _I]),
    # eakv_llama.h
    "eakv_from_llama_state": (_I, [_P, _c.c_size_t, _I, _I, _I, _I, _c.POINTER(_P)]),
    "eakv_from_llama_state_append": (_I, [_P, _P, _c.c_size_t, _I, _I, _I, _I]),
    "eakv_ggml_quantize_row_device": (_I, [_P, _P, _c.c_int64, _P]),
    "eakv_ggml_dequantize_row_device": (_I, [_P, _P, _c.c_int64, _P]),
    "eakv_ggml_vec_dot_device": (_I, [_I, _P, _c.c_size_t, _P, _c.c_size_t, _P, _c.c_size_t, _I,
                                      _P]),
}

_lib = None


def lib():
    """The loaded libeakv_b200.so (raises if it is absent: no fallback)."""
    global _lib
    if _lib is None:
        if not os.path.exists(LIB_PATH):
            raise RuntimeError(
                f"{LIB_PATH} is missing; build it with `python -m eakv_b200.build`")
        L = ctypes.CDLL(LIB_PATH)
        for name, (res, args) in SIGNATURES.items():
            fn = getattr(L, name)
            fn.restype = res
            fn.argtypes = args
        _lib = L
    return _lib


def last_error():
    L = lib()
    return L.eakv_last_error(), (L.eakv_last_error_string() or b"").decode()


class EakvError(RuntimeError):
    def __init__(self, rc, what):
        code, msg = last_error()
        super().__init__(f"{what} failed: rc={rc} ({msg})")
        self.rc = rc


def _ptr(x):
    """Pointer of a numpy array (host) or of an object with data_ptr()."""
    if x is None:
        return None
    if isinstance(x, np.ndarray):
        return x.ctypes.data
    if hasattr(x, "data_ptr"):
        return x.data_ptr()
    if isinstance(x, int):
        return x
    raise TypeError(f"cannot take a pointer of {type(x)}")


def _f32(a):
    a = np.ascontiguousarray(a, dtype=np.float32)
    return a


def _check(rc, what):
    if rc != EAKV_OK:
        raise EakvError(rc, what)
    return rc


class Cache:
    """Owning wrapper of one eakv_cache_t (device-resident Q4 cache)."""

    def __init__(self, n_layers=None, n_kv_heads=None, head_dim=None, max_seq_len=None,
                 _handle=None):
        L = lib()
        if _handle is not None:
            self.h = _handle
        else:
            self.h = L.eakv_cache_create(n_layers, n_kv_heads, head_dim, max_seq_len)
            if not self.h:
                raise EakvError(None, "eakv_cache_create")
        # fixed for the cache's life: (layers, KV heads, head_dim, device)
        self.shape = (L.eakv_cache_n_layers(self.h), L.eakv_cache_n_heads(self.h),
                      L.eakv_cache_head_dim(self.h), L.eakv_cache_device(self.h))

    # --- lifecycle ---------------------------------------------------------
    def free(self):
        if self.h:
            lib().eakv_cache_free(self.h)
            self.h = None

    def __del__(self):
        try:
            self.free()
        except Exception:
            pass

    def __enter__(self):
        return self

    def __exit__(self, *exc):
        self.free()

    @classmethod
    def load(cls, path):
        out = ctypes.c_void_p()
        _check(lib().eakv_cache_load(os.fsencode(path), ctypes.byref(out)), "eakv_cache_load")
        return cls(_handle=out.value)

    @classmethod
    def from_llama_state(cls, state, n_layers, n_kv_heads, head_dim, max_seq_len):
        """eakv_from_llama_state on a host bytes object (a llama.cpp
        sequence state); raises EakvError with the reference's code."""
        buf = np.frombuffer(state, np.uint8)
        out = ctypes.c_void_p()
        _check(lib().eakv_from_llama_state(_ptr(buf), buf.size, n_layers, n_kv_heads, head_dim,
                                           max_seq_len, ctypes.byref(out)),
               "eakv_from_llama_state")
        return cls(_handle=out.value)

    def append_llama_state(self, state, n_layers, n_kv_heads, head_dim, start_pos):
        """eakv_from_llama_state_append; returns the reference's code."""
        buf = np.frombuffer(state, np.uint8)
        return lib().eakv_from_llama_state_append(self.h, _ptr(buf), buf.size, n_layers,
                                                  n_kv_heads, head_dim, start_pos)

    # --- inspection ----------------------------------------------------------------
    def validate(self):
        """eakv_cache_validate: int32[n_layers*2] codes (0 ok, 1 NaN scale,
        2 NaN bias, 3 negative scale), index layer*2 + kv."""
        codes = np.zeros(self.n_layers * 2, np.int32)
        _check(lib().eakv_cache_validate(self.h, _ptr(codes)), "eakv_cache_validate")
        return codes

    def dequantize(self, layer, kv_idx, pos_begin, pos_end):
        """f32[n_kv_heads][pos_end - pos_begin][head_dim] on the host."""
        out = np.zeros((self.n_kv_heads, max(pos_end - pos_begin, 0), self.head_dim), np.float32)
        _check(lib().eakv_cache_dequantize(self.h, layer, kv_idx, pos_begin, pos_end, _ptr(out)),
               "eakv_cache_dequantize")
        return out

    def dequantize_device(self, layer, kv_idx, pos_begin, pos_end, d_out, stream=None):
        return _check(lib().eakv_cache_dequantize_device(self.h, layer, kv_idx, pos_begin,
                                                         pos_end, _ptr(d_out), stream),
                      "eakv_cache_dequantize_device")

    # --- copies -----------------------------------------------------------------
    def fork(self, n, max_seq_len=None):
        """eakv_cache_fork: a new cache holding the first n positions, as the cache's own
        stream leaves them (work on other streams is ordered before it by the caller)."""
        out = ctypes.c_void_p()
        if max_seq_len is None:
            max_seq_len = self.max_seq_len
        _check(lib().eakv_cache_fork(self.h, n, max_seq_len, ctypes.byref(out)), "eakv_cache_fork")
        return Cache(_handle=out.value)

    def compact(self, begin, index, stream=None):
        """eakv_cache_compact: position begin + j becomes position index[..., j].
        index: int32 device tensor [n], [heads, n] or [layers, heads, n] (a
        size of 1 is shared). stream None is the cache's own, which is not ordered
        with torch's current one."""
        index, ls, hs = _index(index, self)
        return _check(lib().eakv_cache_compact(self.h, begin, _ptr(index), ls, hs, index.shape[-1],
                                               stream), "eakv_cache_compact")

    # --- info ----------------------------------------------------------------
    @property
    def seq_len(self):
        return lib().eakv_cache_seq_len(self.h)

    @property
    def n_layers(self):
        return lib().eakv_cache_n_layers(self.h)

    @property
    def n_kv_heads(self):
        return lib().eakv_cache_n_heads(self.h)

    @property
    def head_dim(self):
        return lib().eakv_cache_head_dim(self.h)

    @property
    def max_seq_len(self):
        return lib().eakv_cache_max_seq_len(self.h)

    @property
    def device(self):
        return lib().eakv_cache_device(self.h)

    @property
    def device_bytes(self):
        return lib().eakv_cache_device_bytes(self.h)

    def compression_ratio(self):
        return lib().eakv_cache_compression_ratio(self.h)

    # --- quantize --------------------------------------------------------------
    def load_raw(self, data, seq_len):
        data = _f32(data)
        return lib().eakv_cache_load_raw(self.h, _ptr(data), seq_len)

    def append(self, data, layer, kv_idx, n_tokens):
        data = _f32(data)
        return lib().eakv_cache_append(self.h, _ptr(data), layer, kv_idx, n_tokens)

    def advance(self, n):
        return lib().eakv_cache_advance(self.h, n)

    def clear(self):
        lib().eakv_cache_clear(self.h)

    def checkpoint(self):
        return lib().eakv_checkpoint(self.h)

    def restore(self, seq_len):
        return lib().eakv_restore(self.h, seq_len)

    def save(self, path):
        return lib().eakv_cache_save(self.h, os.fsencode(path))

    # --- attention (host buffers, reference contract) -------------------------
    def scores(self, queries, layer, n_q, n_kv):
        q = _f32(queries)
        out = np.empty(n_q * self.seq_len, np.float32)
        lib().eakv_attention_scores(self.h, _ptr(q), layer, n_q, n_kv, _ptr(out))
        return out

    def output(self, weights, layer, n_q, n_kv):
        w = _f32(weights)
        out = np.empty(n_q * self.head_dim, np.float32)
        lib().eakv_attention_output(self.h, _ptr(w), layer, n_q, n_kv, _ptr(out))
        return out

    def fused(self, queries, layer, n_q, n_kv):
        q = _f32(queries)
        out = np.empty(n_q * self.head_dim, np.float32)
        _check(lib().eakv_attention_fused(self.h, _ptr(q), layer, n_q, n_kv, _ptr(out)),
               "eakv_attention_fused")
        return out

    # --- device entry points ------------------------------------------------------
    def scores_device(self, d_queries, layer, n_q, n_kv, d_scores):
        """eakv_attention_scores_device: f32[n_q][seq_len] scores on the device."""
        return _check(lib().eakv_attention_scores_device(self.h, _ptr(d_queries), layer, n_q, n_kv,
                                                         _ptr(d_scores)),
                      "eakv_attention_scores_device")

    def output_device(self, d_weights, layer, n_q, n_kv, d_output):
        """eakv_attention_output_device: f32[n_q][head_dim] outputs on the device."""
        return _check(lib().eakv_attention_output_device(self.h, _ptr(d_weights), layer, n_q, n_kv,
                                                         _ptr(d_output)),
                      "eakv_attention_output_device")

    def load_raw_device(self, d_data, seq_len):
        return lib().eakv_cache_load_raw_device(self.h, _ptr(d_data), seq_len)

    def append_device(self, d_data, layer, kv_idx, n_tokens):
        return lib().eakv_cache_append_device(self.h, _ptr(d_data), layer, kv_idx, n_tokens)

    def append_step_device(self, d_data, n_tokens):
        return lib().eakv_cache_append_step_device(self.h, _ptr(d_data), n_tokens)

    def set_stream(self, stream_handle):
        return _check(lib().eakv_cache_set_stream(self.h, stream_handle), "set_stream")

    def synchronize(self):
        return _check(lib().eakv_cache_synchronize(self.h), "synchronize")


def _handles(caches):
    arr = (ctypes.c_void_p * len(caches))(*[c.h for c in caches])
    return arr


def decode_attention(caches, d_queries, n_q_heads, d_output, stream=None):
    """Batched fused decode over device buffers (see eakv_cuda.h)."""
    arr = _handles(caches)
    return _check(lib().eakv_decode_attention(arr, len(caches), _ptr(d_queries), n_q_heads,
                                              _ptr(d_output), stream),
                  "eakv_decode_attention")


def decode_attention_noalloc(caches, d_queries, n_q_heads, d_output, stream=None):
    """eakv_decode_attention without any device allocation (fixed 4 MiB
    workspace in the library; see eakv_cuda.h). Returns the C return code."""
    arr = _handles(caches)
    return lib().eakv_decode_attention_noalloc(arr, len(caches), _ptr(d_queries), n_q_heads,
                                               _ptr(d_output), stream)


def decode_attention_host(caches, queries, n_q_heads, output, stream=None):
    arr = _handles(caches)
    return _check(lib().eakv_decode_attention_host(arr, len(caches), _ptr(queries), n_q_heads,
                                                   _ptr(output), stream),
                  "eakv_decode_attention_host")


def decode_attention_partial(caches, d_queries, n_q_heads, pos_begin, pos_end, d_output,
                             d_lse, stream=None):
    arr = _handles(caches)
    return _check(lib().eakv_decode_attention_partial(arr, len(caches), _ptr(d_queries),
                                                      n_q_heads, pos_begin, pos_end,
                                                      _ptr(d_output), _ptr(d_lse), stream),
                  "eakv_decode_attention_partial")


# --- several tokens per call ------------------------------------------------------
# Streams. Each call runs on `stream`, a CUDA stream's address; None (and 0) is the first
# cache's own stream, in copies and gathers the source's, which waits for no other stream and
# which torch's allocator does not know. So tensors that torch's current stream writes or
# frees are in order with a call only if it runs there:
# stream=torch.cuda.current_stream().cuda_stream or 1 (torch's default stream is 0, whose own
# address is 1), or cache.set_stream() with the same once. Otherwise the caller synchronizes, or orders
# the streams by events and keeps the tensors until the call has run.
EAKV_F32, EAKV_F16, EAKV_BF16 = 0, 1, 2
_DTYPES = {"float32": EAKV_F32, "float16": EAKV_F16, "bfloat16": EAKV_BF16}


class _Rows(ctypes.Structure):
    """eakv_rows_t"""
    _fields_ = [("data", _P), ("token_stride", _c.c_int64), ("head_stride", _c.c_int64), ("dtype", _I)]


# The same as bytes, and C arrays as array.array: a call's arguments take half the
# time of ctypes objects (append_rotary of 16 caches 16 -> 12 us).
_pack_rows = struct.Struct("@Qqqi4x").pack
_pack_rotary = struct.Struct("@QQiiiQqiiiii4x").pack


def _address(values):
    """Address of an array.array, which has to outlive the call."""
    return values.buffer_info()[0]


def _handle_array(caches):
    return array("Q", [c.h or 0 for c in caches])


class _Rotary(ctypes.Structure):
    """eakv_rotary_t"""
    _fields_ = [("cos_table", _P), ("sin_table", _P), ("n_rows", _I), ("rot_dim", _I),
                ("interleaved", _I), ("positions", _P), ("axis_stride", _c.c_int64), ("n_axes", _I),
                ("sections", _I * 4)]


_names = {}   # torch dtype -> its name, filled as types are met


def _name(x):
    name = _names.get(x.dtype)
    if name is None:
        name = _names[x.dtype] = str(x.dtype).replace("torch.", "")
    return name


_codes = {}   # torch dtype -> EAKV_*


def _dtype(x):
    code = _codes.get(x.dtype)
    if code is None:
        code = _DTYPES.get(_name(x))
        if code is None:
            raise TypeError(f"float32, float16 or bfloat16 expected, got {x.dtype}")
        _codes[x.dtype] = code
    return code


def _on(x, cache, what):
    """Refuses a tensor that is not on the cache's device."""
    if x.get_device() != cache.shape[3]:
        raise ValueError(f"{what} is on {x.device}, the cache on cuda:{cache.shape[3]}")
    return x


def _rows(x, cache, heads, tokens, what):
    """eakv_rows_t (its bytes) of a tensor [tokens, heads, head_dim] whose last dim is contiguous."""
    if x is None:
        return None
    _, _, head_dim, device = cache.shape
    if x.shape != (tokens, heads, head_dim):
        raise ValueError(f"{what}: shape {tuple(x.shape)}, expected {(tokens, heads, head_dim)}")
    t, h, d = x.stride()
    if d != 1:
        raise ValueError(f"{what}: the last dim must be contiguous")
    if x.get_device() != device:
        _on(x, cache, what)   # refuses
    return _pack_rows(x.data_ptr(), t, h, _dtype(x))


def _ints(values, n, what):
    if len(values) != n:
        raise ValueError(f"{what}: {len(values)} entries for {n} caches")
    return array("i", values)


def _contiguous(x, cache, dtype, shape, what):
    if _name(x) != dtype or not x.is_contiguous() or x.shape != shape:
        raise ValueError(f"{what}: a contiguous {dtype} tensor {shape} expected")
    return _on(x, cache, what)


def _index(index, cache):
    """An int32 position list [n], [heads, n] or [layers, heads, n] and its
    layer and head strides (0 where it is shared)."""
    if _name(index) != "int32" or index.dim() not in (1, 2, 3):
        raise ValueError("index: an int32 tensor [n], [heads, n] or [layers, heads, n] expected")
    if index.shape[-1] > 1 and index.stride(-1) != 1:
        raise ValueError("index: the last dim must be contiguous")
    dims, strides = (1, 1, *index.shape)[-3:], (0, 0, *index.stride())[-3:]
    if dims[0] not in (1, cache.shape[0]) or dims[1] not in (1, cache.shape[1]):
        raise ValueError(f"index: {tuple(index.shape)} for {cache.shape[0]} layers, {cache.shape[1]} heads")
    _on(index, cache, "index")
    return index, strides[0] if dims[0] > 1 else 0, strides[1] if dims[1] > 1 else 0


def append_rotary(caches, layer, counts, k, v, q=None, q_out=None, cos=None, sin=None,
                  positions=None, sections=None, interleaved=False, stream=None):
    """eakv_append_rotary. k, v: [total, n_kv_heads, head_dim] (any token and
    head stride), q and q_out: [total, n_q_heads, head_dim] (q_out defaults to
    q); counts[i] tokens of each cache, packed. cos, sin: f32 tables [rows,
    rot_dim/2]; positions: int32 [axes, total] (or [total]); sections: pairs
    that follow each axis. Without tables K goes in as it is. stream None is the
    first cache's own, which is not ordered with torch's current one (see above)."""
    c, counts = caches[0], list(counts)
    total, nkv = sum(counts), c.shape[1]
    if q is not None and q_out is None:
        q_out = q
    nq = q.shape[1] if q is not None else nkv
    rk, rv = _rows(k, c, nkv, total, "k"), _rows(v, c, nkv, total, "v")
    rq, ro = _rows(q, c, nq, total, "q"), _rows(q_out, c, nq, total, "q_out")
    rot = None
    if cos is None or sin is None or positions is None:
        if not cos is sin is positions is None:
            raise ValueError("cos, sin and positions go together")
    else:
        if positions.dim() == 1:
            positions = positions[None]
        if cos.dim() != 2 or cos.dtype != sin.dtype:
            raise ValueError("cos, sin: f32 tables [rows, rot_dim/2] expected")
        n_rows, pairs = shape = cos.shape
        _contiguous(cos, c, "float32", shape, "cos")
        _contiguous(sin, c, "float32", shape, "sin")
        axes, n = positions.shape if positions.dim() == 2 else (0, 0)
        if (_name(positions) != "int32" or not 1 <= axes <= 4 or n != total or
                (total > 1 and positions.stride(1) != 1)):
            raise ValueError(f"positions: int32 [1..4, {total}] expected")
        _on(positions, c, "positions")
        sections = list(sections) if sections is not None else [pairs]
        if len(sections) != axes:
            raise ValueError(f"{len(sections)} sections for {axes} axes")
        if not all(isinstance(s, int) and 0 <= s <= pairs for s in sections):
            raise ValueError(f"sections: integers in 0 .. {pairs} expected")
        rot = _pack_rotary(cos.data_ptr(), sin.data_ptr(), n_rows, 2 * pairs, 1 if interleaved else 0,
                           positions.data_ptr(), positions.stride(0) if axes > 1 else 0, axes, *sections,
                           *(0,) * (4 - axes))
    hs, n_new = _handle_array(caches), _ints(counts, len(caches), "counts")
    return _check(lib().eakv_append_rotary(_address(hs), len(caches), layer, _address(n_new), rk, rv, rq, ro,
                                           nq, rot, stream), "eakv_append_rotary")


def extend_workspace(caches, counts, dtype, n_q_heads, window=0, tree=False, depth=False):
    """Bytes of workspace eakv_extend_attention takes for this call; dtype is
    EAKV_F32, EAKV_F16 or EAKV_BF16; tree, depth: whether they are given."""
    out = ctypes.c_size_t()
    hs, n_new = _handle_array(caches), _ints(counts, len(caches), "counts")
    _check(lib().eakv_extend_workspace(_address(hs), len(caches), _address(n_new), dtype, n_q_heads, window,
                                       2 if depth else int(bool(tree)), ctypes.byref(out)),
           "eakv_extend_workspace")
    return out.value


def extend_attention(caches, layer, counts, q, out, window=0, tree=None, lse=None, scale=0.0,
                     workspace=None, stream=None, depth=None):
    """eakv_extend_attention. q, out: [total, n_q_heads, head_dim] (any token
    and head stride); tree: int64 or uint64 [total] bit masks over the cache's
    new tokens; lse: f32 [total, n_q_heads]; workspace: a uint8 tensor, zeroed
    once, or None for the first cache's scratch. depth: int32 [total], each tree
    token's number of ancestors, by which a window goes in place of slots
    (eakv_extend_attention_depths). stream None is the first cache's own, which is
    not ordered with torch's current one (see above)."""
    c, counts = caches[0], list(counts)
    total, nq = sum(counts), q.shape[1]
    rq, ro = _rows(q, c, nq, total, "q"), _rows(out, c, nq, total, "out")
    if tree is not None:
        kind = "uint64" if _name(tree) == "uint64" else "int64"
        _contiguous(tree, c, kind, (total,), "tree")
    if depth is not None:
        _contiguous(depth, c, "int32", (total,), "depth")
    if lse is not None:
        _contiguous(lse, c, "float32", (total, nq), "lse")
    size = 0
    if workspace is not None:
        size = workspace.numel()
        _contiguous(workspace, c, "uint8", (size,), "workspace")
    hs, n_new = _handle_array(caches), _ints(counts, len(caches), "counts")
    return _check(lib().eakv_extend_attention_depths(
        _address(hs), len(caches), layer, _address(n_new), rq, ro, nq, scale, window, _ptr(tree),
        _ptr(depth), _ptr(lse), _ptr(workspace), size, stream), "eakv_extend_attention")


def copy_positions(dsts, dst_pos, src, src_pos, n, stream=None):
    """eakv_cache_copy: positions [src_pos, src_pos + n) of src to dst_pos.. of
    every cache of dsts, whose seq_len becomes dst_pos + n. stream None is src's own;
    what runs on the destinations' streams is the caller's to order behind it."""
    hs = _handle_array(dsts)
    return _check(lib().eakv_cache_copy(_address(hs), len(dsts), dst_pos, src.h, src_pos, n, stream),
                  "eakv_cache_copy")


def gather_positions(dst, dst_pos, src, index, stream=None):
    """eakv_cache_gather: position dst_pos + j of dst becomes position
    index[..., j] of src. index: int32 [n], [heads, n] or [layers, heads, n]. stream
    None is src's own, which is not ordered with torch's current one (see above)."""
    index, ls, hs = _index(index, src)
    return _check(lib().eakv_cache_gather(dst.h, dst_pos, src.h, _ptr(index), ls, hs, index.shape[-1],
                                          stream), "eakv_cache_gather")


def read_positions(caches, begins, counts, out, layer=0, stream=None):
    """eakv_cache_read: the values of positions [begins[i], begins[i] +
    counts[i]) of each cache, into out [layers, 2, total, n_kv_heads, head_dim]
    (layers from `layer` on; K then V). stream None is the first cache's own, which
    is not ordered with torch's current one (see above)."""
    c, counts = caches[0], list(counts)
    total = sum(counts)
    if out.dim() != 5 or out.shape[1] != 2:
        raise ValueError("out: [layers, 2, total, n_kv_heads, head_dim] expected")
    if out.shape[0] == 0:
        raise ValueError("out: no layers")
    if out.shape[2:] != (total, c.shape[1], c.shape[2]):
        raise ValueError(f"out: {tuple(out.shape)}, expected [.., 2, {total}, {c.shape[1]}, {c.shape[2]}]")
    layers, kv, tok, head, last = out.stride()
    if last != 1:
        raise ValueError("out: the last dim must be contiguous")
    if kv < c.shape[2]:
        raise ValueError("out: K and V overlap")
    _on(out, c, "out")
    code, at = _dtype(out), out.data_ptr()
    hs, begin = _handle_array(caches), _ints(begins, len(caches), "begins")
    n = _ints(counts, len(caches), "counts")
    return _check(lib().eakv_cache_read(_address(hs), len(caches), layer, out.shape[0], _address(begin),
                                        _address(n), _pack_rows(at, tok, head, code),
                                        _pack_rows(at and at + kv * out.element_size(), tok, head, code),
                                        layers, stream), "eakv_cache_read")


def lse_combine(n_parts, n_rows, head_dim, d_parts, d_lse, d_output, d_lse_out=None,
                stream=None):
    return _check(lib().eakv_lse_combine(n_parts, n_rows, head_dim, _ptr(d_parts), _ptr(d_lse),
                                         _ptr(d_output), _ptr(d_lse_out), stream),
                  "eakv_lse_combine")


# --- sequence split over NCCL (include/eakv_nccl.h) -------------------------------
NCCL_ID_BYTES = 128


def nccl_version():
    """NCCL version code of the library's NCCL (< 0: unavailable)."""
    return lib().eakv_nccl_version()


def nccl_unique_id():
    """A new NCCL unique id (bytes) for eakv_nccl_comm_init."""
    buf = ctypes.create_string_buffer(NCCL_ID_BYTES)
    _check(lib().eakv_nccl_unique_id(buf), "eakv_nccl_unique_id")
    return buf.raw


class NcclComm:
    """A communicator of the library's NCCL (eakv_nccl_comm_init): n_ranks
    ranks, this one `rank`, on CUDA device `device`; blocks until every rank
    has joined."""

    def __init__(self, n_ranks, unique_id, rank, device):
        if len(unique_id) != NCCL_ID_BYTES:
            raise ValueError("bad NCCL unique id")
        h = ctypes.c_void_p()
        buf = ctypes.create_string_buffer(bytes(unique_id), NCCL_ID_BYTES)
        _check(lib().eakv_nccl_comm_init(ctypes.byref(h), n_ranks, buf, rank, device),
               "eakv_nccl_comm_init")
        self.h = h.value
        self.n_ranks, self.rank, self.device = n_ranks, rank, device

    def destroy(self):
        if self.h:
            _check(lib().eakv_nccl_comm_destroy(self.h), "eakv_nccl_comm_destroy")
            self.h = None

    def abort(self):
        if self.h:
            lib().eakv_nccl_comm_abort(self.h)
            self.h = None


def decode_attention_split(caches, d_queries, n_q_heads, d_output, comm, pos_begin=0,
                           pos_end=-1, stream=None):
    """eakv_decode_attention_split: this rank's slice of every sequence,
    merged with the other ranks' over `comm` (an NcclComm)."""
    arr = _handles(caches)
    return _check(lib().eakv_decode_attention_split(arr, len(caches), _ptr(d_queries), n_q_heads,
                                                    pos_begin, pos_end, _ptr(d_output), comm.h,
                                                    stream),
                  "eakv_decode_attention_split")


def decode_attention_split_host(caches, queries, n_q_heads, output, comm, stream=None):
    """eakv_decode_attention_split_host: host queries in, merged host output
    out, copies overlapped with the chunks' split steps."""
    arr = _handles(caches)
    return _check(lib().eakv_decode_attention_split_host(arr, len(caches), _ptr(queries),
                                                         n_q_heads, _ptr(output), comm.h, stream),
                  "eakv_decode_attention_split_host")


def decode_launches(caches, n_q_heads):
    return lib().eakv_decode_launches(_handles(caches), len(caches), n_q_heads)


def decode_splits(caches, n_q_heads):
    """Sequence splits per row the planner picks for these caches."""
    return lib().eakv_decode_splits(_handles(caches), len(caches), n_q_heads)


def set_device(device):
    """Selects the device for caches created later on this thread."""
    return _check(lib().eakv_set_device(int(device)), "eakv_set_device")


def device_status(device=0, reset=False):
    return lib().eakv_device_status(device, 1 if reset else 0)


def force_splits(n):
    lib().eakv_test_force_splits(int(n))


def choose_splits(items, max_pages, lo, hi, per_sm, sms):
    """The decode planner's split count for `items` rows of max_pages pages,
    searched in [lo, hi], with per_sm CTAs resident on each of `sms` SMs
    (host code only: runs without a GPU)."""
    return lib().eakv_test_choose_splits(int(items), int(max_pages), int(lo), int(hi),
                                         int(per_sm), int(sms))


def separate_merge(on):
    """Test aid: merge sequence splits in a second kernel (True) instead of
    inside the decode kernel (False, the default)."""
    lib().eakv_test_separate_merge(1 if on else 0)


def force_path(path):
    """Decode kernel of later calls on this thread: 1 the CUDA-core kernel, 2 the
    mma.sync tensor-core kernel, 3 the tcgen05 tensor-core kernel (head_dim
    128), 0 the automatic choice."""
    lib().eakv_test_force_path(int(path))


def extend_registers(n):
    """Registers per thread that extend_attention's tcgen05 kernel counts as built with
    (0: what it was built with); with another number than its own it is left out."""
    lib().eakv_test_extend_registers(int(n))


def test_stall(page, wait_budget=0):
    """Failure-detection aid: decode kernels never request `page` of a work
    item (page < 0: off) and give up each wait after `wait_budget` polls."""
    lib().eakv_test_stall(int(page), int(wait_budget))


# --- q4_1_eakv ggml block type on device buffers (include/eakv_ggml.h) ------------
def ggml_quantize_row_device(d_src, d_dst, k, stream=None):
    return _check(lib().eakv_ggml_quantize_row_device(_ptr(d_src), _ptr(d_dst), int(k),
                                                      stream), "ggml_quantize_row_device")


def ggml_dequantize_row_device(d_src, d_dst, k, stream=None):
    return _check(lib().eakv_ggml_dequantize_row_device(_ptr(d_src), _ptr(d_dst), int(k),
                                                        stream), "ggml_dequantize_row_device")


def ggml_vec_dot_device(n, d_s, bs, d_vx, bx, d_vy, by, nrc, stream=None):
    return _check(lib().eakv_ggml_vec_dot_device(int(n), _ptr(d_s), bs, _ptr(d_vx), bx,
                                                 _ptr(d_vy), by, int(nrc), stream),
                  "ggml_vec_dot_device")
