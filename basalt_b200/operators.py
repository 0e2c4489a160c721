"""The serving operators of libbasalt_cuda.so on torch tensors: a cache of keys and values held in
4 bits, bf16 or float32, attention over it, attention over packed prompts, and drawing tokens.

Tensors stay on the GPU: every call takes their device pointers, queues its kernels on ``stream`` (a
torch.cuda.Stream or a cudaStream_t as a number; torch's current stream of the tensors' device by
default) and returns without waiting. Outputs and
workspaces come from torch's allocator, for that stream of that device, unless given, so calls can be
captured into a CUDA graph (call once before the capture, which loads the kernels). ``include/basalt_cuda.h`` has
the operators' definitions; a rejected argument raises the exception of its status.

A batch is a list of sequences: ``lengths[s]`` counts the tokens of sequence s with this call's
included, ``starts`` ([count + 1], omitted when every sequence has one token) says where its tokens
begin in the packed tensors, ``rows`` its row of the cache (s when omitted). Index tensors are int32
on the device. Packed tokens that no sequence owns are neither read nor written: what they hold in a
new output is undefined, in a given one it stays.
"""
from __future__ import annotations

import ctypes

from . import _lib
from .text_engine import (BasaltShapeException, BasaltUnsupportedOperationException,
                          IllegalArgumentException, _raise)

_KEPT = 256   # workspace sizes that a cache keeps: batches come in ever new counts
_CODES = {}   # torch dtype -> BST_DTYPE_*, filled with the module below
_module = None
_raw_stream = None   # device index -> its current cudaStream_t


def _torch():
    global _module, _raw_stream
    if _module is None:
        import torch

        # The stream's pointer without a Stream object around it (0.1 instead of 2.2 us a call).
        _raw_stream = getattr(torch._C, "_cuda_getCurrentRawStream", None) or (
            lambda index: torch.cuda.current_stream(index).cuda_stream)
        _CODES.update({torch.float32: _lib.DTYPE_F32, torch.bfloat16: _lib.DTYPE_BF16})
        _module = torch
    return _module


def _dtype(name, t):
    if _module is None:
        _torch()
    code = _CODES.get(t.dtype)
    if code is None:
        raise BasaltUnsupportedOperationException(
            f"{name}: {t.dtype} is not float32 or bfloat16", _lib.BST_UNSUPPORTED)
    return code


def _on(device, name, t):
    if t.device != device or not t.is_cuda:
        raise IllegalArgumentException(f"{name} is on {t.device}, expected "
                                       f"{device if device.type == 'cuda' else 'a CUDA device'}",
                                       _lib.BST_INVALID)


def _index(device, name, t, size=None):
    """The pointer of an int32 index tensor, or None."""
    if t is None:
        return None
    if t.device != device:
        _on(device, name, t)
    if t.dtype is not _module.int32 or t.dim() != 1 or not t.is_contiguous():
        raise IllegalArgumentException(f"{name} must be a contiguous int32 vector",
                                       _lib.BST_INVALID)
    if size is not None and t.shape[0] != size:
        raise BasaltShapeException(f"{name} has {t.shape[0]} entries, expected {size}",
                                   _lib.BST_SHAPE)
    return t.data_ptr()


def _packed(device, name, t, heads=None, head_dim=None):
    """Checks a [tokens, heads, head_dim] tensor whose heads are contiguous; its token stride."""
    if t.device != device:
        _on(device, name, t)
    shape = t.shape
    if len(shape) != 3:
        raise BasaltShapeException(f"{name} must be [tokens, heads, head_dim], got "
                                   f"{tuple(shape)}", _lib.BST_SHAPE)
    n, h, d = shape
    if (heads is not None and h != heads) or (head_dim is not None and d != head_dim):
        raise BasaltShapeException(f"{name} is {tuple(shape)}, expected [tokens, {heads}, "
                                   f"{head_dim}]", _lib.BST_SHAPE)
    stride = t.stride()
    if (d > 1 and stride[2] != 1) or (h > 1 and stride[1] != d):
        raise IllegalArgumentException(f"{name}: the heads of a token must be contiguous",
                                       _lib.BST_INVALID)
    return stride[0] if n > 1 else max(stride[0], h * d)


def _empty(shape, dtype, device, stream):
    """A tensor whose memory is reused in the order of ``stream`` (None: the current one)."""
    if stream is None:
        return _module.empty(*shape, dtype=dtype, device=device)
    with _module.cuda.stream(_module.cuda.ExternalStream(stream, device)):
        return _module.empty(shape, dtype=dtype, device=device)


def _given(device, stream):
    """The pointer of a given stream (a torch.cuda.Stream of the device, or the pointer itself); None
    for none."""
    pointer = getattr(stream, "cuda_stream", stream)
    if pointer is not stream and stream.device != device:
        raise IllegalArgumentException(f"stream is on {stream.device}, expected {device}",
                                       _lib.BST_INVALID)
    return pointer


def _stream(device, stream):
    if stream is not None:
        return stream
    return _raw_stream(device.index)


class KvCache:
    """A cache of keys and values over the caller's device tensors.

    ``k`` and ``v``: [rows, kv_heads, slots, head_dim] float32 or bfloat16, or for a 4-bit cache
    [rows, kv_heads, slots, head_dim / 2] uint8 with ``k_scale`` and ``v_scale``
    [rows, kv_heads, slots, head_dim / 32, 2] bfloat16. All contiguous.
    """

    def __init__(self, k, v, k_scale=None, v_scale=None):
        _torch()
        self.k, self.v, self.k_scale, self.v_scale = k, v, k_scale, v_scale
        self.device = k.device
        self._sizes = {}  # workspace bytes by what they depend on
        u4 = str(k.dtype) == "torch.uint8"
        if u4 != (k_scale is not None) or u4 != (v_scale is not None):
            raise IllegalArgumentException("a 4-bit cache, and only that, has scales",
                                           _lib.BST_INVALID)
        if k.dim() != 4 or k.shape != v.shape or k.dtype != v.dtype:
            raise BasaltShapeException("k and v must be alike, [rows, kv_heads, slots, width]",
                                       _lib.BST_SHAPE)
        self.rows, self.kv_heads, self.slots, width = k.shape
        self.head_dim = 2 * width if u4 else width
        self.storage = _lib.DTYPE_U4 if u4 else _dtype("k", k)
        if u4:
            want = (self.rows, self.kv_heads, self.slots, self.head_dim // 32, 2)
            for name, t in (("k_scale", k_scale), ("v_scale", v_scale)):
                if tuple(t.shape) != want or str(t.dtype) != "torch.bfloat16":
                    raise BasaltShapeException(f"{name} must be bfloat16 {want}", _lib.BST_SHAPE)
        for name, t in (("k", k), ("v", v), ("k_scale", k_scale), ("v_scale", v_scale)):
            if t is not None:
                _on(self.device, name, t)
                if not t.is_contiguous():
                    raise IllegalArgumentException(f"{name} must be contiguous", _lib.BST_INVALID)
        s = _lib.KvCacheStruct()
        s.storage, s.rows, s.kv_heads = self.storage, self.rows, self.kv_heads
        s.slots, s.head_dim = self.slots, self.head_dim
        s.k, s.v = k.data_ptr(), v.data_ptr()
        s.k_scale = k_scale.data_ptr() if u4 else None
        s.v_scale = v_scale.data_ptr() if u4 else None
        self._struct = s
        self._ref = ctypes.byref(s)

    @staticmethod
    def allocate(rows: int, kv_heads: int, slots: int, head_dim: int, storage: str = "u4",
                 device="cuda") -> "KvCache":
        """A zeroed cache: ``storage`` is "u4", "bf16" or "f32"."""
        torch = _torch()
        if head_dim not in (32, 64, 128):
            raise BasaltUnsupportedOperationException(
                f"head dimension {head_dim} is not one of 32, 64, 128", _lib.BST_UNSUPPORTED)
        if storage == "u4":
            codes = [torch.zeros((rows, kv_heads, slots, head_dim // 2), dtype=torch.uint8,
                                 device=device) for _ in range(2)]
            scales = [torch.zeros((rows, kv_heads, slots, head_dim // 32, 2), dtype=torch.bfloat16,
                                  device=device) for _ in range(2)]
            return KvCache(*codes, *scales)
        if storage not in ("f32", "bf16"):
            raise IllegalArgumentException(f"unknown cache storage {storage!r}", _lib.BST_INVALID)
        dtype = torch.float32 if storage == "f32" else torch.bfloat16
        return KvCache(*[torch.zeros((rows, kv_heads, slots, head_dim), dtype=dtype, device=device)
                         for _ in range(2)])


def _sequences(device, tokens, lengths, starts, rows):
    """The batch's struct; the tensors it points to belong to the caller."""
    if lengths is not None:
        at = _index(device, "lengths", lengths)
        count = lengths.shape[0]
    else:
        if starts is None:
            raise IllegalArgumentException("starts must be given", _lib.BST_INVALID)
        at, count = None, starts.shape[0] - 1
        if count < 0:
            raise BasaltShapeException("starts must have one entry more than there are sequences",
                                       _lib.BST_SHAPE)
    return _lib.SequencesStruct(count, tokens, _index(device, "rows", rows, count),
                                _index(device, "starts", starts, count + 1), at)


def kv_append(cache: KvCache, k, v, lengths, starts=None, rows=None, stream=None):
    """Stores the batch's keys and values ([tokens, kv_heads, head_dim], float32 or bfloat16) in
    their slots of ``cache``."""
    device = cache.device
    stream = _given(device, stream)
    k_stride = _packed(device, "k", k, cache.kv_heads, cache.head_dim)
    v_stride = _packed(device, "v", v, cache.kv_heads, cache.head_dim)
    if k.dtype != v.dtype or k.shape[0] != v.shape[0]:
        raise BasaltShapeException("k and v must have the same type and tokens", _lib.BST_SHAPE)
    s = _sequences(device, k.shape[0], lengths, starts, rows)
    _raise(_lib.load().bst_kv_append(device.index, _stream(device, stream), cache._ref, s,
                                     k.data_ptr(), k_stride, v.data_ptr(), v_stride,
                                     _dtype("k", k)))


def kv_read(cache: KvCache, lengths, starts=None, rows=None, tokens=None, dtype=None, out=None,
            stream=None):
    """The values (k, v) that the batch's slots stand for, [tokens, kv_heads, head_dim]: ``tokens``
    is the packed count (the number of sequences without ``starts``), ``out`` a pair of tensors to
    fill; otherwise new ones of ``dtype`` (float32)."""
    device = cache.device
    stream = _given(device, stream)
    if out is None:
        if tokens is None:
            if starts is not None:
                raise IllegalArgumentException("kv_read needs tokens or out beside starts",
                                               _lib.BST_INVALID)
            tokens = lengths.shape[0]
        shape = (tokens, cache.kv_heads, cache.head_dim)
        dtype = dtype or _module.float32
        k = _empty(shape, dtype, device, stream)
        v = _empty(shape, dtype, device, stream)
        k_stride = v_stride = cache.kv_heads * cache.head_dim
    else:
        k, v = out
        k_stride = _packed(device, "k", k, cache.kv_heads, cache.head_dim)
        v_stride = _packed(device, "v", v, cache.kv_heads, cache.head_dim)
        tokens = k.shape[0]
        if k.dtype != v.dtype or tokens != v.shape[0]:
            raise BasaltShapeException("k and v must have the same type and tokens",
                                       _lib.BST_SHAPE)
    s = _sequences(device, tokens, lengths, starts, rows)
    _raise(_lib.load().bst_kv_read(device.index, _stream(device, stream), cache._ref, s,
                                   k.data_ptr(), k_stride, v.data_ptr(), v_stride,
                                   _dtype("k", k)))
    return k, v


def _spec(q, kv_heads, window, sinks, scale):
    _, heads, dim = q.shape
    return _lib.AttentionSpecStruct(heads, kv_heads, dim, _dtype("q", q),
                                    _lib.int32(window), _lib.int32(sinks),
                                    dim ** -0.5 if scale is None and dim else scale or 0.0, 0)


def _out(device, q, out, stream):
    if out is None:
        if stream is None:
            out = _module.empty_like(q, memory_format=_module.contiguous_format)
        else:
            out = _empty(q.shape, q.dtype, device, stream)
        return out, q.shape[1] * q.shape[2]
    if out.dtype != q.dtype or out.shape != q.shape:
        raise BasaltShapeException("out must be like q", _lib.BST_SHAPE)
    return out, _packed(device, "out", out)


def _workspace(device, size, workspace, stream):
    """(pointer, bytes, tensor) of a workspace of at least ``size`` bytes."""
    if workspace is None:
        if size == 0:
            return None, 0, None
        workspace = _empty((size,), _module.uint8, device, stream)
        return workspace.data_ptr(), size, workspace
    _on(device, "workspace", workspace)
    if not workspace.is_contiguous():
        raise IllegalArgumentException("workspace must be contiguous", _lib.BST_INVALID)
    return workspace.data_ptr(), workspace.numel() * workspace.element_size(), workspace


def attention_cached(cache: KvCache, q, lengths, starts=None, rows=None, window: int = 0,
                     sinks: int = 0, scale=None, out=None, workspace=None, stream=None):
    """Attention of q ([tokens, heads, head_dim]) over the sequences' rows of ``cache``, whose
    current tokens were appended before. ``window`` and ``sinks``: a query sees the last ``window``
    keys (0: all) and the first ``sinks``. ``scale`` is 1 / sqrt(head_dim) by default. ``out`` may be
    ``q`` itself."""
    device = cache.device
    stream = _given(device, stream)
    q_stride = _packed(device, "q", q, None, cache.head_dim)
    out, out_stride = _out(device, q, out, stream)
    s = _sequences(device, q.shape[0], lengths, starts, rows)
    a = _spec(q, cache.kv_heads, window, sinks, scale)
    lib = _lib.load()
    key = (s.count, s.tokens, starts is None, a.heads, a.dtype, window, sinks)
    needed = cache._sizes.get(key)
    if needed is None:
        size = ctypes.c_int64(0)
        _raise(lib.bst_attention_cached_workspace(cache._ref, s, a, size))
        if len(cache._sizes) >= _KEPT:
            cache._sizes.clear()
        needed = cache._sizes[key] = size.value
    pointer, room, workspace = _workspace(device, needed, workspace, stream)
    _raise(lib.bst_attention_cached(device.index, _stream(device, stream), cache._ref, s, a,
                                    q.data_ptr(), q_stride, out.data_ptr(), out_stride, pointer,
                                    room))
    return out


def attention_packed(q, k, v, starts, window: int = 0, sinks: int = 0, scale=None, out=None,
                     workspace=None, stream=None):
    """Causal attention of packed sequences over their own keys and values: q [tokens, heads,
    head_dim], k and v [tokens, kv_heads, head_dim], all of one type. ``out`` must not overlap them."""
    _torch()
    device = q.device
    stream = _given(device, stream)
    _on(device, "q", q)
    q_stride = _packed(device, "q", q)
    k_stride = _packed(device, "k", k, None, q.shape[2])
    v_stride = _packed(device, "v", v, k.shape[1], q.shape[2])
    if not q.dtype == k.dtype == v.dtype or not q.shape[0] == k.shape[0] == v.shape[0]:
        raise BasaltShapeException("q, k and v must have the same type and tokens", _lib.BST_SHAPE)
    out, out_stride = _out(device, q, out, stream)
    s = _sequences(device, q.shape[0], None, starts, None)
    a = _spec(q, k.shape[1], window, sinks, scale)
    lib = _lib.load()
    size = ctypes.c_int64(0)
    _raise(lib.bst_attention_packed_workspace(s, a, size))
    pointer, room, workspace = _workspace(device, size.value, workspace, stream)
    _raise(lib.bst_attention_packed(device.index, _stream(device, stream), s, a, q.data_ptr(),
                                    q_stride, k.data_ptr(), k_stride, v.data_ptr(), v_stride,
                                    out.data_ptr(), out_stride, pointer, room))
    return out


def _setting(device, rows, name, value, dtype):
    """(scalar, pointer) of a sampling setting given as a number or as one value per row."""
    if not hasattr(value, "data_ptr"):
        return (_lib.int32(int(value)) if dtype == "torch.int32" else float(value)), None
    _on(device, name, value)
    if str(value.dtype) != dtype or tuple(value.shape) != (rows,) or not value.is_contiguous():
        raise IllegalArgumentException(f"{name} must be a number or a contiguous {dtype} vector "
                                       f"of {rows}", _lib.BST_INVALID)
    return 0, value.data_ptr()


def sample_tokens(logits, uniforms, temperature=1.0, top_k=0, top_p=1.0, min_p=0.0, out=None,
                  stream=None):
    """int32 tokens drawn from logits [rows, vocabulary] (float32 or bfloat16) with ``uniforms``
    (float64, one in [0, 1) per row). Each setting is a number or one value per row (float32, top_k
    int32, on the device). Rows with nothing to draw give -1."""
    _torch()
    device = logits.device
    stream = _given(device, stream)
    if logits.dim() != 2 or (logits.shape[1] > 1 and logits.stride(1) != 1):
        raise BasaltShapeException("logits must be [rows, vocabulary] with contiguous rows",
                                   _lib.BST_SHAPE)
    _on(device, "logits", logits)
    rows, vocabulary = logits.shape
    _on(device, "uniforms", uniforms)
    if uniforms.dtype is not _module.float64 or tuple(uniforms.shape) != (rows,) or \
            not uniforms.is_contiguous():
        raise IllegalArgumentException(f"uniforms must be a contiguous float64 vector of {rows}",
                                       _lib.BST_INVALID)
    if out is None:
        out = _empty((rows,), _module.int32, device, stream)
    else:
        _index(device, "out", out, rows)
    p = _lib.SamplingStruct()
    p.temperature, p.temperatures = _setting(device, rows, "temperature", temperature,
                                             "torch.float32")
    p.top_k, p.top_ks = _setting(device, rows, "top_k", top_k, "torch.int32")
    p.top_p, p.top_ps = _setting(device, rows, "top_p", top_p, "torch.float32")
    p.min_p, p.min_ps = _setting(device, rows, "min_p", min_p, "torch.float32")
    _raise(_lib.load().bst_sample_tokens(
        device.index, _stream(device, stream), logits.data_ptr(), _dtype("logits", logits), rows,
        vocabulary, logits.stride(0) if rows > 1 else max(vocabulary, logits.stride(0)), p,
        uniforms.data_ptr(), out.data_ptr()))
    return out
