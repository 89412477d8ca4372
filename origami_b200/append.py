"""The new tokens of a step on their way to the paged cache (kernels: csrc/append_kernels.cuh).

norm_rope : RMS norm of queries and keys for each head and the position rotation, one pass.
append_kv : keys and values of new tokens written into one layer's paged cache at their slots
            (slot = block id * block_size + offset, as vLLM's slot_mapping; -1 = no row), the
            keys normed and rotated on the way and, when given, the queries in the same launch.

A row is one head of one token. With a weight, y = x * w / sqrt(mean(x^2) + eps); then pair i
of the first R dims, (i, i + R/2) or (2i, 2i + 1) when interleaved, turns by the angle whose
cosine and sine are cos_sin[position, i] and cos_sin[position, R/2 + i] (R = the table's
width). Arithmetic is fp32 with one rounding at the store. Ops enqueue on the given (or
current) stream of the tensors' device and never synchronise; ``error_count`` (an int32 CUDA
tensor, optional) grows by one for every row that a position outside the table or a slot
outside the cache left unwritten. An output that the call allocates belongs to the stream it
runs on and is not filled beforehand: where a position outside the table leaves its rows
unwritten they hold whatever the memory held, so a caller that cannot rule such positions out
passes ``error_count`` (or an output of its own). No gradients are recorded: the results never
require one, whatever the inputs do. The reference connector leaves these steps to the engine.
"""
from __future__ import annotations

import ctypes

import torch

from origami_b200 import _lib
from origami_b200.layer import paged_desc

_DTYPE = {torch.float16: _lib.ORIGAMI_DTYPE_F16, torch.bfloat16: _lib.ORIGAMI_DTYPE_BF16,
          torch.float32: _lib.ORIGAMI_DTYPE_F32}


def _device_index(t: torch.Tensor, name: str) -> int:
    index = t.get_device()
    if index < 0:
        raise ValueError(f"{name} must be a CUDA tensor")
    return index


def _on(index: int, t: torch.Tensor, name: str) -> None:
    if t.get_device() != index:
        raise ValueError(f"{name} must be a CUDA tensor on the device of the others")


def _rows(t: torch.Tensor, name: str, tokens: int, head_dim: int, index: int) -> _lib.HeadRows:
    _on(index, t, name)
    shape = t.shape
    if len(shape) != 3 or shape[0] != tokens or shape[2] != head_dim:
        raise ValueError(f"{name} must have shape [{tokens}, heads, {head_dim}], got {tuple(shape)}")
    dtype = _DTYPE.get(t.dtype)
    if dtype is None:
        raise ValueError(f"{name} must be float16, bfloat16 or float32")
    token_stride, head_stride, stride = t.stride()
    if stride != 1 and head_dim > 1:
        raise ValueError(f"{name} must be contiguous in its last dimension")
    return _lib.HeadRows(t.data_ptr(), dtype, shape[1], token_stride, head_stride)


def _index(t: torch.Tensor, name: str, tokens: int, index: int) -> int:
    """Bytes per element of a contiguous int32 / int64 vector of one entry per token."""
    _on(index, t, name)
    if t.dtype is not torch.int32 and t.dtype is not torch.int64:
        raise ValueError(f"{name} must be int32 or int64")
    if t.dim() != 1 or t.shape[0] != tokens or not t.is_contiguous():
        raise ValueError(f"{name} must be a contiguous vector of {tokens} entries, one per token")
    return t.element_size()


def _rotation(positions: torch.Tensor | None, cos_sin: torch.Tensor | None, interleaved: bool, tokens: int, index: int):
    if positions is None and cos_sin is None:
        return None
    if positions is None or cos_sin is None:
        raise ValueError("positions and cos_sin go together")
    width = _index(positions, "positions", tokens, index)
    _on(index, cos_sin, "cos_sin")
    dtype = _DTYPE.get(cos_sin.dtype)
    if cos_sin.dim() != 2 or dtype is None:
        raise ValueError("cos_sin must be a float16, bfloat16 or float32 matrix [max_positions, rotated dims]")
    rows, dims = cos_sin.shape
    row_stride, stride = cos_sin.stride()
    if dims > 1 and stride != 1:
        raise ValueError("cos_sin must be contiguous in its last dimension")
    # a table of one row has no row stride to speak of
    return _lib.Rotation(cos_sin.data_ptr(), dtype, 1 if interleaved else 0, rows, dims, row_stride if rows > 1 else dims,
                         positions.data_ptr(), width)


def _weight(w: torch.Tensor | None, name: str, head_dim: int, index: int) -> tuple[int | None, int]:
    if w is None:
        return None, 0
    _on(index, w, name)
    dtype = _DTYPE.get(w.dtype)
    if dtype is None or w.dim() != 1 or w.shape[0] != head_dim or not w.is_contiguous():
        raise ValueError(f"{name} must be a contiguous float16, bfloat16 or float32 vector of {head_dim} elements")
    return w.data_ptr(), dtype


def _norm(query_weight: torch.Tensor | None, key_weight: torch.Tensor | None, eps: float, head_dim: int, index: int):
    if query_weight is None and key_weight is None:
        return None
    q, q_dtype = _weight(query_weight, "query_weight", head_dim, index)
    k, k_dtype = _weight(key_weight, "key_weight", head_dim, index)
    return _lib.HeadNorm(q, k, q_dtype, k_dtype, eps)


def _error(error_count: torch.Tensor | None, index: int):
    if error_count is None:
        return None
    _on(index, error_count, "error_count")
    if error_count.dtype not in (torch.int32, torch.uint32) or error_count.numel() < 1:
        raise ValueError("error_count must be an int32 tensor of one element")
    return error_count.data_ptr()


def _empty_like(t: torch.Tensor, stream: torch.cuda.Stream | None) -> torch.Tensor:
    """A dense tensor of t's shape and type, from the pool of the stream that will write it."""
    if stream is None:
        return torch.empty_like(t)
    with torch.cuda.stream(stream):
        return torch.empty_like(t)


def _launch(index: int, stream: torch.cuda.Stream | None, what: str, entry, *args) -> None:
    """Calls a library entry point on the tensors' device with the stream's handle last."""
    if stream is not None and stream.device_index != index:
        raise ValueError("stream must be a stream of the tensors' device")
    handle = torch._C._cuda_getCurrentRawStream(index) if stream is None else stream.cuda_stream
    if torch._C._cuda_getDevice() == index:
        rc = entry(*args, handle)
    else:
        with torch.cuda.device(index):
            rc = entry(*args, handle)
    _lib.check(rc, what)


def _ref(struct):
    return ctypes.byref(struct) if struct is not None else None


def norm_rope(query: torch.Tensor, key: torch.Tensor, positions: torch.Tensor, cos_sin: torch.Tensor, *,
              query_weight: torch.Tensor | None = None, key_weight: torch.Tensor | None = None, eps: float = 1e-6,
              interleaved: bool = False, query_out: torch.Tensor | None = None, key_out: torch.Tensor | None = None,
              stream: torch.cuda.Stream | None = None,
              error_count: torch.Tensor | None = None) -> tuple[torch.Tensor, torch.Tensor]:
    """Norm (where a weight is given) and rotate query [T, Hq, D] and key [T, Hk, D].

    query and key may be strided slices of one projection's output; query_out / key_out may
    be query / key themselves (in place). Returns (query_out, key_out)."""
    index = _device_index(query, "query")
    if query.dim() != 3:
        raise ValueError(f"query must have shape [tokens, heads, head_dim], got {tuple(query.shape)}")
    tokens, _, head_dim = query.shape
    q = _rows(query, "query", tokens, head_dim, index)
    k = _rows(key, "key", tokens, head_dim, index)
    if positions is None or cos_sin is None:
        raise ValueError("norm_rope needs positions and cos_sin")
    rot = _rotation(positions, cos_sin, interleaved, tokens, index)
    norm = _norm(query_weight, key_weight, eps, head_dim, index)
    err = _error(error_count, index)
    if query_out is None:
        query_out = _empty_like(query, stream)
    if key_out is None:
        key_out = _empty_like(key, stream)
    qo = _rows(query_out, "query_out", tokens, head_dim, index)
    ko = _rows(key_out, "key_out", tokens, head_dim, index)
    if tokens > 0:
        _launch(index, stream, "origami_norm_rope", _lib.lib().origami_norm_rope, ctypes.byref(q), ctypes.byref(qo),
                ctypes.byref(k), ctypes.byref(ko), tokens, head_dim, _ref(rot), _ref(norm), err)
    return query_out, key_out


def append_kv(kv_layer: torch.Tensor, key: torch.Tensor, value: torch.Tensor, slots: torch.Tensor, *,
              query: torch.Tensor | None = None, positions: torch.Tensor | None = None,
              cos_sin: torch.Tensor | None = None, query_weight: torch.Tensor | None = None,
              key_weight: torch.Tensor | None = None, eps: float = 1e-6, interleaved: bool = False,
              query_out: torch.Tensor | None = None, stream: torch.cuda.Stream | None = None,
              error_count: torch.Tensor | None = None) -> torch.Tensor | None:
    """Write key / value [T, Hk, D] of new tokens into the cache rows `slots` names, the keys
    normed and rotated; returns the normed and rotated query (None without one).

    kv_layer is a paged cache layer in either layout of `layer.cache_layout`, bf16 or fp16;
    key, value and query share a type (bf16, fp16 or fp32). A token with slot -1 gets no
    cache row; its query is still written. Slots must differ from one another. query_out may
    be query itself; no other input may share memory with an output or the cache."""
    index = _device_index(kv_layer, "the paged KV cache")
    desc = paged_desc(kv_layer)
    cache_dtype = _DTYPE.get(kv_layer.dtype)
    if cache_dtype is None:
        raise ValueError("the paged KV cache must be float16 or bfloat16")
    tokens, head_dim = key.shape[0], desc.head_dim
    k = _rows(key, "key", tokens, head_dim, index)
    v = _rows(value, "value", tokens, head_dim, index)
    width = _index(slots, "slots", tokens, index)
    rot = _rotation(positions, cos_sin, interleaved, tokens, index)
    norm = _norm(query_weight, key_weight, eps, head_dim, index)
    err = _error(error_count, index)
    q = qo = None
    if query is not None:
        q = _rows(query, "query", tokens, head_dim, index)
        if query_out is None:
            query_out = _empty_like(query, stream)
        qo = _rows(query_out, "query_out", tokens, head_dim, index)
    elif query_out is not None or query_weight is not None:
        raise ValueError("query_out and query_weight need a query")
    if tokens > 0:
        _launch(index, stream, "origami_append_kv", _lib.lib().origami_append_kv, ctypes.byref(k), ctypes.byref(v), _ref(q),
                _ref(qo), ctypes.byref(desc), cache_dtype, slots.data_ptr(), width, tokens, _ref(rot), _ref(norm), err)
    return query_out
