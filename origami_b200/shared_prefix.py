"""Attention of a ragged batch over a paged prefix that all its requests share and each
request's own paged suffix (kernels: csrc/shared_prefix_kernels.cuh, tcgen05 tensor cores).

``shared_prefix_attention`` takes the new tokens of a step: query token j of request b (of n)
attends to all ``prefix_tokens`` keys of the shared prefix and to the first
``suffix_lens[b] - n + j + 1`` keys of the request's suffix, which holds its new tokens
already (`append.append_kv` writes them). The prefix's keys and values are read once for all
requests, as one problem per KV head, instead of once per request; the blocks can be ones
that `layer.restore_layer` filled. Scores and sums are fp32; the probabilities are rounded to
the type of the values for the tensor cores. The lists stay on the device, so a captured call
replays with other suffix lengths, tables and divisions of the tokens among requests;
``prefix_tokens``, ``softmax_scale`` and all shapes are the host's and stay as captured: another
prefix length needs another capture. The op enqueues on the given (or current) stream of the
query's device and never synchronises. No gradients are recorded. The reference's attention
takes one request a call.
"""
from __future__ import annotations

import ctypes
from contextlib import nullcontext

import torch

from origami_b200 import _lib
from origami_b200.append import _DTYPE, _device_index, _empty_like, _error, _launch, _on, _rows
from origami_b200.layer import paged_desc


def workspace_bytes(tokens: int, query_heads: int, kv_heads: int, head_dim: int, requests: int,
                    device: torch.device | int | None = None) -> int:
    """Workspace the kernels need for these shapes on `device`."""
    entry, out = _lib.lib().origami_shared_prefix_attention_workspace, ctypes.c_int64(0)
    args = (tokens, query_heads, kv_heads, head_dim, requests, ctypes.byref(out))
    if device is None or device == torch.cuda.current_device():
        rc = entry(*args)
    else:
        with torch.cuda.device(device):
            rc = entry(*args)
    _lib.check(rc, "origami_shared_prefix_attention_workspace")
    return out.value


def _ints(t: torch.Tensor, name: str, dims: int, index: int) -> None:
    _on(index, t, name)
    if t.dtype is not torch.int32 or t.dim() != dims:
        raise ValueError(f"{name} must be an int32 tensor of {dims} dimension{'s' if dims > 1 else ''}")
    if t.shape[-1] > 1 and t.stride(-1) != 1:
        raise ValueError(f"{name} must be contiguous in its last dimension")


def shared_prefix_attention(query: torch.Tensor, kv_layer: torch.Tensor, query_start: torch.Tensor,
                            prefix_blocks: torch.Tensor, prefix_tokens: int, suffix_blocks: torch.Tensor,
                            suffix_lens: torch.Tensor, *, softmax_scale: float | None = None,
                            out: torch.Tensor | None = None, lse: torch.Tensor | None = None,
                            workspace: torch.Tensor | None = None, stream: torch.cuda.Stream | None = None,
                            error_flags: torch.Tensor | None = None) -> torch.Tensor:
    """Attention of query [T, Hq, D] over one layer's paged cache; returns out (allocated when
    omitted, on the stream the call runs on).

    query_start [B + 1]: request b's tokens are query_start[b] .. query_start[b + 1] - 1, one
    request after the other; tokens before the first and behind the last are left as they are
    in out and lse. prefix_blocks: the prefix's block ids; suffix_blocks [B, W]: each
    request's block ids behind the prefix (rows may be a slice of wider tables); suffix_lens
    [B]: each request's keys behind the prefix, its new tokens included (0: the prefix
    alone). All int32 on the device. query, out and kv_layer share a type (bf16 or fp16) and
    D is 64 or 128; softmax_scale defaults to D ** -0.5. lse [T, Hq] float32, optional,
    receives each row's log of the sum of exponentials. A row without keys gives zeros and
    -inf; a block id outside the cache reads as zero keys and values that still take part. A
    value that a row does not see but a later row of its request does meets it with weight
    zero: if it is infinite or NaN, so becomes the row.

    workspace: a uint8 tensor of workspace_bytes(...) bytes, allocated per call when omitted;
    calls that share one must not overlap; it grows with 8 bytes x tokens x query heads x D (537 MB
    for 16384 tokens of 32 heads of 128). error_flags (int32): bit 31 is set if a bounded wait
    inside the kernel ran out (out and lse are void then), bit 30 if query_start decreases (nothing
    is written then). An out that the call allocates is not filled beforehand: what the call
    leaves, as said above, holds whatever the memory held."""
    index = _device_index(query, "query")
    if query.dim() != 3:
        raise ValueError(f"query must have shape [tokens, heads, head_dim], got {tuple(query.shape)}")
    tokens, heads, head_dim = query.shape
    q = _rows(query, "query", tokens, head_dim, index)
    _on(index, kv_layer, "the paged KV cache")
    desc = paged_desc(kv_layer)
    cache_dtype = _DTYPE.get(kv_layer.dtype)
    if cache_dtype is None:
        raise ValueError("the paged KV cache must be float16 or bfloat16")
    _ints(query_start, "query_start", 1, index)
    _ints(prefix_blocks, "prefix_blocks", 1, index)
    _ints(suffix_blocks, "suffix_blocks", 2, index)
    _ints(suffix_lens, "suffix_lens", 1, index)
    requests, width = suffix_blocks.shape
    if suffix_lens.shape[0] != requests or query_start.shape[0] != requests + 1:
        raise ValueError("suffix_lens needs one entry and query_start one more than suffix_blocks has rows")
    if lse is not None:
        _on(index, lse, "lse")
        if lse.dtype is not torch.float32 or tuple(lse.shape) != (tokens, heads) or not lse.is_contiguous():
            raise ValueError(f"lse must be a contiguous float32 tensor of shape [{tokens}, {heads}]")
    err = _error(error_flags, index)
    scale = head_dim ** -0.5 if softmax_scale is None else float(softmax_scale)
    if out is None:
        out = _empty_like(query, stream)
    o = _rows(out, "out", tokens, head_dim, index)
    if workspace is None:
        need = workspace_bytes(tokens, heads, desc.num_heads, head_dim, requests, index)
        with torch.cuda.stream(stream) if stream is not None else nullcontext():
            workspace = query.new_empty((need,), dtype=torch.uint8)
    _on(index, workspace, "workspace")
    if workspace.dtype is not torch.uint8 or not workspace.is_contiguous():
        raise ValueError("workspace must be a contiguous uint8 tensor")
    _launch(index, stream, "origami_shared_prefix_attention", _lib.lib().origami_shared_prefix_attention, ctypes.byref(q),
            ctypes.byref(o), lse.data_ptr() if lse is not None else None, tokens, head_dim, ctypes.byref(desc), cache_dtype,
            prefix_blocks.data_ptr(), prefix_blocks.shape[0], int(prefix_tokens), suffix_blocks.data_ptr(),
            suffix_blocks.stride(0), width, suffix_lens.data_ptr(), query_start.data_ptr(), requests, scale,
            workspace.data_ptr(), workspace.numel(), err)
    return out
