"""Refusals of origami_shared_prefix_attention and its workspace query: the host-side checks come
before any CUDA call."""
import ctypes

import pytest
import torch

from origami_b200 import _lib
from origami_b200.shared_prefix import shared_prefix_attention

FAKE = 1 << 12  # never dereferenced: validation fails first
F16, BF16, F32 = _lib.ORIGAMI_DTYPE_F16, _lib.ORIGAMI_DTYPE_BF16, _lib.ORIGAMI_DTYPE_F32


def rows(dtype=BF16, heads=8, token=None, head=64, data=FAKE):
    return _lib.HeadRows(data, dtype, heads, heads * 64 if token is None else token, head)


def ref(x):
    return None if x is None else ctypes.byref(x)


def call(cache=None, **change):
    L = _lib.lib()
    a = dict(q=rows(), o=rows(data=FAKE * 4), lse=None, tokens=3, head_dim=64, cache_dtype=BF16, prefix_blocks=FAKE,
             num_prefix=4, prefix=64, suffix_blocks=FAKE, stride=2, width=2, lens=FAKE, start=FAKE, requests=2,
             scale=0.125, ws=FAKE, ws_bytes=1 << 40)
    a.update(change)
    c = dict(d_data=FAKE, layout=0, elem_bytes=2, num_blocks=16, block_size=16, num_heads=2, head_dim=64)
    c.update(cache or {})
    kv = _lib.PagedKV(*[c[f] for f, _ in _lib.PagedKV._fields_])
    rc = L.origami_shared_prefix_attention(
        ref(a["q"]), ref(a["o"]), a["lse"], a["tokens"], a["head_dim"], ctypes.byref(kv), a["cache_dtype"],
        a["prefix_blocks"], a["num_prefix"], a["prefix"], a["suffix_blocks"], a["stride"], a["width"], a["lens"],
        a["start"], a["requests"], a["scale"], a["ws"], a["ws_bytes"], None, None)
    return rc, L.origami_last_error().decode()


@pytest.mark.parametrize("change, message", [
    (dict(cache=dict(d_data=None)), "kv cache is null"),
    (dict(cache=dict(layout=5)), "unknown kv cache layout"),
    (dict(cache=dict(d_data=FAKE + 8)), "16-byte aligned"),
    (dict(cache=dict(head_dim=128)), "does not match query"),
    (dict(cache=dict(num_heads=3)), "divisible"),
    (dict(cache=dict(num_blocks=1 << 30)), "too many token rows"),
    (dict(q=None), "both needed"),
    (dict(o=None), "both needed"),
    (dict(q=rows(dtype=F32)), "query must be float16 or bfloat16"),
    (dict(q=rows(data=FAKE + 1)), "2-byte aligned"),
    (dict(q=rows(token=-1)), "negative stride"),
    (dict(q=rows(heads=512)), "query heads per KV head"),
    (dict(o=rows(token=64)), "output has rows that overlap"),
    (dict(o=rows(dtype=F16)), "output dtype"),
    (dict(o=rows(heads=4)), "heads of query"),
    (dict(cache_dtype=F16), "kv_cache dtype"),
    (dict(head_dim=96), "head_dim 64 and 128"),
    (dict(tokens=-1), "must be positive"),
    (dict(tokens=1 << 25), "too many query rows"),
    (dict(requests=0), "at least one request"),
    (dict(prefix=-1), "not be negative"),
    (dict(width=-1), "not be negative"),
    (dict(prefix=65), "too short for prefix_tokens"),
    (dict(scale=0.0), "finite and positive"),
    (dict(scale=-1.0), "finite and positive"),
    (dict(scale=float("inf")), "finite and positive"),
    (dict(scale=float("nan")), "finite and positive"),
    (dict(start=None), "query_start and suffix_lens"),
    (dict(lens=FAKE + 2), "query_start and suffix_lens"),
    (dict(prefix_blocks=None), "prefix_blocks must be"),
    (dict(suffix_blocks=None), "suffix_blocks must be"),
    (dict(stride=-1), "negative stride"),
    (dict(lse=FAKE + 2), "lse must be"),
    (dict(tokens=1 << 24, width=1 << 24, requests=1 << 20), "too many tiles"),
])
def test_refusals(change, message):
    rc, msg = call(**change)
    assert rc in (-1, -2)
    assert message in msg


@pytest.mark.parametrize("scale", [1e-300, 1e-46, 1e-39, 2.4e38, 1e300])
def test_scales_that_32_bits_do_not_hold(scale):
    """The kernel takes scale * log2(e) in 32 bits: neither zero, nor without all its digits, nor infinite."""
    rc, msg = call(scale=scale)
    assert rc == -1
    assert "32 bits" in msg


def test_no_tokens_is_no_launch():
    assert call(tokens=0)[0] == 0


@pytest.mark.parametrize("args, message", [
    ((1, 8, 3, 64, 1), "divisible"), ((1, 8, 2, 80, 1), "head_dim 64 and 128"), ((-1, 8, 2, 64, 1), "must be positive"),
    ((1, 8, 2, 64, 0), "at least one request"), ((1, 0, 2, 64, 1), "must be positive"),
    ((1, 8, 0, 64, 1), "divisible"),
])
def test_workspace_refusals(args, message):
    L = _lib.lib()
    out = ctypes.c_int64(0)
    assert L.origami_shared_prefix_attention_workspace(*args, ctypes.byref(out)) in (-1, -2)
    assert message in L.origami_last_error().decode()
    assert L.origami_shared_prefix_attention_workspace(1, 8, 2, 64, 1, None) == -1


def test_host_tensors_are_refused():
    q = torch.zeros(2, 4, 64, dtype=torch.bfloat16)
    i = torch.zeros(3, dtype=torch.int32)
    with pytest.raises(ValueError, match="CUDA tensor"):
        shared_prefix_attention(q, torch.zeros(2, 4, 16, 4, 64, dtype=torch.bfloat16), i, i, 8, i[None], i)
