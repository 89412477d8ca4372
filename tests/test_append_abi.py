"""Refusals of origami_norm_rope / origami_append_kv: the library's host-side checks come before
any CUDA call, and the Python front end's before the library."""
import ctypes

import pytest
import torch

from origami_b200 import _lib
from origami_b200.append import append_kv, norm_rope

FAKE = 1 << 12  # never dereferenced: validation fails first
F16, BF16, F32 = _lib.ORIGAMI_DTYPE_F16, _lib.ORIGAMI_DTYPE_BF16, _lib.ORIGAMI_DTYPE_F32
D = 64


def rows(dtype=BF16, heads=4, token=None, head=D, data=FAKE):
    return _lib.HeadRows(data, dtype, heads, heads * D if token is None else token, head)


def rotation(**kw):
    r = dict(d_cos_sin=FAKE, table_dtype=F32, interleaved=0, max_positions=16, rotary_dim=D, row_stride=D,
             d_positions=FAKE, position_bytes=8)
    r.update(kw)
    return _lib.Rotation(*[r[f] for f, _ in _lib.Rotation._fields_])


def norm(**kw):
    n = dict(d_query_weight=FAKE, d_key_weight=FAKE, query_weight_dtype=BF16, key_weight_dtype=BF16, eps=1e-6)
    n.update(kw)
    return _lib.HeadNorm(*[n[f] for f, _ in _lib.HeadNorm._fields_])


def ref(x):
    return None if x is None else ctypes.byref(x)


@pytest.mark.parametrize("change, message", [
    (dict(tokens=-1), "tokens must be"),
    (dict(head_dim=0), "head_dim must be"),
    (dict(q=None), "query and query_out are both needed"),
    (dict(ko=None), "key and key_out are both needed"),
    (dict(q=rows(dtype=9)), "query must be float16"),
    (dict(q=rows(heads=0)), "heads"),
    (dict(q=rows(data=None)), "query is null"),
    (dict(q=rows(data=FAKE + 1)), "not aligned"),
    (dict(k=rows(token=-1)), "negative stride"),
    (dict(qo=rows(token=D)), "query_out has rows that overlap"),
    (dict(qo=rows(token=0)), "query_out has rows that overlap"),
    (dict(qo=rows(head=D - 1, data=FAKE * 2)), "query_out has rows that overlap"),
    (dict(qo=rows(dtype=F16)), "query_out must have the type"),
    (dict(ko=rows(heads=5, data=FAKE * 8)), "key_out must have the heads"),
    (dict(qo=rows(token=8 * D, data=FAKE)), "must then have its strides"),
    (dict(k=rows(dtype=F32), ko=rows(dtype=F32, data=FAKE * 8)), "query and key must have the same type"),
    (dict(ko=rows(data=FAKE * 4)), "query_out and key_out are the same rows"),
    (dict(rot=None), "rotation is null"),
    (dict(rot=rotation(d_positions=None)), "positions"),
    (dict(rot=rotation(table_dtype=0)), "cos_sin must be"),
    (dict(rot=rotation(d_cos_sin=FAKE + 2)), "cos_sin is not aligned"),
    (dict(rot=rotation(rotary_dim=7)), "even in number"),
    (dict(rot=rotation(rotary_dim=D + 2)), "at most head_dim"),
    (dict(rot=rotation(rotary_dim=0)), "even in number"),
    (dict(rot=rotation(max_positions=0)), "no rows"),
    (dict(rot=rotation(row_stride=D - 1)), "rows overlap"),
    (dict(rot=rotation(position_bytes=2)), "positions must be int32 or int64"),
    (dict(rot=rotation(d_positions=FAKE + 4)), "positions are not aligned"),
    (dict(norm=norm(eps=-1.0)), "eps"),
    (dict(norm=norm(eps=float("nan"))), "eps"),
    (dict(norm=norm(eps=float("inf"))), "eps"),
    (dict(norm=norm(key_weight_dtype=0)), "norm weights must be"),
    (dict(norm=norm(d_query_weight=FAKE + 1)), "norm weights are not aligned"),
])
def test_norm_rope_refusals(change, message):
    L = _lib.lib()
    a = dict(q=rows(), qo=rows(data=FAKE * 4), k=rows(data=FAKE * 2), ko=rows(data=FAKE * 8), tokens=3, head_dim=D,
             rot=rotation(), norm=norm())
    a.update(change)
    rc = L.origami_norm_rope(ref(a["q"]), ref(a["qo"]), ref(a["k"]), ref(a["ko"]), a["tokens"], a["head_dim"],
                             ref(a["rot"]), ref(a["norm"]), None, None)
    assert rc == -1
    assert message in L.origami_last_error().decode()


@pytest.mark.parametrize("change, message", [
    (dict(cache=dict(d_data=None)), "kv cache is null"),
    (dict(cache=dict(layout=7)), "unknown kv cache layout"),
    (dict(cache=dict(d_data=FAKE + 2)), "16-byte aligned"),
    (dict(cache=dict(block_size=0)), "dimensions must be positive"),
    (dict(cache_dtype=F32), "paged cache must be"),
    (dict(slot_bytes=2), "slots must be int32 or int64"),
    (dict(slots=None), "slots are null"),
    (dict(slots=FAKE + 4), "not aligned"),
    (dict(k=None), "key and value are both needed"),
    (dict(v=None), "key and value are both needed"),
    (dict(v=rows(dtype=F16)), "key and value must have the same type"),
    (dict(k=rows(heads=2)), "the cache's 4 heads"),
    (dict(v=rows(heads=8)), "the cache's 4 heads"),
    (dict(q=rows(heads=8)), "query and query_out are both needed"),
    (dict(q=rows(dtype=F32), qo=rows(dtype=F32, data=FAKE * 4)), "query and key must have the same type"),
    (dict(rot=rotation(rotary_dim=D + 2)), "at most head_dim"),
    (dict(tokens=1 << 31), "tokens must be"),
])
def test_append_refusals(change, message):
    L = _lib.lib()
    a = dict(k=rows(), v=rows(data=FAKE * 2), q=None, qo=None, cache_dtype=BF16, slots=FAKE, slot_bytes=8, tokens=3,
             rot=rotation(), norm=None)
    c = dict(d_data=FAKE, layout=0, elem_bytes=2, num_blocks=8, block_size=16, num_heads=4, head_dim=D)
    c.update(change.get("cache", {}))
    a.update({k: v for k, v in change.items() if k != "cache"})
    cache = _lib.PagedKV(*[c[f] for f, _ in _lib.PagedKV._fields_])
    rc = L.origami_append_kv(ref(a["k"]), ref(a["v"]), ref(a["q"]), ref(a["qo"]), ctypes.byref(cache), a["cache_dtype"],
                             a["slots"], a["slot_bytes"], a["tokens"], ref(a["rot"]), ref(a["norm"]), None, None)
    assert rc in (-1, -2)
    assert message in L.origami_last_error().decode()


def test_no_tokens_is_no_launch():
    L = _lib.lib()
    cache = _lib.PagedKV(FAKE, 0, 2, 8, 16, 4, D)
    assert L.origami_append_kv(None, None, None, None, ctypes.byref(cache), BF16, None, 8, 0, None, None, None, None) == 0
    assert L.origami_norm_rope(None, None, None, None, 0, D, None, None, None, None) == 0


def test_host_tensors_are_refused():
    q = torch.zeros(2, 4, D)
    table = torch.zeros(8, D)
    with pytest.raises(ValueError, match="CUDA tensor"):
        norm_rope(q, q, torch.zeros(2, dtype=torch.int64), table)
    with pytest.raises(ValueError, match="CUDA tensor"):
        append_kv(torch.zeros(2, 4, 16, 4, D, dtype=torch.bfloat16), q, q, torch.zeros(2, dtype=torch.int64))
