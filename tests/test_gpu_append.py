"""norm_rope and append_kv against the formulas in 64 bits.

Tolerance of an element y = a cos - b sin (or b cos + a sin), derived: the store rounds by at
most half a step, eps/2 |y| (fp16: at least half its smallest step, 2^-25); in fp32 the norm's
sum of squares has at most D/32 + 15 roundings a path in either kernel (16 + 5 and D/32 + 5),
its square root halves them, and five more follow (division, eps, root, reciprocal, two
products), so a and b are off by less than 2^-18 relative (D <= 512: (31 / 2 + 6) 2^-24); the
rotation's three roundings add 3 * 2^-24 of |a cos| + |b sin|."""
from __future__ import annotations

import pytest
import torch

from origami_b200 import append, workloads

pytestmark = pytest.mark.gpu
EPS = 1e-5
BF16, F16, F32 = torch.bfloat16, torch.float16, torch.float32


def half_step(dtype):
    return torch.finfo(dtype).eps / 2, 2.0 ** -25 if dtype == F16 else 0.0


def expected(x, weight, positions, table, interleaved):
    """(value, allowance) of normed and rotated rows in 64 bits."""
    x = x.double()
    if weight is not None:
        x = x / (x.pow(2).mean(-1, keepdim=True) + EPS).sqrt() * weight.double()
    y, size = x.clone(), x.abs()
    if table is not None:
        R = table.shape[1]
        cs = table.double()[positions.long()][:, None]
        c, s = cs[..., :R // 2], cs[..., R // 2:]
        i = torch.arange(R // 2, device=x.device)
        i, j = (2 * i, 2 * i + 1) if interleaved else (i, i + R // 2)
        a, b = x[..., i], x[..., j]
        y[..., i], y[..., j] = a * c - b * s, b * c + a * s
        size[..., i], size[..., j] = (a * c).abs() + (b * s).abs(), (b * c).abs() + (a * s).abs()
    return y, size * (2.0 ** -18 + 3 * 2.0 ** -24)


def assert_rows(got, want, allowance, dtype):
    rel, least = half_step(dtype)
    off = (got.double() - want).abs()
    bound = allowance + torch.clamp(rel * (want.abs() + allowance), min=least)
    assert bool((off <= bound).all()), float((off - bound).max())


def table_for(R, n, dtype, dev):
    ang = torch.arange(n, dtype=torch.float64)[:, None] * 10000.0 ** (-torch.arange(0, R, 2, dtype=torch.float64) / R)
    return torch.cat([ang.cos(), ang.sin()], 1).to(dtype).to(dev)


def make(T, Hq, Hk, D, dtype, dev, packed, seed, shift=0):
    g = torch.Generator(device=dev).manual_seed(seed)
    n = (Hq + 2 * Hk) * D
    if packed:
        flat = torch.randn(T * n + shift, generator=g, device=dev).to(dtype)[shift:].view(T, n)
        return [x.unflatten(1, (-1, D)) for x in flat.split([Hq * D, Hk * D, Hk * D], 1)]
    return [torch.randn(T, h, D, generator=g, device=dev).to(dtype) for h in (Hq, Hk, Hk)]


SHAPES = [  # T, Hq, Hk, D, R, interleaved
    (1, 32, 8, 128, 128, False),
    (5, 28, 4, 128, 128, False),
    (300, 3, 1, 64, 64, False),
    (7, 8, 8, 256, 64, False),     # partial, wide head
    (33, 5, 1, 96, 96, False),     # 6 of 8 lanes
    (9, 2, 1, 80, 80, True),
    (9, 2, 1, 80, 40, False),      # 20 pairs: the kernel for any layout
    (11, 4, 2, 72, 24, True),      # 9 chunks, 3 of them turned
    (11, 4, 2, 40, 8, True),
    (3, 2, 1, 512, 512, False),
    (3, 2, 1, 520, 520, False),    # past the fast kernel's widest head
    (6, 3, 3, 7, 6, False),        # odd heads
    (6, 3, 3, 1, 0, False),
    (2, 1, 1, 2, 2, True),
    (5000, 4, 1, 64, 32, True),
    # a walker steps through several tokens, the last pass being partial
    (4001, 28, 4, 128, 128, False),
    (12000, 5, 2, 96, 48, False),
    (9600, 3, 5, 40, 16, True),    # more key heads than the query heads' walkers
]


@pytest.mark.parametrize("norm", [True, False])
@pytest.mark.parametrize("dtype", [BF16, F16, F32])
@pytest.mark.parametrize("T, Hq, Hk, D, R, interleaved", [s for s in SHAPES if s[4] > 0])
def test_norm_rope(cuda, T, Hq, Hk, D, R, interleaved, dtype, norm):
    q, k, _ = make(T, Hq, Hk, D, dtype, cuda, T % 2 == 1, T + D)
    table = table_for(R, 4096, F32, cuda)
    pos = torch.randint(0, 4096, (T,), generator=torch.Generator().manual_seed(D)).to(cuda)
    qw = (torch.rand(D, device=cuda) + 0.5).to(dtype) if norm else None
    kw = (torch.rand(D, device=cuda) + 0.5).to(F32) if norm else None
    qo, ko = append.norm_rope(q, k, pos, table, query_weight=qw, key_weight=kw, eps=EPS, interleaved=interleaved)
    for got, x, w in ((qo, q, qw), (ko, k, kw)):
        assert got.dtype == dtype and got.shape == x.shape
        assert_rows(got, *expected(x, w, pos, table, interleaved), dtype)
    # in place, 32-bit positions: the same bits
    q2, k2 = q.clone(), k.clone()
    append.norm_rope(q2, k2, pos.int(), table, query_weight=qw, key_weight=kw, eps=EPS, interleaved=interleaved,
                     query_out=q2, key_out=k2)
    assert torch.equal(q2, qo) and torch.equal(k2, ko)


@pytest.mark.parametrize("table_dtype", [F32, BF16, F16])
@pytest.mark.parametrize("shift", [0, 1, 8])
def test_norm_rope_packed_in_place_and_tables(cuda, table_dtype, shift):
    """Slices of a fused projection rewritten in place, at any alignment; the value slice stays."""
    T, Hq, Hk, D = 41, 6, 2, 128
    q, k, v = make(T, Hq, Hk, D, BF16, cuda, True, 3, shift)
    table = table_for(D, 64, table_dtype, cuda)
    pos = torch.arange(T, device=cuda)
    w = torch.full((D,), 0.75, dtype=BF16, device=cuda)
    want = [expected(q, w, pos, table, False), expected(k, None, pos, table, False)]
    v0 = v.clone()
    append.norm_rope(q, k, pos, table, query_weight=w, eps=EPS, query_out=q, key_out=k)
    assert_rows(q, *want[0], BF16)
    assert_rows(k, *want[1], BF16)
    assert torch.equal(v, v0)


def flat_slots(cache, kv_first):
    """[2, slots, H, D] copy of a cache."""
    by_kv = cache if kv_first else cache.transpose(0, 1)
    return by_kv.flatten(1, 2).clone()


@pytest.mark.parametrize("kv_first", [True, False])
@pytest.mark.parametrize("dtype, cache_dtype", [(BF16, BF16), (F16, F16), (F16, BF16), (BF16, F16), (F32, BF16), (F32, F16)])
@pytest.mark.parametrize("T, Hq, Hk, D, R, interleaved, bs", [
    (1, 32, 8, 128, 128, False, 16),
    (19, 28, 4, 128, 128, False, 32),
    (300, 0, 2, 64, 32, True, 5),
    (23, 3, 1, 96, 48, False, 1),
    (10, 2, 2, 80, 0, False, 7),
    (12, 3, 3, 7, 6, True, 3),
    (4001, 28, 4, 128, 128, False, 16),
    (20011, 0, 2, 64, 32, False, 5),
    (12000, 5, 1, 72, 0, False, 8),
])
def test_append(cuda, T, Hq, Hk, D, R, interleaved, bs, dtype, cache_dtype, kv_first):
    q, k, v = make(T, max(Hq, 1), Hk, D, dtype, cuda, T % 2 == 1, T + D)
    blocks = T // bs + 4
    shape = (2, blocks, bs, Hk, D) if kv_first else (blocks, 2, bs, Hk, D)
    cache = torch.randn(shape, device=cuda).to(cache_dtype)
    before = flat_slots(cache, kv_first)
    slots = torch.randperm(blocks * bs, generator=torch.Generator().manual_seed(T))[:T].to(cuda)
    slots[T // 2:T // 2 + (T > 4)] = -1  # a padded token
    table = table_for(R, 4096, F32, cuda) if R else None
    pos = torch.randint(0, 4096, (T,), generator=torch.Generator().manual_seed(D)).to(cuda) if R else None
    kw = (torch.rand(D, device=cuda) + 0.5).to(F16)
    err = torch.zeros(1, dtype=torch.int32, device=cuda)
    out = append.append_kv(cache, k, v, slots, query=q if Hq else None, positions=pos, cos_sin=table, key_weight=kw,
                           eps=EPS, interleaved=interleaved, error_count=err)
    after = flat_slots(cache, kv_first)
    live = slots >= 0
    want, allow = expected(k, kw, pos, table, interleaved)
    assert_rows(after[0][slots[live]], want[live], allow[live], cache_dtype)
    assert torch.equal(after[1][slots[live]], v[live].float().to(cache_dtype))
    other = torch.ones(blocks * bs, dtype=torch.bool, device=cuda)
    other[slots[live]] = False
    assert torch.equal(after[:, other], before[:, other])
    assert int(err) == 0
    if Hq:
        assert_rows(out, *expected(q, None, pos, table, interleaved), dtype)
    else:
        assert out is None


@pytest.mark.parametrize("D", [64, 10])
def test_bad_slots_and_positions_are_skipped_and_counted(cuda, D):
    T, Hq, Hk, bs, blocks = 6, 3, 2, 4, 5
    q, k, v = make(T, Hq, Hk, D, BF16, cuda, False, 1)
    cache = torch.zeros((2, blocks, bs, Hk, D), dtype=BF16, device=cuda)
    table = table_for(D, 8, F32, cuda)
    slots = torch.tensor([3, blocks * bs, -2, -1, 7, -1], dtype=torch.int32, device=cuda)
    pos = torch.tensor([0, 1, 2, 7, 8, -1], dtype=torch.int64, device=cuda)
    out = torch.full_like(q, 9.0)
    err = torch.zeros(1, dtype=torch.int32, device=cuda)
    append.append_kv(cache, k, v, slots, query=q, positions=pos, cos_sin=table, query_out=out, error_count=err)
    # token 1 and 2: K and V rows; 4: query, K and V rows; 5: query rows
    assert int(err) == 2 * 2 * Hk + (Hq + 2 * Hk) + Hq
    assert bool((out[4:] == 9.0).all()) and bool((out[:4] != 9.0).any(-1).all())
    flat = flat_slots(cache, True)
    assert torch.equal(flat[1][3], v[0])
    flat[:, 3] = 0
    assert not flat.any()


def test_skipped_and_padded_tokens_between_others_of_a_long_step(cuda):
    T, Hq, Hk, D, bs = 12007, 5, 2, 64, 16
    q, k, v = make(T, Hq, Hk, D, BF16, cuda, True, 8)
    blocks = T // bs + 1
    cache = torch.full((blocks, 2, bs, Hk, D), 3.0, dtype=BF16, device=cuda)
    i = torch.arange(T, device=cuda)
    slots = torch.randperm(blocks * bs, generator=torch.Generator().manual_seed(1))[:T].to(cuda)
    padded, outside, bad = i % 7 == 2, i % 11 == 3, i % 13 == 4
    slots[outside] = blocks * bs + 5
    slots[padded] = -1
    outside &= ~padded
    pos = i % 100
    pos[bad] = 100
    table = table_for(D, 100, F32, cuda)
    out = torch.full_like(q, 9.0)
    err = torch.zeros(1, dtype=torch.int32, device=cuda)
    append.append_kv(cache, k, v, slots, query=q, positions=pos, cos_sin=table, query_out=out, error_count=err)
    written = ~(padded | outside | bad)
    assert int(err) == int(bad.sum()) * Hq + int((outside | (bad & ~padded)).sum()) * 2 * Hk
    want, allow = expected(q, None, pos.clamp(max=99), table, False)
    assert_rows(out[~bad], want[~bad], allow[~bad], BF16)
    assert bool((out[bad] == 9.0).all())
    flat = flat_slots(cache, False)
    want, allow = expected(k, None, pos.clamp(max=99), table, False)
    assert_rows(flat[0][slots[written]], want[written], allow[written], BF16)
    assert torch.equal(flat[1][slots[written]], v[written])
    flat[:, slots[written]] = 3.0
    assert bool((flat == 3.0).all())


def test_non_finite_rows_stay_in_their_rows(cuda):
    T, H, D = 8, 4, 128
    q, k, _ = make(T, H, H, D, BF16, cuda, False, 5)
    q[2, 1, 5], q[3, 0, 100] = float("nan"), float("inf")
    table = table_for(64, 64, F32, cuda)
    pos = torch.arange(T, device=cuda)
    out, _ = append.norm_rope(q, k, pos, table, eps=EPS)
    bad = ~torch.isfinite(out)
    # without a norm a pair spreads to its partner only, and an unturned dim to nothing
    assert bad[2, 1].nonzero().flatten().tolist() == [5, 37]
    assert bad[3, 0].nonzero().flatten().tolist() == [100]
    assert int(bad.sum()) == 3


def test_far_cache_rows(cuda):
    """Element offsets past 2^32: the last block of a cache of 8.6 GB."""
    H, D, bs = 8, 128, 16
    blocks = (1 << 32) // (2 * bs * H * D) + 3
    cache = torch.zeros((blocks, 2, bs, H, D), dtype=BF16, device=cuda)
    _, k, v = make(1, 1, H, D, BF16, cuda, False, 2)
    slot = torch.tensor([blocks * bs - 1], device=cuda)
    append.append_kv(cache, k, v, slot)
    assert torch.equal(cache[-1, 0, -1], k[0]) and torch.equal(cache[-1, 1, -1], v[0])
    assert int(cache[:-1].view(torch.int16).count_nonzero()) == 0


def test_streams_and_graph(cuda):
    T, Hq, Hk, D, bs = 16, 8, 2, 128, 16
    q, k, v = make(T, Hq, Hk, D, BF16, cuda, True, 9)
    table = table_for(D, 256, F32, cuda)
    slots, pos = torch.arange(T, device=cuda), torch.arange(T, device=cuda)
    cache = torch.zeros((2, 4, bs, Hk, D), dtype=BF16, device=cuda)
    want = append.append_kv(cache, k, v, slots, query=q, positions=pos, cos_sin=table)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    cache2 = torch.zeros_like(cache)
    side.wait_stream(torch.cuda.current_stream())
    got = append.append_kv(cache2, k, v, slots, query=q, positions=pos, cos_sin=table, stream=side)
    side.synchronize()
    assert torch.equal(got, want) and torch.equal(cache2, cache)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got = append.append_kv(cache2, k, v, slots, query=q, positions=pos, cos_sin=table)
    # a replay reads what the tensors hold then
    slots.add_(bs)
    pos.add_(100)
    cache2.zero_()
    cache.zero_()
    graph.replay()
    want = append.append_kv(cache, k, v, slots, query=q, positions=pos, cos_sin=table)
    assert torch.equal(got, want) and torch.equal(cache2, cache)


def test_front_end_refusals(cuda):
    T, H, D = 4, 2, 64
    q, k, v = make(T, H, H, D, BF16, cuda, False, 1)
    cache = torch.zeros((2, 4, 16, H, D), dtype=BF16, device=cuda)
    slots = torch.arange(T, device=cuda)
    table, pos = table_for(D, 8, F32, cuda), torch.arange(T, device=cuda)
    for call, message in (
            (lambda: append.append_kv(cache, k[:, :1], v, slots), "the cache's 2 heads"),
            (lambda: append.append_kv(cache, k.transpose(1, 2).contiguous().transpose(1, 2), v, slots), "last dimension"),
            (lambda: append.append_kv(cache, k, v, slots[:2]), "one per token"),
            (lambda: append.append_kv(cache, k, v, slots.float()), "int32 or int64"),
            (lambda: append.append_kv(cache, k, v, slots, positions=pos), "go together"),
            (lambda: append.append_kv(cache.float(), k, v, slots), "16-bit"),
            (lambda: append.append_kv(cache, k, v, slots, query_weight=table[0]), "need a query"),
            (lambda: append.append_kv(cache, k, v, slots, key_weight=table[0, :8]), "vector of 64"),
            (lambda: append.norm_rope(q, k, pos, table[:, :63]), "even in number"),
            (lambda: append.norm_rope(q, k, pos.cpu(), table), "CUDA tensor"),
            (lambda: append.norm_rope(q, k, pos, table, query_out=q[:, :1].expand(T, H, D)), "rows that overlap"),
            (lambda: append.norm_rope(q, k, pos, table, query_out=k, key_out=k), "same rows"),
            (lambda: append.norm_rope(q.double(), k, pos, table), "float16, bfloat16 or float32"),
    ):
        with pytest.raises((ValueError, RuntimeError), match=message):
            call()
    empty = q[:0]
    a, b = append.norm_rope(empty, empty, pos[:0], table)
    assert a.shape == (0, H, D) and b.shape == (0, H, D)


def test_appended_rows_pack_and_restore(cuda):
    """A request appended token by token is what pack_layer saves and restore_layer brings back."""
    from origami_b200 import BYTE_PLANES, LayerFormat
    from origami_b200.layer import pack_layer, restore_layer

    T, H, D, bs = 53, 4, 128, 16
    _, k, v = make(T, 1, H, D, BF16, cuda, True, 4)
    nb = (T + bs - 1) // bs
    ids = workloads.permuted_block_table(nb, nb + 3, seed=7)
    t = torch.arange(T)
    slots = (ids[t // bs] * bs + t % bs).to(cuda)
    table = table_for(D, 64, F32, cuda)
    cache = torch.zeros((2, nb + 3, bs, H, D), dtype=BF16, device=cuda)
    for a, b in ((0, 40), (40, 41), (41, T)):
        append.append_kv(cache, k[a:b], v[a:b], slots[a:b], positions=t[a:b].to(cuda), cos_sin=table)
    fmt = LayerFormat(T, H, D, BYTE_PLANES)
    fresh = torch.zeros_like(cache)
    restore_layer(pack_layer(cache, ids, fmt), fmt, fresh, ids)
    assert torch.equal(fresh, cache)
    want, allow = expected(k, None, t.to(cuda), table, False)
    assert_rows(workloads.tokens_from_cache(fresh, ids, T)[0], want, allow, BF16)


def at_odd_element(t):
    """A contiguous copy of t that starts one element behind an aligned address."""
    flat = torch.empty(t.numel() + 1, dtype=t.dtype, device=t.device)
    return flat[1:].view_as(t).copy_(t)


@pytest.mark.parametrize("T", [1, 3, 6001])
@pytest.mark.parametrize("weight_dtype", [F32, BF16])
def test_results_do_not_depend_on_where_weights_lie(cuda, T, weight_dtype):
    """Weights that are slices of a flat parameter buffer: the same bits as with aligned ones."""
    Hq, Hk, D, bs = 8, 2, 128, 16
    q, k, v = make(T, Hq, Hk, D, F32, cuda, True, 12)
    table, pos = table_for(D, 512, F32, cuda), torch.arange(T, device=cuda) % 512
    qw, kw = ((torch.rand(D, device=cuda) + 0.5).to(weight_dtype) for _ in range(2))
    want = append.norm_rope(q, k, pos, table, query_weight=qw, key_weight=kw, eps=EPS)
    got = append.norm_rope(q, k, pos, table, query_weight=at_odd_element(qw), key_weight=at_odd_element(kw), eps=EPS)
    assert torch.equal(got[0], want[0]) and torch.equal(got[1], want[1])
    slots = torch.randperm(T + 7, generator=torch.Generator().manual_seed(3))[:T].to(cuda)
    caches, outs = [], []
    for w in (kw, at_odd_element(kw)):
        caches.append(torch.zeros((2, (T + 7) // bs + 1, bs, Hk, D), dtype=F16, device=cuda))
        outs.append(append.append_kv(caches[-1], k, v, slots, query=q, query_weight=qw, key_weight=w, eps=EPS,
                                     positions=pos, cos_sin=table))
    assert torch.equal(caches[0], caches[1]) and torch.equal(outs[0], outs[1])


@pytest.mark.parametrize("T, H", [(1, 8), (5001, 1), (1, 1)])
def test_results_do_not_depend_on_strides_that_nothing_uses(cuda, T, H):
    """The token stride of one token and the head stride of one head are any number."""
    D = 128
    q, k, _ = make(T, H, H, D, F32, cuda, False, 14)
    table, pos = table_for(D, 512, F32, cuda), torch.arange(T, device=cuda) % 512
    w = torch.rand(D, device=cuda) + 0.5
    want = append.norm_rope(q, k, pos, table, query_weight=w, key_weight=w, eps=EPS)

    def odd(t):
        return t.as_strided(t.shape, (t.stride(0) if T > 1 else D * H + 1, t.stride(1) if H > 1 else D + 1, 1))

    out = [torch.empty_like(t) for t in (q, k)]
    got = append.norm_rope(odd(q), odd(k), pos, table, query_weight=w, key_weight=w, eps=EPS, query_out=odd(out[0]),
                           key_out=odd(out[1]))
    assert torch.equal(got[0], want[0]) and torch.equal(got[1], want[1])
