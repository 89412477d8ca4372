"""shared_prefix_attention against the formula in 64 bits.

Tolerance of an element, derived. With u half a step of the type, A = sum p |v| / sum p:
the probabilities' rounding gives u A and the store u |out|. A score is off by at most
e = scale (D / 8) 2^-22 |q|.|k| (the tensor cores add 8 or more products a step in fp32,
possibly truncating: a whole step 2^-23 each, twice that allowed) plus 2^-22 (1 + max |s|)
for the exponent's argument and ex2; it moves numerator and denominator by e each: 2 e A. The
sums over N keys add at most (N / 8 + 64) 2^-23 of A (as many accumulations, sums of 16 or
more at a time and the joins). lse is off by e and the sum's part."""
from __future__ import annotations

import math

import pytest
import torch

from origami_b200 import shared_prefix, workloads
from origami_b200.append import append_kv
from origami_b200.shared_prefix import shared_prefix_attention

pytestmark = pytest.mark.gpu
BF16, F16 = torch.bfloat16, torch.float16


class Batch:
    """A paged cache with a shared prefix and one suffix per request; everything no request may
    read is NaN."""

    def __init__(self, dev, new, suffix, prefix, Hq, Hk, D, bs, dtype, kv_first=True, seed=0, k_std=1.0):
        g = torch.Generator(device=dev).manual_seed(seed)
        self.new, self.suffix, self.prefix, self.bs, self.kv_first = new, suffix, prefix, bs, kv_first
        self.Hq, self.Hk, self.D, self.dtype, self.dev = Hq, Hk, D, dtype, dev
        nblk = lambda n: (n + bs - 1) // bs
        blocks = nblk(prefix) + sum(nblk(s) for s in suffix) + 2
        shape = (2, blocks, bs, Hk, D) if kv_first else (blocks, 2, bs, Hk, D)
        self.cache = torch.full(shape, float("nan"), dtype=dtype, device=dev)
        ids = torch.randperm(blocks, generator=torch.Generator().manual_seed(seed)).to(torch.int32)
        self.prefix_blocks = ids[:nblk(prefix)].to(dev)
        at = nblk(prefix)
        table = torch.full((len(new), max(1, max(nblk(s) for s in suffix))), -7, dtype=torch.int32)
        for b, s in enumerate(suffix):
            table[b, :nblk(s)] = ids[at:at + nblk(s)]
            at += nblk(s)
        self.suffix_blocks = table.to(dev)
        self.suffix_lens = torch.tensor(suffix, dtype=torch.int32, device=dev)
        self.query_start = torch.tensor([0] + list(torch.tensor(new).cumsum(0)), dtype=torch.int32, device=dev)
        self.q = torch.randn(sum(new), Hq, D, generator=g, device=dev).to(dtype)
        fill = lambda n: torch.stack([torch.randn(n, Hk, D, generator=g, device=dev) * k_std,
                                      torch.randn(n, Hk, D, generator=g, device=dev)]).to(dtype)
        self.pkv = fill(prefix)
        self.skv = [fill(s) for s in suffix]
        if prefix:
            self.write(self.pkv, self.prefix_blocks)
        for b, s in enumerate(suffix):
            if s:
                self.write(self.skv[b], self.suffix_blocks[b])

    def write(self, kv, ids):
        n = kv.shape[1]
        t = torch.arange(n, device=self.dev)
        blk, off = ids.long()[t // self.bs], t % self.bs
        by_kv = self.cache if self.kv_first else self.cache.transpose(0, 1)
        by_kv[:, blk, off] = kv

    def run(self, **kw):
        args = dict(query=self.q, kv_layer=self.cache, query_start=self.query_start, prefix_blocks=self.prefix_blocks,
                    prefix_tokens=self.prefix, suffix_blocks=self.suffix_blocks, suffix_lens=self.suffix_lens)
        args.update(kw)
        return shared_prefix_attention(**args)

    def check(self, out, lse=None, scale=None):
        scale = self.D ** -0.5 if scale is None else scale
        g = self.Hq // self.Hk
        u = torch.finfo(self.dtype).eps / 2
        at = 0
        for b, (n, s) in enumerate(zip(self.new, self.suffix)):
            if n == 0:
                continue
            kv = torch.cat([self.pkv, self.skv[b]], 1).double()
            k, v = (x.repeat_interleave(g, 1).transpose(0, 1) for x in kv)  # [Hq, N, D]
            q = self.q[at:at + n].double().transpose(0, 1)
            N = k.shape[1]
            seen = torch.arange(N, device=self.dev)[None] < (self.prefix + (s - n + torch.arange(n, device=self.dev) + 1)
                                                             .clamp(min=0))[:, None]
            sc = (q @ k.transpose(1, 2) * scale).masked_fill(~seen, -math.inf)
            mag = (q.abs() @ k.abs().transpose(1, 2) * scale).masked_fill(~seen, 0)
            err = (mag.amax(-1) if N else torch.zeros(self.Hq, n, device=self.dev).double()) * (self.D / 8) * 2.0 ** -22
            smax = sc.masked_fill(~seen, 0).abs().amax(-1) if N else torch.zeros_like(err)
            err = err + 2.0 ** -22 * (1 + smax)
            z = torch.logsumexp(sc, -1) if N else torch.full((self.Hq, n), -math.inf, device=self.dev).double()
            empty = ~seen.any(-1) if N else torch.ones(n, dtype=torch.bool, device=self.dev)
            p = torch.exp(sc - z.masked_fill(empty[None], 0)[..., None])
            want, A = p @ v, p @ v.abs()
            sums = (N / 8 + 64) * 2.0 ** -23
            tol = (u + 2 * err[..., None] + sums) * A + u * want.abs() + (2.0 ** -25 if self.dtype == F16 else 0)
            off = (out[at:at + n].double().transpose(0, 1) - want).abs()
            assert bool((off <= tol).all()), (b, float((off - tol).nan_to_num(1e9).max()), float(off.nan_to_num(1e9).max()))
            if lse is not None:
                got = lse[at:at + n].double().T
                assert bool((got[:, empty] == -math.inf).all())
                d = (got - z)[:, ~empty].abs()
                assert bool((d <= (err + sums + 2.0 ** -22 * (1 + z.abs()))[:, ~empty]).all()), float(d.max())
            at += n


CASES = [  # new, suffix, prefix, Hq, Hk, D, block size
    ([1], [1], 1, 1, 1, 64, 16),
    ([1], [1], 0, 4, 1, 128, 16),
    ([1], [0], 128, 8, 8, 128, 16),
    ([1, 1], [1, 40], 512, 32, 8, 128, 16),
    ([1, 1, 1], [129, 0, 5], 127, 28, 4, 128, 32),
    ([1, 3, 2, 5], [7, 3, 300, 250], 130, 28, 4, 128, 32),
    ([5, 1, 4], [2, 0, 4], 0, 6, 2, 64, 16),          # rows without a key
    ([3, 0, 2], [3, 9, 2], 33, 8, 2, 128, 5),         # a request without new tokens, odd pages
    ([1] * 40, list(range(40)), 1000, 32, 8, 128, 16),  # 160 rows a KV head: pair
    ([1] * 33, [64] * 33, 2000, 8, 2, 64, 16),        # 132 rows: pair with 4 rows in its second tile
    ([1] * 70, [3] * 70, 300, 4, 1, 128, 16),         # 280 rows: a pair, then one row tile
    ([1] * 9, [128] * 9, 128, 32, 1, 64, 1),          # pages of one token
    ([300, 1, 77], [500, 2, 77], 257, 16, 2, 64, 16), # chunks of prompts
    ([130], [130], 0, 5, 5, 128, 7),                  # a whole prompt, no prefix
    ([40, 40], [40, 90], 64, 128, 1, 128, 16),        # 128 query heads a KV head
    ([7, 9], [7, 20], 50, 100, 1, 64, 48),
    ([1], [5], 40000, 8, 1, 128, 16),                 # one long prefix over every CTA
    ([1], [30000], 5, 8, 1, 128, 16),                 # one long suffix over every CTA
    ([2] * 300, [2 + i % 200 for i in range(300)], 90, 2, 2, 64, 16),
    # blocks of 8, 24, 64 and 256 rows: every size of box, boxes beside rows copied one by one
    ([1, 2, 1], [200, 129, 31], 517, 8, 2, 128, 8),
    ([1, 2, 1], [200, 129, 31], 517, 8, 2, 64, 24),
    ([1] * 50, [1 + 13 * i for i in range(50)], 1025, 16, 4, 128, 64),
    ([3, 1], [700, 300], 900, 8, 2, 64, 256),
    # thousands of rows: several a warp in the join, of few partials each and of many, some without a key
    ([200, 193, 7], [150, 193, 60], 0, 6, 2, 128, 16),
    ([300, 300], [300, 350], 100, 24, 2, 64, 16),
    ([20], [25], 12000, 128, 1, 64, 16),
    ([64] * 6, [64 + i for i in range(6)], 700, 32, 4, 128, 16),
]


@pytest.mark.parametrize("dtype", [BF16, F16])
@pytest.mark.parametrize("case", range(len(CASES)))
def test_against_the_formula(cuda, case, dtype):
    new, suffix, prefix, Hq, Hk, D, bs = CASES[case]
    x = Batch(cuda, new, suffix, prefix, Hq, Hk, D, bs, dtype, kv_first=(case + (dtype == F16)) % 2 == 0, seed=case)
    lse = torch.empty(sum(new), Hq, dtype=torch.float32, device=cuda)
    flags = torch.zeros(1, dtype=torch.int32, device=cuda)
    out = x.run(lse=lse, error_flags=flags)
    assert int(flags) == 0
    x.check(out, lse)
    # no lse, a given scale, a workspace full of NaN: the order of the sums does not change
    ws = torch.full((shared_prefix.workspace_bytes(sum(new), Hq, Hk, D, len(new), cuda),), 0xFF, dtype=torch.uint8,
                    device=cuda)
    again = x.run(softmax_scale=D ** -0.5, workspace=ws)
    assert torch.equal(out, again)
    odd = torch.empty(out.numel() + 1, dtype=dtype, device=cuda)[1:].view_as(out)  # an output at an odd element
    assert torch.equal(x.run(out=odd), out)


@pytest.mark.parametrize("k_std", [0.01, 8.0, 40.0])
def test_flat_and_peaked_scores(cuda, k_std):
    """Maxima that grow from tile to tile (rescaled sums) and scores that are all alike."""
    x = Batch(cuda, [1] * 20, [30 + 17 * i for i in range(20)], 3000, 16, 2, 128, 16, BF16, seed=3, k_std=k_std)
    lse = torch.empty(20, 16, dtype=torch.float32, device=cuda)
    x.check(x.run(lse=lse), lse)


@pytest.mark.parametrize("scale", [1e-4, 1.0])
def test_scales(cuda, scale):
    x = Batch(cuda, [2] * 3, [40] * 3, 200, 4, 2, 64, 16, F16, seed=4)
    x.check(x.run(softmax_scale=scale), scale=scale)


def test_strided_unaligned_and_padded(cuda):
    """A query slice of a fused projection at an odd element, an output of other strides, tables
    that are slices of wider ones, tokens behind the last request left alone."""
    x = Batch(cuda, [1, 2, 1], [20, 35, 1], 150, 8, 2, 128, 16, BF16, seed=5)
    T, Hq, D = x.q.shape
    for shift in (0, 1):
        flat = torch.zeros((T + 3) * (Hq + 4) * D + shift, dtype=BF16, device=cuda)
        wide = flat[shift:].view(T + 3, Hq + 4, D)
        wide[:T, :Hq] = x.q
        wide[T:] = float("nan")
        store = torch.full((Hq * (T + 3) * D + shift,), 9.0, dtype=BF16, device=cuda)
        out = store[shift:].view(Hq, T + 3, D).transpose(0, 1)
        lse = torch.full((T + 3, Hq), 5.0, device=cuda)
        tables = torch.cat([torch.full((3, 2), 10 ** 6, dtype=torch.int32, device=cuda), x.suffix_blocks], 1)
        got = x.run(query=wide[:, :Hq], out=out, lse=lse, suffix_blocks=tables[:, 2:])
        assert got is out
        x.check(out[:T], lse[:T])
        assert bool((out[T:] == 9.0).all()) and bool((lse[T:] == 5.0).all())


def test_blocks_outside_the_cache_read_as_zeros(cuda):
    x = Batch(cuda, [1, 1], [40, 3], 64, 4, 2, 64, 16, BF16, seed=6)
    x.prefix_blocks[1] = 10 ** 6
    x.pkv[:, 16:32] = 0
    x.suffix_blocks[0, 2] = -1
    x.skv[0][:, 32:40] = 0
    x.check(x.run())


def test_lengths_are_clamped_to_the_tables(cuda):
    x = Batch(cuda, [1, 1], [32, 48], 64, 4, 2, 64, 16, BF16, seed=7)
    want = x.run()
    x.suffix_lens[1] = 10 ** 9
    assert torch.equal(x.run(), want)
    x.suffix_lens[0] = -5
    x.suffix[0], x.skv[0] = 0, x.skv[0][:, :0]
    x.check(x.run())


def test_non_finite_values_reach_their_rows_only(cuda):
    x = Batch(cuda, [1, 1, 1], [20, 20, 20], 100, 4, 2, 64, 16, BF16, seed=8)
    x.skv[1][1, 3, 0, 5] = float("inf")
    x.skv[2][0, 4, 1, 7] = float("nan")
    x.write(x.skv[1], x.suffix_blocks[1])
    x.write(x.skv[2], x.suffix_blocks[2])
    out = x.run()
    assert bool(torch.isfinite(out[0]).all())
    assert bool(torch.isinf(out[1, :2, 5]).all()) and int((~torch.isfinite(out[1])).sum()) == 2
    assert bool(torch.isnan(out[2, 2:]).all()) and bool(torch.isfinite(out[2, :2]).all())
    x.q[0, 0, 0] = float("nan")
    out = x.run()
    assert bool(torch.isnan(out[0, 0]).all()) and bool(torch.isfinite(out[0, 1:]).all())


@pytest.mark.parametrize("B, Hq, Hk, D, prefix", [(64, 32, 8, 128, 16384), (200, 32, 8, 128, 8192), (96, 8, 2, 64, 20000)])
def test_under_load(cuda, B, Hq, Hk, D, prefix):
    """Segments of every kind in every CTA with the memory busy: the same bits each time."""
    x = Batch(cuda, [1] * B, [1 + 37 * i % 700 for i in range(B)], prefix, Hq, Hk, D, 16, BF16, seed=B)
    flags = torch.zeros(1, dtype=torch.int32, device=cuda)
    out = x.run(error_flags=flags)
    x.check(out)
    for _ in range(20):
        assert torch.equal(x.run(error_flags=flags), out)
    assert int(flags) == 0


def test_tokens_before_the_first_request_and_empty_tables(cuda):
    x = Batch(cuda, [2, 1], [3, 0], 70, 4, 2, 64, 16, BF16, seed=13)
    wide = torch.cat([torch.full_like(x.q[:2], float("nan")), x.q])
    out = torch.full_like(wide, 7.0)
    x.run(query=wide, query_start=x.query_start + 2, out=out)
    x.check(out[2:])
    assert bool((out[:2] == 7.0).all())
    # no suffix columns at all, and no prefix either
    x.suffix, x.skv = [0, 0], [kv[:, :0] for kv in x.skv]
    x.check(x.run(suffix_blocks=x.suffix_blocks[:, :0]))
    out = x.run(suffix_blocks=x.suffix_blocks[:, :0], prefix_blocks=x.prefix_blocks[:0], prefix_tokens=0)
    assert not out.any()


def test_query_start_that_falls_or_is_empty_writes_nothing(cuda):
    x = Batch(cuda, [2, 1, 1], [30, 9, 200], 70, 4, 2, 64, 16, BF16, seed=16)
    flags = torch.zeros(1, dtype=torch.int32, device=cuda)
    want, lse = x.run(), torch.full((4, 4), 5.0, device=cuda)
    ws = torch.empty(shared_prefix.workspace_bytes(4, 4, 2, 64, 3, cuda), dtype=torch.uint8, device=cuda)
    for starts, flag in (([0, 3, 2, 4], 1 << 30), ([4, 0, 4, 0], 1 << 30), ([0, 0, 0, 0], 0)):
        out = torch.full_like(x.q, 7.0)
        flags.zero_()
        x.run(query_start=torch.tensor(starts, dtype=torch.int32, device=cuda), out=out, lse=lse, error_flags=flags, workspace=ws)
        assert bool((out == 7.0).all()) and bool((lse == 5.0).all()) and int(flags) == flag, starts
        assert torch.equal(x.run(workspace=ws), want)


def test_calls_that_share_a_workspace_in_turn(cuda):
    """Other shapes, and a captured call, over the workspace another call left behind."""
    x = Batch(cuda, [1] * 3, [20, 300, 4], 500, 8, 2, 128, 16, BF16, seed=14)
    y = Batch(cuda, [5, 1], [5, 90], 40, 32, 2, 64, 16, F16, seed=15)
    need = max(shared_prefix.workspace_bytes(3, 8, 2, 128, 3, cuda), shared_prefix.workspace_bytes(6, 32, 2, 64, 2, cuda))
    ws = torch.empty(need, dtype=torch.uint8, device=cuda)
    a, b = x.run(), y.run()
    assert torch.equal(x.run(workspace=torch.empty(need + 16, dtype=torch.uint8, device=cuda)[16:]), a)  # 16-byte aligned
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        ga = x.run(workspace=ws)
    for _ in range(3):
        assert torch.equal(y.run(workspace=ws), b)
        graph.replay()
        assert torch.equal(ga, a)
        assert torch.equal(y.run(workspace=ws), b)


def test_streams_graph_and_changed_lengths(cuda):
    x = Batch(cuda, [1, 2, 1], [20, 35, 4], 300, 8, 2, 128, 16, BF16, seed=9)
    want = x.run()
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    got = x.run(stream=side)
    side.synchronize()
    assert torch.equal(got, want)
    graphs, outs = [], []
    for _ in range(2):  # two graphs, each with a workspace of its own pool
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            outs.append(x.run())
        graphs.append(g)
    x.suffix_lens.copy_(torch.tensor([7, 30, 2], dtype=torch.int32))
    x.query_start.copy_(torch.tensor([0, 2, 3, 4], dtype=torch.int32))
    for g in graphs:
        g.replay()
    x.new, x.suffix = [2, 1, 1], [7, 30, 2]
    x.skv = [kv[:, :s] for kv, s in zip(x.skv, x.suffix)]
    for o in outs:
        x.check(o)
    assert torch.equal(outs[0], outs[1])


def test_far_cache_rows(cuda):
    """Element offsets past 2^32."""
    Hk, D, bs = 8, 128, 16
    x = Batch(cuda, [1, 1], [17, 5], 40, 16, Hk, D, bs, BF16, kv_first=False, seed=10)
    blocks = (1 << 32) // (2 * bs * Hk * D) + x.cache.shape[0]
    far = torch.zeros((blocks, 2, bs, Hk, D), dtype=BF16, device=cuda)
    shift = blocks - x.cache.shape[0]
    far[shift:] = x.cache
    out = x.run(kv_layer=far, prefix_blocks=x.prefix_blocks + shift, suffix_blocks=x.suffix_blocks + shift)
    assert torch.equal(out, x.run())
    x.check(out)


def test_front_end_refusals(cuda):
    x = Batch(cuda, [1, 1], [17, 5], 40, 8, 2, 64, 16, BF16, seed=11)
    for kw, message in (
            (dict(query=x.q[..., :32]), "head_dim"),
            (dict(query=x.q.half()), "dtype must match"),
            (dict(query=x.q.float()), "float16 or bfloat16"),
            (dict(query=x.q[:, :7]), "divisible"),
            (dict(prefix_tokens=10 ** 4), "too short"),
            (dict(prefix_tokens=-1), "not be negative"),
            (dict(suffix_lens=x.suffix_lens.long()), "int32"),
            (dict(suffix_lens=x.suffix_lens[:1]), "one entry"),
            (dict(query_start=x.query_start[:2]), "one more"),
            (dict(suffix_blocks=x.suffix_blocks.T.contiguous().T), "last dimension"),
            (dict(softmax_scale=0.0), "finite and positive"),
            (dict(softmax_scale=float("nan")), "finite and positive"),
            (dict(out=x.q[:1]), "shape"),
            (dict(out=x.q[:1].expand_as(x.q)), "overlap"),
            (dict(lse=torch.empty(2, 8, device=cuda, dtype=BF16)), "lse must be"),
            (dict(workspace=torch.empty(16, dtype=torch.uint8, device=cuda)), "workspace must be"),
            (dict(query_start=x.query_start.cpu()), "CUDA tensor"),
    ):
        with pytest.raises((ValueError, RuntimeError), match=message):
            x.run(**kw)
    empty = x.run(query=x.q[:0])
    assert empty.shape == (0, 8, 64)


def test_step_over_a_restored_prefix(cuda):
    """The ops as a step uses them: a packed prefix restored into the cache, three steps of new
    tokens appended (norm, rotation, paged write), each attending to prefix and suffix."""
    from origami_b200 import BYTE_PLANES, LayerFormat
    from origami_b200.layer import pack_layer, restore_layer

    B, P, Hq, Hk, D, bs, steps = 5, 77, 8, 2, 128, 16, 3
    g = torch.Generator(device=cuda).manual_seed(12)
    table = torch.cat([f(torch.arange(256, dtype=torch.float64)[:, None] * 10000.0 ** (-torch.arange(0, D, 2) / D)[None])
                       for f in (torch.cos, torch.sin)], 1).float().to(cuda)
    rnd = lambda *s: torch.randn(*s, generator=g, device=cuda).to(BF16)
    nb = (P + bs - 1) // bs
    ids = workloads.permuted_block_table(nb + B, nb + B + 2, seed=3)
    saved = torch.zeros((2, nb + B + 2, bs, Hk, D), dtype=BF16, device=cuda)
    kv = torch.stack([rnd(P, Hk, D), rnd(P, Hk, D)])
    workloads.scatter_into_cache(saved, kv, ids[:nb])
    fmt = LayerFormat(P, Hk, D, BYTE_PLANES)
    cache = torch.full_like(saved, float("nan"))
    restore_layer(pack_layer(saved, ids[:nb], fmt), fmt, cache, ids[:nb])
    x = Batch.__new__(Batch)
    x.prefix, x.bs, x.kv_first, x.Hq, x.Hk, x.D, x.dtype, x.dev = P, bs, True, Hq, Hk, D, BF16, cuda
    x.cache, x.pkv = cache, kv
    x.prefix_blocks, x.suffix_blocks = ids[:nb].int().to(cuda), ids[nb:].int()[:, None].to(cuda)
    x.new, x.query_start = [1] * B, torch.arange(B + 1, dtype=torch.int32, device=cuda)
    x.skv = [torch.empty(2, 0, Hk, D, dtype=BF16, device=cuda) for _ in range(B)]
    w = (rnd(D).float() * 0.1 + 1).to(BF16)
    for step in range(steps):
        q, k, v = (t.unflatten(1, (-1, D)) for t in rnd(B, (Hq + 2 * Hk) * D).split([Hq * D, Hk * D, Hk * D], 1))
        slots = ids[nb:].to(cuda) * bs + step
        pos = torch.full((B,), P + step, device=cuda)
        x.q = append_kv(cache, k, v, slots, query=q, positions=pos, cos_sin=table, query_weight=w, key_weight=w)
        x.suffix = [step + 1] * B
        x.suffix_lens = torch.full((B,), step + 1, dtype=torch.int32, device=cuda)
        written = cache[:, ids[nb:].to(cuda), step]
        x.skv = [torch.cat([kv_b, written[:, b:b + 1]], 1) for b, kv_b in enumerate(x.skv)]
        x.check(x.run())


@pytest.mark.parametrize("nats", [10.0, 14.0, 16.0, 17.0, 17.5, 19.0])
@pytest.mark.parametrize("spread", [0.0, 0.5])
def test_fp16_keys_far_below_one_that_stands_out(cuda, nats, spread):
    """An attention sink: the first key's score lies `nats` above all others and its value is zero, so that
    the row is made of the others' small probabilities alone; many heads, so that a CTA has it beside most
    of them. Beside the tolerance above: the kernel's fp16 probabilities have their largest at 2^9 or more,
    so one below 2^-14 is off by at most half of the smallest step, 2^-25: 2^-34 of |v| a key."""
    H, g, N, D = 80, 2, 4100, 64
    x = Batch(cuda, [1, 1], [1, 40], N, H * g, H, D, 16, F16, seed=21)
    x.q.zero_()
    x.q[..., 0] = 1
    for kv in [x.pkv, *x.skv]:
        kv[0] = 0
        kv[0, ..., 0] = torch.randn(kv.shape[1:3], device=cuda) * spread * D ** 0.5
        kv[1] += 1  # values that do not cancel
    x.pkv[0, 0, :, 0] = nats * D ** 0.5
    x.pkv[1, 0] = 0
    x.write(x.pkv, x.prefix_blocks)
    for b, kv in enumerate(x.skv):
        x.write(kv, x.suffix_blocks[b])
    out = x.run().double()
    u = torch.finfo(F16).eps / 2
    for b, kv in enumerate(x.skv):
        k, v = (t.double().transpose(0, 1) for t in torch.cat([x.pkv, kv], 1))  # [H, N, D]
        p = torch.softmax(k[..., 0] * D ** -0.5, -1)
        want, A = ((p[:, None] @ t)[:, 0].repeat_interleave(g, 0) for t in (v, v.abs()))
        err = nats * (D / 8) * 2.0 ** -22 + 2.0 ** -22 * (1 + nats)
        tol = (u + 2 * err + (k.shape[1] / 8 + 64) * 2.0 ** -23) * A + u * want.abs() + 2.0 ** -25
        tol += 2.0 ** -34 * v.abs().sum(1).repeat_interleave(g, 0)
        off = (out[b] - want).abs()
        assert bool((off <= tol).all()), (b, float((off / want.abs()).max()), float((off - tol).max()))


@pytest.mark.parametrize("k_std", [0.01, 8.0, 40.0])
def test_flat_and_peaked_scores_fp16(cuda, k_std):
    x = Batch(cuda, [1] * 20, [30 + 17 * i for i in range(20)], 3000, 16, 2, 128, 16, F16, seed=3, k_std=k_std)
    lse = torch.empty(20, 16, dtype=torch.float32, device=cuda)
    x.check(x.run(lse=lse), lse)


def test_more_requests_than_places_of_two_searches(cuda):
    """A token's request is found among over 1024, many of them without new tokens."""
    new = [(7 * i % 5) % 3 for i in range(1500)]
    x = Batch(cuda, new, [n + i % 9 for i, n in enumerate(new)], 40, 2, 1, 64, 16, BF16, seed=18)
    lse = torch.empty(sum(new), 2, dtype=torch.float32, device=cuda)
    x.check(x.run(lse=lse), lse)


def test_smallest_scale(cuda):
    """Every key of like weight: the mean of the values."""
    x = Batch(cuda, [2] * 3, [40] * 3, 200, 4, 2, 64, 16, BF16, seed=19)
    x.check(x.run(softmax_scale=1e-38), scale=1e-38)
