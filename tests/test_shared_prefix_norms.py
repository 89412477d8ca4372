"""shared_prefix_attention against the formula in 64 bits, by the norm of the difference: a lost or
stale key tile, which moves every element of a row by less than its own worst case, shows there.

Bound, derived. u is half a step of the type. The store is off by at most u of each element, so by
u of the norm. The probabilities' roundings give sum p_i d_i v_i with |d_i| <= u; the values are
random, independent of the d_i and of mean zero, so that its square has at most u^2 times the
expectation of the output's own. Both together: sqrt(2) u in the worst case, 0.6 u if the roundings
fall evenly (0.42 u each). Scores (2 (D / 8) 2^-22 scale |q||k|, about 2^-15) and sums
((N / 8 + 64) 2^-23) are off by less than 2^-12 each at these sizes, in keys of either sign: they
enter as random errors too, below 2^-13 of the norm. The bound is 1.5 u + 2^-13 of each KV head's
norm over all tokens (1024 elements and more). One lost key of N with like scores moves the norm by
about N^-1/2 of it."""
from __future__ import annotations

import math

import pytest
import torch

from test_gpu_shared_prefix import BF16, F16, Batch

CASES = [  # new, suffix, prefix, Hq, Hk, D, block size
    ([1], [5], 40000, 8, 1, 128, 16),
    ([1], [30000], 5, 8, 1, 128, 16),
    ([1, 3, 2, 5], [700, 3, 300, 250], 4099, 28, 4, 128, 32),
    ([300, 1, 77], [500, 2, 77], 2000, 16, 2, 64, 16),
    ([300, 1, 77], [500, 2, 77], 2000, 16, 2, 128, 16),
    ([2] * 100, [2 + 3 * i for i in range(100)], 1500, 8, 2, 64, 24),
    ([1] * 40, [50 * i for i in range(40)], 3001, 8, 2, 128, 5),
]
LOADS = [  # requests, Hq, Hk, D, prefix
    (64, 32, 8, 128, 16384),
    (200, 32, 8, 128, 8192),
    (96, 8, 2, 64, 20000),
]


def bound(dtype):
    return 1.5 * torch.finfo(dtype).eps / 2 + 2.0 ** -13


def formula(x, lost=0, rounded=False):
    """(out, lse) in 64 bits; with the values of `lost` prefix keys from the 1000th missing, and with the
    probabilities (of the largest, as the kernel has them) and the output rounded to the type."""
    g, at = x.Hq // x.Hk, 0
    outs, lses = [], []
    for b, (n, s) in enumerate(zip(x.new, x.suffix)):
        k, v = torch.cat([x.pkv, x.skv[b]], 1).double()
        if lost:
            v[1000:1000 + lost] = 0
        q = x.q[at:at + n].double().unflatten(1, (x.Hk, g))
        sc = torch.einsum("thgd,khd->thgk", q, k) * x.D ** -0.5
        seen = x.prefix + (s - n + 1 + torch.arange(n, device=x.dev)).clamp(min=0)
        sc = sc.masked_fill(torch.arange(k.shape[0], device=x.dev) >= seen[:, None, None, None], -math.inf)
        p = (sc - sc.amax(-1, keepdim=True)).exp()
        l = p.sum(-1, keepdim=True)
        if rounded:
            p = p.to(x.dtype).double()
        out = torch.einsum("thgk,khd->thgd", p, v) / l
        outs.append(out.to(x.dtype).double() if rounded else out)
        lses.append(torch.logsumexp(sc, -1).flatten(1))
        at += n
    return torch.cat(outs), torch.cat(lses)  # [T, Hk, g, D], [T, Hq]


def off(out, want):
    """Norm of the difference over the norm, the largest of the KV heads."""
    d = (out.double().reshape(want.shape) - want).transpose(0, 1).flatten(1).norm(dim=1)
    return float((d / want.transpose(0, 1).flatten(1).norm(dim=1)).max())


@pytest.mark.parametrize("dtype", [BF16, F16])
def test_the_bound_takes_the_roundings_and_no_lost_keys(dtype):
    """(on the CPU, in the formula)"""
    x = Batch(torch.device("cpu"), [1] * 4, [1, 30, 50, 7], 16384, 8, 2, 64, 16, dtype, seed=1)
    want, _ = formula(x)
    assert off(formula(x, rounded=True)[0], want) < 0.7 * bound(dtype)
    for lost in (2, 16, 128):
        assert off(formula(x, lost=lost)[0], want) > bound(dtype), lost


def check(x, repeats=0):
    flags = torch.zeros(1, dtype=torch.int32, device=x.dev)
    lse = torch.empty(sum(x.new), x.Hq, device=x.dev)
    out = x.run(lse=lse, error_flags=flags)
    want, z = formula(x)
    assert off(out, want) < bound(x.dtype)
    N = x.prefix + max(x.suffix)
    e = float(x.q.double().norm(dim=-1).max() * max(float(kv[0].double().norm(dim=-1).max()) for kv in [x.pkv, *x.skv] if kv.numel()))
    e *= x.D ** -0.5 * (x.D / 8) * 2.0 ** -22
    assert bool(((lse - z).abs() <= e + (N / 8 + 64) * 2.0 ** -23 + 2.0 ** -21 * (1 + z.abs())).all())
    for _ in range(repeats):
        again = torch.empty_like(lse)
        assert torch.equal(x.run(lse=again, error_flags=flags), out) and torch.equal(again, lse)
    assert int(flags) == 0


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [BF16, F16])
@pytest.mark.parametrize("case", range(len(CASES)))
def test_norm_of_the_difference(cuda, case, dtype):
    check(Batch(cuda, *CASES[case], dtype, kv_first=case % 2 == 0, seed=30 + case))


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [BF16, F16])
@pytest.mark.parametrize("B, Hq, Hk, D, prefix", LOADS)
def test_under_load(cuda, B, Hq, Hk, D, prefix, dtype):
    """Segments of every kind in every CTA with the memory busy: no key tile lost, the same bits each time."""
    check(Batch(cuda, [1] * B, [1 + 37 * i % 700 for i in range(B)], prefix, Hq, Hk, D, 16, dtype, seed=B), repeats=10)
