"""The decode-step operators around the paged KV cache, as they are measured.

    norm_rope                norms of queries and keys for each head, with the position
                             rotation in the same pass
    append_kv                keys and values of new tokens written into a paged cache, keys
                             (and queries) normed and rotated on the way
    shared_prefix_attention  attention of a ragged batch of new tokens over a prefix that all
                             its requests share (computed once for all rows) and each
                             request's own paged suffix

`run` computes them in plain torch operations in 32 bits when `own` is false, and through
this package when it is true. Shapes are those of the package's workloads (Llama-3-8B-shaped:
32 query / 8 KV heads of 128; Qwen2-7B-shaped: 28 / 4; 70B-shaped: 64 / 8 in blocks of 32) or
generic ones.
"""
from __future__ import annotations

import math
import random

import torch

own = False

MAX_POS = 131072  # rows of the rotation table
EPS = 1e-6
DTYPES = {"bf16": torch.bfloat16, "fp16": torch.float16, "fp32": torch.float32}


# ------------------------------------------------------------------------------- cases
def listed():
    return [
        # one new token of one request: the launch is what counts
        dict(name="norm_rope_one_token", op="norm_rope", tokens=1, q_heads=32, kv_heads=8, head_dim=128, rotary=128,
             interleaved=False, norm=True, dtype="bf16", packed=True),
        # a mid-sized chunk in 32 bits, half of each head rotated in neighbouring pairs, separate tensors
        dict(name="norm_rope_chunk_fp32", op="norm_rope", tokens=1531, q_heads=16, kv_heads=4, head_dim=64, rotary=32,
             interleaved=True, norm=True, dtype="fp32", packed=False),
        # a long prompt's queries and keys as slices of the fused projection's output
        dict(name="norm_rope_prompt", op="norm_rope", tokens=16384, q_heads=32, kv_heads=8, head_dim=128, rotary=128,
             interleaved=False, norm=True, dtype="bf16", packed=True),
        # one decode step of one request
        dict(name="append_one_token", op="append_kv", tokens=1, pad=0, q_heads=32, kv_heads=8, head_dim=128, rotary=128,
             interleaved=False, norm=False, dtype="bf16", packed=True, block_size=16, kv_first=True),
        # a decode step of a batch padded to a captured size, 7 query heads a KV head, fp16, blocks of 32
        dict(name="append_padded_batch", op="append_kv", tokens=256, pad=17, q_heads=28, kv_heads=4, head_dim=128,
             rotary=128, interleaved=False, norm=True, dtype="fp16", packed=False, block_size=32, kv_first=False),
        # a 32768-token prompt of the default benchmark's request
        dict(name="append_prompt", op="append_kv", tokens=32768, pad=0, q_heads=32, kv_heads=8, head_dim=128, rotary=128,
             interleaved=False, norm=True, dtype="bf16", packed=True, block_size=16, kv_first=True),
        # two requests that have just begun behind a short system prompt
        dict(name="shared_two_short", op="shared_prefix_attention", requests=2, q_len=1, prefix=512, suffix_min=1,
             suffix_max=40, q_heads=32, kv_heads=8, head_dim=128, block_size=16, kv_first=True, dtype="bf16", lse=False),
        # drafted tokens: one to five new tokens a request, a prefix that ends inside a page, some empty suffixes
        dict(name="shared_drafted_fp16", op="shared_prefix_attention", requests=17, q_len=5, prefix=4099, suffix_min=0,
             suffix_max=700, q_heads=28, kv_heads=4, head_dim=128, block_size=32, kv_first=False, dtype="fp16", lse=True),
        # chunks of prompts behind a shared prefix, heads of 64
        dict(name="shared_chunks_d64", op="shared_prefix_attention", requests=13, q_len=300, prefix=2000, suffix_min=0,
             suffix_max=900, q_heads=16, kv_heads=2, head_dim=64, block_size=16, kv_first=True, dtype="bf16", lse=False),
        # a serving batch over a 32768-token prefix
        dict(name="shared_batch_64", op="shared_prefix_attention", requests=64, q_len=1, prefix=32768, suffix_min=64,
             suffix_max=1024, q_heads=32, kv_heads=8, head_dim=128, block_size=16, kv_first=True, dtype="bf16", lse=False),
        # a few requests over a very long document, 70B-shaped heads
        dict(name="shared_document", op="shared_prefix_attention", requests=8, q_len=1, prefix=131072, suffix_min=1,
             suffix_max=4096, q_heads=64, kv_heads=8, head_dim=128, block_size=32, kv_first=True, dtype="fp16", lse=True),
        # a large decode batch: 1024 query rows a KV head, the products are what counts
        dict(name="shared_batch_256", op="shared_prefix_attention", requests=256, q_len=1, prefix=32768, suffix_min=16,
             suffix_max=256, q_heads=32, kv_heads=8, head_dim=128, block_size=16, kv_first=True, dtype="bf16", lse=False),
    ]


def _log_int(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    op = rng.choice(["norm_rope", "append_kv", "shared_prefix_attention", "shared_prefix_attention"])
    kv_heads = rng.choice([1, 2, 4, 8])
    group = rng.choice([1, 2, 4, 5, 7, 8])
    if op != "shared_prefix_attention":
        head_dim = rng.choice([64, 80, 96, 128, 256])
        rotary = rng.choice([head_dim, head_dim, head_dim // 2])
        heads = kv_heads * (group + 2)
        most = min(32768, 32768 * 48 * 128 // (heads * head_dim))
        case = dict(op=op, tokens=_log_int(rng, 1, most), q_heads=kv_heads * group, kv_heads=kv_heads, head_dim=head_dim,
                    rotary=rotary, interleaved=rng.random() < 0.3, norm=rng.random() < 0.6,
                    dtype=rng.choice(["bf16", "bf16", "fp16", "fp32"] if op == "norm_rope" else ["bf16", "bf16", "fp16"]),
                    packed=rng.random() < 0.5)
        if case["dtype"] == "fp32":
            case["tokens"] = max(1, case["tokens"] // 2)
        if op == "append_kv":
            case.update(pad=rng.randrange(0, case["tokens"]) // 4, block_size=rng.choice([8, 16, 16, 32, 48]),
                        kv_first=rng.random() < 0.6)
        return case
    head_dim = rng.choice([64, 128, 128])
    requests = _log_int(rng, 1, 256)
    q_len = rng.choice([1, 1, 1, 2, 4, 16, 128])
    prefix = _log_int(rng, 1, 65536)
    suffix_max = _log_int(rng, 1, 4096)
    # no more query rows a pass, cached rows or products than the largest listed case has
    requests = max(1, min(requests, 1024 // (q_len * group), 65536 // suffix_max))
    prefix = max(1, min(prefix, 32768 * 8192 // (requests * q_len * group * kv_heads) - suffix_max))
    return dict(op=op, requests=requests, q_len=q_len, prefix=prefix, suffix_min=rng.randrange(0, suffix_max + 1),
                suffix_max=suffix_max, q_heads=kv_heads * group, kv_heads=kv_heads, head_dim=head_dim,
                block_size=rng.choice([8, 16, 16, 32, 48]), kv_first=rng.random() < 0.6,
                dtype=rng.choice(["bf16", "fp16"]), lse=rng.random() < 0.5)


# ------------------------------------------------------------------------------ inputs
def _lengths(case):
    """New tokens and suffix keys of each request (the same for every seed of a case)."""
    rng = random.Random(case["requests"] * 1000003 + case["prefix"] * 101 + case["suffix_max"])
    new, suffix = [], []
    for _ in range(case["requests"]):
        n = rng.randint(1, case["q_len"])
        s = rng.randint(case["suffix_min"], case["suffix_max"])
        # a chunk's own keys are in its suffix; an empty suffix (attention to the prefix alone) stays for single tokens
        if n > 1 or s > 0:
            s = max(s, n)
        new.append(n)
        suffix.append(s)
    return new, suffix


def _generator(seed):
    return torch.Generator(device="cuda").manual_seed(seed)


def _normal(g, shape, dtype, std=1.0):
    return (torch.randn(shape, generator=g, device="cuda") * std).to(dtype)


def _rotation_table(rotary):
    """cos | sin of position * 10000^(-2i / rotary), angles in 64 bits."""
    inv = 10000.0 ** (-torch.arange(0, rotary, 2, dtype=torch.float64, device="cuda") / rotary)
    ang = torch.arange(MAX_POS, dtype=torch.float64, device="cuda")[:, None] * inv[None, :]
    return torch.cat([ang.cos(), ang.sin()], 1).float()


def prepare(case, seed):
    g = _generator(seed)
    dt = DTYPES[case["dtype"]]
    hq, hk, d = case["q_heads"], case["kv_heads"], case["head_dim"]
    st = dict(case=case)
    if case["op"] != "shared_prefix_attention":
        t = case["tokens"]
        # activations with some strong channels, as a projection gives them
        gain = torch.exp(torch.randn((hq + 2 * hk) * d, generator=g, device="cuda"))
        qkv = (torch.randn((t, (hq + 2 * hk) * d), generator=g, device="cuda") * gain).to(dt)
        q, k, v = (x.view(t, -1, d) for x in qkv.split([hq * d, hk * d, hk * d], 1))
        if not case["packed"]:
            q, k, v = q.contiguous(), k.contiguous(), v.contiguous()
        st.update(q=q, k=k, v=v, table=_rotation_table(case["rotary"]))
        start = torch.randint(0, MAX_POS - t, (1,), generator=g, device="cuda")
        if t > 1024:  # a prompt's consecutive positions; else a step of unrelated requests
            st["positions"] = torch.arange(t, device="cuda") + start
        else:
            st["positions"] = torch.randint(0, MAX_POS, (t,), generator=g, device="cuda")
        st["qw"] = st["kw"] = None
        if case["norm"]:
            st["qw"] = _normal(g, (d,), torch.float32, 0.2).add(1).to(dt)
            st["kw"] = _normal(g, (d,), torch.float32, 0.2).add(1).to(dt)
        if case["op"] == "append_kv":
            bs = case["block_size"]
            n = t - case["pad"]
            blocks = (t + bs - 1) // bs + 3 if t > 1024 else t + 3
            ids = torch.randperm(blocks, generator=g, device="cuda")
            i = torch.arange(n, device="cuda")
            if t > 1024:
                slots = ids[i // bs] * bs + i % bs
            else:  # each request writes one row of a block of its own
                slots = ids[:n] * bs + torch.randint(0, bs, (n,), generator=g, device="cuda")
            st["slots"] = torch.cat([slots, torch.full((case["pad"],), -1, dtype=torch.int64, device="cuda")])
            shape = (2, blocks, bs, hk, d) if case["kv_first"] else (blocks, 2, bs, hk, d)
            st["cache"] = _normal(g, shape, dt)
            st["written"] = n
        return st
    new, suffix = _lengths(case)
    bs, b = case["block_size"], case["requests"]
    pre_blocks = (case["prefix"] + bs - 1) // bs
    own_blocks = [(s + bs - 1) // bs for s in suffix]
    width = max(1, max(own_blocks))
    blocks = pre_blocks + sum(own_blocks) + 3
    shape = (2, blocks, bs, hk, d) if case["kv_first"] else (blocks, 2, bs, hk, d)
    cache = torch.randn(shape, generator=g, device="cuda", dtype=torch.float32 if blocks * bs * hk * d < 1 << 26 else dt)
    gain = torch.exp(torch.empty(hk, d, device="cuda").uniform_(math.log(0.5), math.log(2.0), generator=g))
    kv = (cache if case["kv_first"] else cache.transpose(0, 1))
    kv[0].mul_(gain * 1.4)  # keys: scores of a few units, so that some keys stand out
    kv[1].mul_(0.5)
    st["cache"] = cache.to(dt)
    st["q"] = _normal(g, (sum(new), hq, d), dt, 1.2)
    ids = torch.randperm(blocks, generator=g, device="cuda").to(torch.int32)
    st["prefix_blocks"] = ids[:pre_blocks].contiguous()
    table = torch.zeros((b, width), dtype=torch.int32)
    at = pre_blocks
    ids_host = ids.cpu()
    for r, m in enumerate(own_blocks):
        table[r, :m] = ids_host[at:at + m]
        at += m
    st["suffix_blocks"] = table.cuda()
    st["suffix_lens"] = torch.tensor(suffix, dtype=torch.int32, device="cuda")
    starts = [0]
    for n in new:
        starts.append(starts[-1] + n)
    st["query_start"] = torch.tensor(starts, dtype=torch.int32, device="cuda")
    st["max_new"] = max(new)
    st["scale"] = d ** -0.5
    return st


# ------------------------------------------------------------------------------- plain
def _norm_rotate(x, weight, st):
    x = x.float()
    if weight is not None:
        x = x * torch.rsqrt(x.pow(2).mean(-1, keepdim=True) + EPS) * weight.float()
    rot = st["case"]["rotary"]
    cs = st["table"][st["positions"]][:, None, :]
    c, s = cs[..., :rot // 2], cs[..., rot // 2:]
    y = x.clone()
    if st["case"]["interleaved"]:
        a, b = x[..., 0:rot:2], x[..., 1:rot:2]
        y[..., 0:rot:2] = a * c - b * s
        y[..., 1:rot:2] = b * c + a * s
    else:
        a, b = x[..., :rot // 2], x[..., rot // 2:rot]
        y[..., :rot // 2] = a * c - b * s
        y[..., rot // 2:rot] = b * c + a * s
    return y


def _rows(cache, kv_first, which, blocks, offsets):
    return cache[which, blocks, offsets] if kv_first else cache[blocks, which, offsets]


def _softmax_parts(scores, values):
    """Running maximum, sum and weighted values of a masked score matrix."""
    m = scores.amax(-1, keepdim=True)
    p = torch.exp(scores - torch.where(m == -math.inf, torch.zeros_like(m), m))
    return m, p.sum(-1, keepdim=True), p @ values


def _attend_plain(st):
    case = st["case"]
    hq, hk, d, bs, n_pre = case["q_heads"], case["kv_heads"], case["head_dim"], case["block_size"], case["prefix"]
    g = hq // hk
    q = st["q"].float()
    t = q.shape[0]
    dev = q.device
    i = torch.arange(n_pre, device=dev)
    pb = st["prefix_blocks"].long()[i // bs]
    rows = q.view(t, hk, g, d).permute(1, 0, 2, 3).reshape(hk, t * g, d)
    k = _rows(st["cache"], case["kv_first"], 0, pb, i % bs).float().permute(1, 2, 0)
    v = _rows(st["cache"], case["kv_first"], 1, pb, i % bs).float().permute(1, 0, 2)
    mp, lp, op = _softmax_parts(rows @ k * st["scale"], v)
    mp, lp, op = (x.view(hk, t, g, -1).permute(1, 0, 2, 3) for x in (mp, lp, op))
    # suffixes: padded to the longest, queries padded to the most new tokens
    starts = st["query_start"].long()
    new = starts[1:] - starts[:-1]
    lens = st["suffix_lens"].long()
    b, width, mq = new.shape[0], st["suffix_blocks"].shape[1] * bs, st["max_new"]
    j = torch.arange(mq, device=dev)
    tok = (starts[:-1, None] + j[None]).clamp(max=t - 1)
    i = torch.arange(width, device=dev)
    sb = st["suffix_blocks"].long()[:, i // bs]
    k = _rows(st["cache"], case["kv_first"], 0, sb, (i % bs)[None].expand_as(sb)).float().permute(0, 2, 3, 1)
    v = _rows(st["cache"], case["kv_first"], 1, sb, (i % bs)[None].expand_as(sb)).float().permute(0, 2, 1, 3)
    qs = q.view(t, hk, g, d)[tok].permute(0, 2, 1, 3, 4).reshape(b, hk, mq * g, d)
    seen = (lens - new)[:, None] + j[None] + 1  # keys that new token j sees
    mask = i[None, None] < torch.minimum(seen, lens[:, None])[:, :, None]
    mask = mask[:, None, :, None].expand(b, hk, mq, g, width).reshape(b, hk, mq * g, width)
    s = torch.where(mask, qs @ k * st["scale"], torch.full((), -math.inf, device=dev))
    ms, ls, os = _softmax_parts(s, v)
    r = torch.searchsorted(starts, torch.arange(t, device=dev), right=True) - 1
    jj = torch.arange(t, device=dev) - starts[r]
    ms, ls, os = (x.view(b, hk, mq, g, -1)[r, :, jj] for x in (ms, ls, os))
    m = torch.maximum(mp, ms)
    wp, ws = torch.exp(mp - m), torch.exp(ms - m)
    total = lp * wp + ls * ws
    out = {"out": ((op * wp + os * ws) / total).reshape(t, hq, d).to(st["q"].dtype)}
    if case["lse"]:
        out["lse"] = (m + total.log()).reshape(t, hq)
    return out


def run(state):
    case = state["case"]
    if own:
        return _run_own(state)
    if case["op"] == "shared_prefix_attention":
        return _attend_plain(state)
    q = _norm_rotate(state["q"], state["qw"], state).to(state["q"].dtype)
    k = _norm_rotate(state["k"], state["kw"], state).to(state["k"].dtype)
    if case["op"] == "norm_rope":
        return {"query": q, "key": k}
    n, bs = state["written"], case["block_size"]
    b, o = state["slots"][:n] // bs, state["slots"][:n] % bs
    if case["kv_first"]:
        state["cache"][0, b, o] = k[:n]
        state["cache"][1, b, o] = state["v"][:n]
    else:
        state["cache"][b, 0, o] = k[:n]
        state["cache"][b, 1, o] = state["v"][:n]
    return {"query": q, "cache": state["cache"]}


def _run_own(state):
    from origami_b200.append import append_kv, norm_rope
    from origami_b200.shared_prefix import shared_prefix_attention

    case = state["case"]
    if case["op"] == "norm_rope":
        q, k = norm_rope(state["q"], state["k"], state["positions"], state["table"], query_weight=state["qw"],
                         key_weight=state["kw"], eps=EPS, interleaved=case["interleaved"])
        return {"query": q, "key": k}
    if case["op"] == "append_kv":
        q = append_kv(state["cache"], state["k"], state["v"], state["slots"], query=state["q"],
                      positions=state["positions"], cos_sin=state["table"], query_weight=state["qw"],
                      key_weight=state["kw"], eps=EPS, interleaved=case["interleaved"])
        return {"query": q, "cache": state["cache"]}
    lse = None
    if case["lse"]:
        lse = torch.empty(state["q"].shape[:2], dtype=torch.float32, device="cuda")
    out = shared_prefix_attention(state["q"], state["cache"], state["query_start"], state["prefix_blocks"],
                                  case["prefix"], state["suffix_blocks"], state["suffix_lens"],
                                  softmax_scale=state["scale"], lse=lse)
    return {"out": out, "lse": lse} if case["lse"] else {"out": out}


# ------------------------------------------------------------------------------- exact
def _exact_rows(x, weight, case, st):
    """Each pair as a complex number times e^(i angle), the angle's cosine and sine as the table gives them."""
    x = x.double()
    if weight is not None:
        x = x / (x.square().sum(-1, keepdim=True) / x.shape[-1] + EPS).sqrt() * weight.double()
    rot = case["rotary"]
    turn = st["table"].double().index_select(0, st["positions"])
    turn = torch.complex(turn[:, :rot // 2].contiguous(), turn[:, rot // 2:].contiguous()).unsqueeze(1)
    head, tail = x[..., :rot], x[..., rot:]
    if case["interleaved"]:
        pairs = head.unflatten(-1, (rot // 2, 2))
    else:
        pairs = head.unflatten(-1, (2, rot // 2)).transpose(-1, -2)
    z = torch.view_as_real(torch.view_as_complex(pairs.contiguous()) * turn)
    head = z.flatten(-2) if case["interleaved"] else z.transpose(-1, -2).flatten(-2)
    return torch.cat([head, tail], -1)


def exact(case, seed):
    st = prepare(case, seed)
    if case["op"] == "norm_rope":
        return {"query": _exact_rows(st["q"], st["qw"], case, st), "key": _exact_rows(st["k"], st["kw"], case, st)}
    if case["op"] == "append_kv":
        key = _exact_rows(st["k"], st["kw"], case, st)
        cache = st["cache"].double()
        by_kv = cache if case["kv_first"] else cache.transpose(0, 1)
        bs, n = case["block_size"], st["written"]
        flat = torch.stack([st["slots"][:n] // bs, st["slots"][:n] % bs])
        by_kv[0].index_put_(tuple(flat), key[:n])
        by_kv[1].index_put_(tuple(flat), st["v"][:n].double())
        return {"query": _exact_rows(st["q"], st["qw"], case, st), "cache": cache}
    hq, hk, d, bs = case["q_heads"], case["kv_heads"], case["head_dim"], case["block_size"]
    g, n_pre = hq // hk, case["prefix"]
    new, suffix = _lengths(case)
    cache = st["cache"] if case["kv_first"] else st["cache"].transpose(0, 1)

    def keys_values(ids, n):  # [2, hk, n, d] in 64 bits
        x = cache.index_select(1, ids.long()).flatten(1, 2)[:, :n]
        return x.permute(0, 2, 1, 3).double()

    pk, pv = keys_values(st["prefix_blocks"], n_pre)
    out = torch.empty(st["q"].shape, dtype=torch.float64, device="cuda")
    lse = torch.empty(st["q"].shape[:2], dtype=torch.float64, device="cuda")
    at = 0
    for r in range(case["requests"]):
        n, s = new[r], suffix[r]
        q = st["q"][at:at + n].double().unflatten(1, (hk, g)).permute(1, 0, 2, 3).flatten(1, 2)  # [hk, n * g, d]
        sc = q @ pk.transpose(1, 2)
        sk, sv = keys_values(st["suffix_blocks"][r, :(s + bs - 1) // bs], s)
        own_sc = q @ sk.transpose(1, 2)
        for j in range(n):
            own_sc[:, j * g:(j + 1) * g, s - n + j + 1:] = -math.inf
        sc = torch.cat([sc, own_sc], 2) * st["scale"]
        z = torch.logsumexp(sc, -1)
        p = (sc - z.unsqueeze(-1)).exp()
        o = p[..., :n_pre] @ pv + p[..., n_pre:] @ sv
        out[at:at + n] = o.unflatten(1, (n, g)).permute(1, 0, 2, 3).flatten(1, 2)
        lse[at:at + n] = z.unflatten(1, (n, g)).permute(1, 0, 2).flatten(1, 2)
        at += n
    return {"out": out, "lse": lse} if case["lse"] else {"out": out}


# -------------------------------------------------------------------------------- work
def work(case):
    size = 4 if case["dtype"] == "fp32" else 2
    hq, hk, d = case["q_heads"], case["kv_heads"], case["head_dim"]
    if case["op"] != "shared_prefix_attention":
        t = case["tokens"]
        small = t * (case["rotary"] * 4 + 8) + (2 * d * size if case["norm"] else 0)
        flops = t * (hq + hk) * (3 * case["rotary"] + (4 * d if case["norm"] else 0))
        if case["op"] == "norm_rope":
            return {"bytes": 2 * t * (hq + hk) * d * size + small, "flops": flops}
        n = t - case["pad"]
        return {"bytes": 2 * (t * hq + 2 * n * hk) * d * size + small + t * 8, "flops": flops}
    new, suffix = _lengths(case)
    t, bs = sum(new), case["block_size"]
    cached = case["prefix"] + sum(suffix)
    pairs = t * case["prefix"] + sum(sum(max(0, min(s, s - n + j + 1)) for j in range(n)) for n, s in zip(new, suffix))
    small = 4 * ((case["prefix"] + bs - 1) // bs + sum((s + bs - 1) // bs for s in suffix) + 2 * len(new) + 1)
    return {"bytes": 2 * cached * hk * d * size + 2 * t * hq * d * size + small + (t * hq * 4 if case["lse"] else 0),
            "flops": 4 * pairs * hq * d}
