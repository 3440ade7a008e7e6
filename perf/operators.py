"""Operators of the serving path around the paged key-value cache, case by case: what fills the cache and what reads it.

Kinds of case
  store    ``glue.qk_norm_rope_kv_store``: RMS norm of every query and key head, position rotation, rows into the cache
  decode   ``attention.paged_decode_attention``: one new token per request over the pages of its context
  prefill  ``attention.paged_prefill_attention``: the new tokens of every request (whole prompts, chunks of them, a few
           tokens behind a long context) over the pages of its context

Both attentions are causal, over everything, or over a sliding window of the last keys plus a few first ones. A request's
lengths are drawn from the case alone (``_lens``), its values from the seed. Heads are those of this repository's
configurations (16 / 2 of 64, 16 / 2 of 128, 32 / 8 of 128) and, where drawn, other common groupings.
"""

from __future__ import annotations

import math
import random

import torch

#: False: `run` computes the plain forms; True: it calls the package's operators
own = False

DTYPES = {"bf16": torch.bfloat16, "fp16": torch.float16}
EPS = 1e-6
ROPE_THETA = 10000.0


def listed():
    return [
        # one token of one user on its way into the cache: nothing but latency
        dict(name="store_1tok", kind="store", B=1, lo=1, hi=1, heads=16, kv_heads=2, dim=64, page=256, dtype="bf16"),
        # a full prefill batch of the wide decoder: 16 prompts that fill 8192 rows
        dict(name="store_8192tok_wide", kind="store", B=16, lo=512, hi=512, heads=32, kv_heads=8, dim=128, page=256, dtype="bf16"),
        # a ragged handful of prompts in half precision, small pages
        dict(name="store_ragged_fp16", kind="store", B=5, lo=17, hi=150, heads=16, kv_heads=2, dim=128, page=16, dtype="fp16"),
        # one user, a few hundred tokens: latency
        dict(name="decode_1req", kind="decode", B=1, lo=333, hi=333, heads=16, kv_heads=2, dim=64, page=256, dtype="bf16",
             window=0, sinks=0, lse=False),
        # a decode step of 64 concurrent requests with ragged contexts
        dict(name="decode_64req", kind="decode", B=64, lo=128, hi=1024, heads=16, kv_heads=2, dim=64, page=256, dtype="bf16",
             window=0, sinks=0, lse=False),
        # long contexts of the wide decoder, in small pages
        dict(name="decode_48req_long_wide", kind="decode", B=48, lo=500, hi=8192, heads=32, kv_heads=8, dim=128, page=16,
             dtype="bf16", window=0, sinks=0, lse=False),
        # one long conversation alone on the card: all parallelism is in the context's length; half precision, with the
        # log of the sum that a caller needs to join it with a part attended elsewhere
        dict(name="decode_1req_100k_fp16", kind="decode", B=1, lo=100003, hi=100003, heads=32, kv_heads=8, dim=128, page=256,
             dtype="fp16", window=0, sinks=0, lse=True),
        # streaming requests: window of 1024 keys and 4 first ones, the pages between given back to the allocator
        dict(name="decode_128req_window", kind="decode", B=128, lo=3, hi=12000, heads=16, kv_heads=2, dim=128, page=16,
             dtype="bf16", window=1024, sinks=4, lse=False),
        # one short prompt: latency
        dict(name="prefill_37tok", kind="prefill", B=1, lo=37, hi=37, before=0, heads=16, kv_heads=2, dim=64, page=256,
             dtype="bf16", window=0, sinks=0, lse=False),
        # a prefill batch of ragged prompts, causal
        dict(name="prefill_12prompts", kind="prefill", B=12, lo=101, hi=1200, before=0, heads=16, kv_heads=2, dim=64, page=256,
             dtype="bf16", window=0, sinks=0, lse=False),
        # a long prompt of a streaming request in half precision: window of 1024 and 4 first tokens
        dict(name="prefill_8001tok_window_fp16", kind="prefill", B=1, lo=8001, hi=8001, before=0, heads=16, kv_heads=2, dim=128,
             page=16, dtype="fp16", window=1024, sinks=4, lse=False),
        # a chunk of 4096 tokens of a long prompt whose first 12 thousand tokens are in the cache: the most arithmetic
        dict(name="prefill_chunk_wide", kind="prefill", B=1, lo=4096, hi=4096, before=12288, heads=32, kv_heads=8, dim=128, page=256,
             dtype="bf16", window=0, sinks=0, lse=True),
    ]


HEADS = [(16, 2, 64), (16, 2, 128), (32, 8, 128), (8, 8, 64), (12, 4, 64), (14, 2, 64), (24, 8, 64), (16, 1, 128)]


def draw(rng):
    def spread(lo, hi):  # evenly over the logarithm
        return min(hi, max(lo, round(math.exp(rng.uniform(math.log(lo), math.log(hi))))))

    kind = rng.choice(["store", "decode", "decode", "prefill", "prefill"])
    heads, kv_heads, dim = rng.choice(HEADS)
    case = dict(kind=kind, heads=heads, kv_heads=kv_heads, dim=dim, page=rng.choice([8, 16, 32, 48, 64, 128, 256]),
                dtype=rng.choice(["bf16", "bf16", "fp16"]))
    if kind == "store":
        B = spread(1, 64)
        hi = spread(1, max(1, 8192 // B))
        return dict(case, B=B, lo=rng.randint(1, hi), hi=hi)
    window = rng.choice([0, 0, spread(1, 4096)])
    case.update(window=window, sinks=rng.choice([0, 1, 4, spread(1, 300)]) if window else 0, lse=rng.random() < 0.3)
    if kind == "decode":
        B = spread(1, 256)
        hi = spread(1, min(100000, 400000 // B))
        return dict(case, B=B, lo=rng.randint(1, hi), hi=hi)
    B = spread(1, 32)
    hi = spread(1, max(1, 8192 // B))
    return dict(case, B=B, lo=rng.randint(1, hi), hi=hi, before=rng.choice([0, 0, spread(1, 8192 if B * hi <= 4096 else 2048)]))


# ------------------------------------------------------------------------------------------------ lengths and tables
def _lens(case):
    """(new tokens, context with them) of every request."""
    rng = random.Random("%(B)d %(lo)d %(hi)d" % case)
    new = [rng.randint(case["lo"], case["hi"]) for _ in range(case["B"])]
    if case["kind"] == "decode":
        return [1] * case["B"], new
    before = case.get("before", 0)
    return new, [n + (before if case["B"] == 1 else rng.randint(0, before)) for n in new]


def _visible(case, pos):
    """Number of keys that a token at `pos` sees."""
    window = case.get("window", 0)
    first = max(0, pos - window + 1) if window else 0
    return pos + 1 - first + min(first, case.get("sinks", 0))


def _first_kept(case, n, c):
    """First key behind the sinks that the `n` last tokens of a context of `c` see."""
    return max(0, c - n - case["window"] + 1) if case.get("window", 0) else 0


def work(case):
    new, ctx = _lens(case)
    T, row = sum(new), case["dim"] * 2
    if case["kind"] == "store":
        rows = T * (case["heads"] + 2 * case["kv_heads"])
        return {"bytes": 2 * rows * row + max(ctx) * case["dim"] * 4 + 12 * T + 2 * row, "flops": 10 * rows * case["dim"]}
    keys = pairs = 0
    for n, c in zip(new, ctx):
        first = _first_kept(case, n, c)
        keys += c - first + min(first, case["sinks"])
        pairs += sum(_visible(case, p) for p in range(c - n, c))
    return {"bytes": 2 * keys * case["kv_heads"] * row + 2 * T * case["heads"] * row + (4 * T * case["heads"] if case["lse"] else 0),
            "flops": 4 * pairs * case["heads"] * case["dim"]}


def prepare(case, seed):
    dev, dt = torch.device("cuda"), DTYPES[case["dtype"]]
    gen = torch.Generator(device=dev).manual_seed(seed)
    host = random.Random(seed)
    new, ctx = _lens(case)
    T, B, page = sum(new), case["B"], case["page"]
    heads, kv_heads, dim = case["heads"], case["kv_heads"], case["dim"]

    def normal(*shape, scale=1.0):
        return torch.randn(*shape, device=dev, dtype=dt, generator=gen) * scale

    width = max(-(-c // page) for c in ctx)
    n_blocks = sum(-(-c // page) for c in ctx) + 3
    order = torch.randperm(n_blocks, device=dev, generator=gen).tolist()
    tables, slots, positions = [], [], []
    for n, c in zip(new, ctx):
        pages = [order.pop() for _ in range(-(-c // page))]
        positions += range(c - n, c)
        slots += [pages[p // page] * page + p % page for p in range(c - n, c)]
        first, sinks = _first_kept(case, n, c), case.get("sinks", 0)
        # pages that no token of the step sees any more have gone back to the allocator
        kept = [b if i * page < sinks or (i + 1) * page > first else -1 for i, b in enumerate(pages)]
        tables.append(kept + [-1] * (width - len(kept)))
    cu = [0]
    for n in new:
        cu.append(cu[-1] + n)
    state = dict(case=case, k_cache=normal(n_blocks, page, kv_heads, dim), v_cache=normal(n_blocks, page, kv_heads, dim),
                 block_tables=torch.tensor(tables, dtype=torch.int32, device=dev),
                 context_lens=torch.tensor(ctx, dtype=torch.int32, device=dev),
                 cu_seqlens=torch.tensor(cu, dtype=torch.int32, device=dev), max_new=max(new), max_context=max(ctx),
                 scale=dim ** -0.5)
    if case["kind"] == "store":
        # what a qkv projection leaves, heads of very different magnitude among it
        size = torch.exp(torch.randn(heads + 2 * kv_heads, 1, device=dev, generator=gen)).to(dt)
        state["qkv"] = (normal(T, heads + 2 * kv_heads, dim) * size).view(T, -1)
        state["q_weight"] = (1 + 0.2 * torch.randn(dim, device=dev, generator=gen)).to(dt)
        state["k_weight"] = (1 + 0.2 * torch.randn(dim, device=dev, generator=gen)).to(dt)
        inv = ROPE_THETA ** (-torch.arange(0, dim, 2, dtype=torch.float64) / dim)
        angles = torch.outer(torch.arange(max(ctx), dtype=torch.float64), inv).to(dev)
        state["cos"], state["sin"] = angles.cos().float(), angles.sin().float()
        state["positions"] = torch.tensor(positions, dtype=torch.int64, device=dev)
        state["slot_mapping"] = torch.tensor(slots, dtype=torch.int32, device=dev)
        state["q"] = torch.empty(T, heads, dim, device=dev, dtype=dt)
    else:
        # normed heads: scores of a spread of one to three, so that attention is neither flat nor on a single key
        state["q"] = normal(T, heads, dim, scale=1.0 + 2.0 * host.random())
    return state


# --------------------------------------------------------------------------------------------------------- plain forms
def _norm_rotate(x, weight, cos, sin):
    x = x * torch.rsqrt((x * x).mean(-1, keepdim=True) + EPS) * weight
    a, b = x.chunk(2, dim=-1)
    return torch.cat((a * cos - b * sin, b * cos + a * sin), dim=-1)


def _plain_store(s):
    c = s["case"]
    T, heads, kv_heads, dim = s["qkv"].size(0), c["heads"], c["kv_heads"], c["dim"]
    q, k, v = s["qkv"].view(T, -1, dim).split([heads, kv_heads, kv_heads], dim=1)
    cos, sin = s["cos"][s["positions"]].unsqueeze(1), s["sin"][s["positions"]].unsqueeze(1)
    s["q"].copy_(_norm_rotate(q.float(), s["q_weight"].float(), cos, sin))
    at = s["slot_mapping"].long()
    s["k_cache"].view(-1, kv_heads, dim)[at] = _norm_rotate(k.float(), s["k_weight"].float(), cos, sin).to(s["q"].dtype)
    s["v_cache"].view(-1, kv_heads, dim)[at] = v


def _plain_attention(s):
    """All requests side by side, padded to the longest: scores of every (token, key) pair, masked, in 32 bits."""
    c, q = s["case"], s["q"]
    page, kv_heads, dim, dev = c["page"], c["kv_heads"], c["dim"], q.device
    cu, ctx = s["cu_seqlens"].long(), s["context_lens"].long()
    new = cu[1:] - cu[:-1]
    key = torch.arange(s["max_context"], device=dev)
    rows = s["block_tables"].long()[:, key // page].clamp(min=0) * page + key % page
    k, v = (x.view(-1, kv_heads, dim)[rows].float() for x in (s["k_cache"], s["v_cache"]))          # [B, keys, kv heads, dim]
    i = torch.arange(s["max_new"], device=dev)
    padded = q[(cu[:-1, None] + i).clamp(max=q.size(0) - 1)].float()
    padded = padded.view(*padded.shape[:2], kv_heads, -1, dim)                                       # [B, new, kv heads, group, dim]
    pos = (ctx - new)[:, None, None] + i[:, None]
    seen = key <= pos
    if c["window"]:
        seen = seen & ((key > pos - c["window"]) | (key < c["sinks"]))                               # [B, new, keys]
    score = torch.einsum("bihgd,bjhd->bhgij", padded, k).mul_(s["scale"])
    score.masked_fill_(~seen[:, None, None], -math.inf)
    top = score.amax(-1, keepdim=True)
    top = torch.where(top == -math.inf, torch.zeros_like(top), top)
    p = score.sub_(top).exp_()
    total = p.sum(-1, keepdim=True)
    o = torch.einsum("bhgij,bjhd->bihgd", p, v) / total.clamp(min=1e-30).permute(0, 3, 1, 2, 4)
    lse = (top + total.log()).squeeze(-1).permute(0, 3, 1, 2).flatten(2)                             # [B, new, heads]
    token = torch.arange(q.size(0), device=dev)
    request = torch.searchsorted(cu[1:], token, right=True)
    at = (request, token - cu[request])
    return {"out": o.flatten(2, 3)[at].to(q.dtype), **({"lse": lse[at]} if c["lse"] else {})}


def run(state):
    s = state
    c = s["case"]
    if own:
        if c["kind"] == "store":
            from nanovllm_voxcpm_b200 import glue

            glue.qk_norm_rope_kv_store(s["qkv"], c["heads"], c["kv_heads"], c["dim"], s["q_weight"], s["k_weight"], EPS,
                                       positions=s["positions"], cos=s["cos"], sin=s["sin"], k_cache=s["k_cache"],
                                       v_cache=s["v_cache"], slot_mapping=s["slot_mapping"], q_out=s["q"])
            return {"q": s["q"], "k_cache": s["k_cache"], "v_cache": s["v_cache"]}
        from nanovllm_voxcpm_b200 import attention

        if c["kind"] == "decode":
            got = attention.paged_decode_attention(s["q"], s["k_cache"], s["v_cache"], s["block_tables"], s["context_lens"],
                                                   scale=s["scale"], window=c["window"], sinks=c["sinks"], return_lse=c["lse"])
        else:
            got = attention.paged_prefill_attention(s["q"], s["k_cache"], s["v_cache"], s["block_tables"], s["context_lens"],
                                                    s["cu_seqlens"], scale=s["scale"], window=c["window"], sinks=c["sinks"],
                                                    return_lse=c["lse"])
        return {"out": got[0], "lse": got[1]} if c["lse"] else {"out": got}
    if c["kind"] == "store":
        _plain_store(s)
        return {"q": s["q"], "k_cache": s["k_cache"], "v_cache": s["v_cache"]}
    return _plain_attention(s)


# ----------------------------------------------------------------------------------------------------- 64 bits, by definition
def exact(case, seed):
    s = prepare(case, seed)
    new, ctx = _lens(case)
    kv_heads, dim, page = case["kv_heads"], case["dim"], case["page"]
    group = case["heads"] // kv_heads
    if case["kind"] == "store":
        x = s["qkv"].double().view(s["qkv"].size(0), -1, dim)
        T, heads = x.size(0), case["heads"]
        frequency = torch.tensor([ROPE_THETA ** (-2.0 * (j % (dim // 2)) / dim) for j in range(dim)], dtype=torch.float64, device=x.device)
        angle = (s["positions"].double()[:, None] * frequency)[:, None, :]
        weight = torch.ones(heads + 2 * kv_heads, dim, dtype=torch.float64, device=x.device)
        weight[:heads], weight[heads:heads + kv_heads] = s["q_weight"].double(), s["k_weight"].double()
        normed = x / (x.square().sum(-1, keepdim=True) / dim + EPS).sqrt() * weight
        partner = torch.roll(normed, dim // 2, dims=-1)
        partner[..., :dim // 2] *= -1
        turned = normed * angle.cos() + partner * angle.sin()
        k_cache, v_cache = s["k_cache"].double(), s["v_cache"].double()
        for t, slot in enumerate(s["slot_mapping"].tolist()):
            k_cache[slot // page, slot % page] = turned[t, heads:heads + kv_heads]
            v_cache[slot // page, slot % page] = x[t, heads + kv_heads:]
        return {"q": turned[:, :heads].contiguous(), "k_cache": k_cache, "v_cache": v_cache}
    out = torch.zeros(s["q"].shape, dtype=torch.float64, device=s["q"].device)
    lse = torch.zeros(s["q"].shape[:2], dtype=torch.float64, device=s["q"].device)
    tables = s["block_tables"].tolist()
    begin = 0
    for b, (n, c) in enumerate(zip(new, ctx)):
        first = _first_kept(case, n, c)
        keys = sorted(set(range(min(c, case["sinks"]))) | set(range(first, c)))
        place = torch.tensor([tables[b][j // page] * page + j % page for j in keys], device=out.device)
        key = torch.tensor(keys, device=out.device)
        for h in range(kv_heads):
            k = s["k_cache"][:, :, h].reshape(-1, dim)[place].double()
            v = s["v_cache"][:, :, h].reshape(-1, dim)[place].double()
            for i0 in range(0, n, 1024):
                rows = slice(begin + i0, begin + min(n, i0 + 1024))
                pos = torch.arange(c - n + i0, c - n + min(n, i0 + 1024), device=out.device)
                back = pos[:, None] - key
                hidden = back < 0
                if case["window"]:
                    hidden |= (back >= case["window"]) & (key >= case["sinks"])
                for g in range(h * group, (h + 1) * group):
                    x = torch.matmul(s["q"][rows, g].double(), k.T) * s["scale"]
                    x[hidden] = -math.inf
                    lse[rows, g] = torch.logsumexp(x, dim=-1)
                    out[rows, g] = torch.matmul(torch.exp(x - lse[rows, g, None]), v)
        begin += n
    return {"out": out, **({"lse": lse} if case["lse"] else {})}
