"""More operators of the serving path that read the paged key-value cache, case by case.

Kinds of case
  shared_decode   ``attention.shared_prefix_decode_attention``: one new token per request; groups of requests begin with the same
                  tokens (a voice prompt, an instruction), whose keys and values lie in the cache once
  shared_prefill  ``attention.shared_prefix_prefill_attention``: a run of new tokens per request behind such a prefix
  diff_decode     ``attention.differential_decode_attention``: the difference of two softmax maps, one new token per request
  diff_prefill    ``attention.differential_prefill_attention``: the same for packed runs of new tokens
  join            ``attention.join_attention``: results over parts of a context, with the logarithms of their sums, to one

All attentions are causal; the differential ones over everything or over a sliding window of the last keys plus a few first ones.
Lengths are drawn from the case alone (``_lens``), values from the seed. Heads are those of this repository's configurations
(16 / 2 of 64, 16 / 2 of 128, 32 / 8 of 128) and, where drawn, other common groupings.
"""

from __future__ import annotations

import math
import random

import torch

#: False: `run` computes the plain forms; True: it calls the package's operators
own = False

DTYPES = {"bf16": torch.bfloat16, "fp16": torch.float16, "fp32": torch.float32}
EPS = 1e-5


def listed():
    return [
        # two requests of one short voice prompt, their first tokens: latency
        dict(name="shared_decode_2req", kind="shared_decode", groups=1, B=2, plo=300, phi=300, lo=1, hi=20, heads=16, kv_heads=2,
             dim=64, page=256, dtype="bf16", lse=False),
        # a decode step of 64 requests that speak with one voice
        dict(name="shared_decode_64req", kind="shared_decode", groups=1, B=64, plo=2003, phi=2003, lo=10, hi=600, heads=16,
             kv_heads=2, dim=64, page=256, dtype="bf16", lse=False),
        # the wide decoder, 96 requests behind four long instructions, small pages
        dict(name="shared_decode_4groups_wide", kind="shared_decode", groups=4, B=96, plo=3000, phi=9000, lo=50, hi=1500, heads=32,
             kv_heads=8, dim=128, page=16, dtype="bf16", lse=True),
        # a few tokens a request at a time (drafts that are checked) behind a long prefix, half precision
        dict(name="shared_prefill_drafts_fp16", kind="shared_prefill", groups=2, B=24, plo=4000, phi=6000, lo=0, hi=300, nlo=1,
             nhi=12, heads=16, kv_heads=2, dim=128, page=32, dtype="fp16", lse=False),
        # texts of ragged lengths behind one voice prompt
        dict(name="shared_prefill_texts", kind="shared_prefill", groups=1, B=32, plo=1501, phi=1501, lo=0, hi=0, nlo=20, nhi=120,
             heads=16, kv_heads=2, dim=64, page=256, dtype="bf16", lse=False),
        # one user, a few hundred tokens: latency
        dict(name="diff_decode_1req", kind="diff_decode", B=1, lo=333, hi=333, heads=16, kv_heads=2, dim=64, page=256, dtype="bf16",
             window=0, sinks=0, per_token=False, norm=True),
        # long contexts of the wide decoder, in small pages
        dict(name="diff_decode_48req_long_wide", kind="diff_decode", B=48, lo=500, hi=8192, heads=32, kv_heads=8, dim=128, page=16,
             dtype="bf16", window=0, sinks=0, per_token=False, norm=True),
        # streaming requests: a window of 1024 keys and 4 first ones; weights that every token has of its own, no norm
        dict(name="diff_decode_64req_window_fp16", kind="diff_decode", B=64, lo=3, hi=12000, heads=16, kv_heads=2, dim=128, page=16,
             dtype="fp16", window=1024, sinks=4, per_token=True, norm=False),
        # a prefill batch of ragged prompts
        dict(name="diff_prefill_12prompts", kind="diff_prefill", B=12, lo=101, hi=1200, before=0, heads=16, kv_heads=2, dim=64,
             page=256, dtype="bf16", window=0, sinks=0, per_token=False, norm=True),
        # a chunk of a long prompt of the wide decoder whose first tokens are in the cache: the most arithmetic
        dict(name="diff_prefill_chunk_wide", kind="diff_prefill", B=1, lo=2048, hi=2048, before=8192, heads=32, kv_heads=8, dim=128,
             page=256, dtype="bf16", window=0, sinks=0, per_token=False, norm=True),
        # four tokens whose contexts lie in two places: latency
        dict(name="join_4tok", kind="join", parts=2, T=4, heads=16, dim=64, dtype="bf16"),
        # a prefill chunk of the wide decoder, attended in four stretches of its context
        dict(name="join_4096tok_wide", kind="join", parts=4, T=4096, heads=32, dim=128, dtype="bf16"),
    ]


HEADS = [(16, 2, 64), (16, 2, 128), (32, 8, 128), (8, 8, 64), (12, 4, 64), (14, 2, 64), (24, 8, 64), (16, 1, 128)]


def draw(rng):
    def spread(lo, hi):  # evenly over the logarithm
        return min(hi, max(lo, round(math.exp(rng.uniform(math.log(lo), math.log(hi))))))

    kind = rng.choice(["shared_decode", "shared_decode", "shared_prefill", "diff_decode", "diff_decode", "diff_prefill", "join"])
    if kind == "join":
        heads, _, dim = rng.choice(HEADS)
        parts = rng.choice([1, 2, 2, 3, 4, spread(2, 32)])
        return dict(kind=kind, parts=parts, T=spread(1, max(1, 2 ** 25 // (parts * heads * dim))), heads=heads, dim=dim,
                    dtype=rng.choice(["bf16", "bf16", "fp16", "fp32"]))
    heads, kv_heads, dim = rng.choice(HEADS)
    case = dict(kind=kind, heads=heads, kv_heads=kv_heads, dim=dim, page=rng.choice([8, 16, 32, 48, 64, 128, 256]),
                dtype=rng.choice(["bf16", "bf16", "fp16"]))
    if kind.startswith("shared"):
        prefill = kind == "shared_prefill"
        B = spread(1, 64 if prefill else 256)
        groups = min(B, rng.choice([1, 1, 2, spread(1, 16)]))
        phi = spread(1, min(16000, 400000 // B, 60000 // groups))
        case.update(B=B, groups=groups, plo=rng.randint(1, phi), phi=phi, lse=rng.random() < 0.3)
        if not prefill:
            hi = spread(1, min(2000, 100000 // B))
            return dict(case, lo=rng.randint(1, hi), hi=hi)
        hi, nhi = rng.choice([0, spread(1, 500)]), spread(1, max(1, min(1000, 4096 // B)))
        return dict(case, lo=rng.randint(0, hi), hi=hi, nlo=rng.randint(1, nhi), nhi=nhi)
    window = rng.choice([0, 0, spread(1, 4096)])
    case.update(window=window, sinks=rng.choice([0, 1, 4, spread(1, 300)]) if window else 0, per_token=rng.random() < 0.3,
                norm=rng.random() < 0.7)
    if kind == "diff_decode":
        B = spread(1, 256)
        hi = spread(1, min(100000, 250000 // B))
        return dict(case, B=B, lo=rng.randint(1, hi), hi=hi)
    B = spread(1, 32)
    hi = spread(1, max(1, 4096 // B))
    return dict(case, B=B, lo=rng.randint(1, hi), hi=hi, before=rng.choice([0, 0, spread(1, 4096 if B * hi <= 2048 else 1024)]))


# ------------------------------------------------------------------------------------------------ lengths and tables
def _lens(case):
    """(new tokens, context with them, prefix, group) of every request; prefix 0 and group 0 where nothing is shared."""
    rng = random.Random("%(B)d %(lo)d %(hi)d" % case)
    B = case["B"]
    if not case["kind"].startswith("shared"):
        new = [rng.randint(case["lo"], case["hi"]) for _ in range(B)]
        if case["kind"] == "diff_decode":
            return [1] * B, new, [0] * B, [0] * B
        return new, [n + (case["before"] if B == 1 else rng.randint(0, case["before"])) for n in new], [0] * B, [0] * B
    cuts = sorted(rng.sample(range(1, B), case["groups"] - 1))
    group = [sum(i >= c for c in cuts) for i in range(B)]
    prefixes = [rng.randint(case["plo"], case["phi"]) for _ in range(case["groups"])]
    prefix = [prefixes[g] for g in group]
    behind = [rng.randint(case["lo"], case["hi"]) for _ in range(B)]
    if case["kind"] == "shared_decode":  # (of the own tokens the new one is the last)
        return [1] * B, [p + n for p, n in zip(prefix, behind)], prefix, group
    new = [rng.randint(case["nlo"], case["nhi"]) for _ in range(B)]
    return new, [p + b + n for p, b, n in zip(prefix, behind, new)], prefix, group


def _visible(case, pos):
    """Number of keys that a token at `pos` sees."""
    window = case.get("window", 0)
    first = max(0, pos - window + 1) if window else 0
    return pos + 1 - first + min(first, case.get("sinks", 0))


def _first_kept(case, n, c):
    """First key behind the sinks that the `n` last tokens of a context of `c` see."""
    return max(0, c - n - case["window"] + 1) if case.get("window", 0) else 0


def work(case):
    if case["kind"] == "join":
        rows = case["T"] * case["heads"]
        size = DTYPES[case["dtype"]].itemsize
        return {"bytes": rows * ((case["parts"] + 1) * (case["dim"] * size + 4)), "flops": 2 * rows * case["parts"] * case["dim"]}
    new, ctx, prefix, group = _lens(case)
    T, dim, heads = sum(new), case["dim"], case["heads"]
    keys = sum({g: p for g, p in zip(group, prefix)}.values())
    pairs = 0
    for n, c, p in zip(new, ctx, prefix):
        first = _first_kept(case, n, c)
        keys += c - p - first + min(first, case.get("sinks", 0))
        pairs += sum(_visible(case, at) for at in range(c - n, c))
    extra = 4 * T * heads if case.get("lse") else 0
    if case["kind"].startswith("diff"):
        extra += 4 * heads * (T if case["per_token"] else 1) + (2 * dim if case["norm"] else 0)
    per_pair = 6 if case["kind"].startswith("diff") else 4  # two products of half the columns, one or two of all with V
    return {"bytes": 4 * keys * case["kv_heads"] * dim + 4 * T * heads * dim + extra, "flops": per_pair * pairs * heads * dim}


def prepare(case, seed):
    dev, dt = torch.device("cuda"), DTYPES[case["dtype"]]
    gen = torch.Generator(device=dev).manual_seed(seed)
    host = random.Random(seed)
    heads, dim = case["heads"], case["dim"]

    def normal(*shape, scale=1.0):
        return torch.randn(*shape, device=dev, dtype=dt, generator=gen) * scale

    if case["kind"] == "join":
        # stretches of a context hold shares of the whole sum of any size; some hold no key that a token sees
        lse = torch.randn(case["parts"], case["T"], heads, device=dev, generator=gen) * 2 + 5
        none = torch.rand(case["parts"], case["T"], 1, device=dev, generator=gen) < 0.1
        lse.masked_fill_(none, -math.inf)
        outs = normal(case["parts"], case["T"], heads, dim).masked_fill_(none[..., None], 0)
        return dict(case=case, outs=outs, lses=lse)
    new, ctx, prefix, group = _lens(case)
    T, B, page, kv_heads = sum(new), case["B"], case["page"], case["kv_heads"]
    width = max(-(-c // page) for c in ctx)
    n_blocks = sum(-(-c // page) for c in ctx) + 3
    order = torch.randperm(n_blocks, device=dev, generator=gen).tolist()
    k_cache, v_cache = normal(n_blocks, page, kv_heads, dim), normal(n_blocks, page, kv_heads, dim)
    tables = []
    for i, (n, c, p) in enumerate(zip(new, ctx, prefix)):
        pages = [order.pop() for _ in range(-(-c // page))]
        if i > 0 and group[i] == group[i - 1] and p:
            # whole pages of the prefix are the group's; the page that it ends in is a copy
            pages[:p // page] = tables[-1][:p // page]
            if p % page:
                at, its = pages[p // page], tables[-1][p // page]
                k_cache[at, :p % page], v_cache[at, :p % page] = k_cache[its, :p % page], v_cache[its, :p % page]
        first, sinks = _first_kept(case, n, c), case.get("sinks", 0)
        # pages that no token of the step sees any more have gone back to the allocator
        kept = [b if x * page < sinks or (x + 1) * page > first else -1 for x, b in enumerate(pages)]
        tables.append(kept + [-1] * (width - len(kept)))
    cu = [0]
    for n in new:
        cu.append(cu[-1] + n)
    starts = [i for i in range(B) if i == 0 or group[i] != group[i - 1]]

    def ints(values):
        return torch.tensor(values, dtype=torch.int32, device=dev)

    state = dict(case=case, k_cache=k_cache, v_cache=v_cache, block_tables=ints(tables), context_lens=ints(ctx), cu_seqlens=ints(cu),
                 max_new=max(new), max_context=max(ctx), prefix_lens=ints([prefix[i] for i in starts]), cu_groups=ints(starts + [B]),
                 scale=dim ** -0.5)
    # normed heads: scores of a spread of one to three, so that attention is neither flat nor on a single key
    state["q"] = normal(T, heads, dim, scale=1.0 + 2.0 * host.random())
    if case["kind"].startswith("diff"):
        state["scale"] = (dim // 2) ** -0.5
        # weights of the second map as training leaves them: per head, or per token and head
        state["lam"] = torch.sigmoid(torch.randn(*((T, heads) if case["per_token"] else (heads,)), device=dev, generator=gen))
        state["norm_weight"] = (0.8 + 0.2 * torch.randn(dim, device=dev, generator=gen)).to(dt) if case["norm"] else None
    return state


# --------------------------------------------------------------------------------------------------------- plain forms
def _plain_maps(s, q, k_columns):
    """Attention of all requests side by side, padded to the longest, in 32 bits, with the given columns of K: out [T, heads, dim]
    and lse [T, heads]."""
    c = s["case"]
    page, kv_heads, dim, dev = c["page"], c["kv_heads"], c["dim"], q.device
    cu, ctx = s["cu_seqlens"].long(), s["context_lens"].long()
    new = cu[1:] - cu[:-1]
    key = torch.arange(s["max_context"], device=dev)
    rows = s["block_tables"].long()[:, key // page].clamp(min=0) * page + key % page
    k = s["k_cache"].view(-1, kv_heads, dim)[rows][..., k_columns].float()                           # [B, keys, kv heads, columns]
    v = s["v_cache"].view(-1, kv_heads, dim)[rows].float()
    i = torch.arange(s["max_new"], device=dev)
    padded = q[(cu[:-1, None] + i).clamp(max=q.size(0) - 1)].float()
    padded = padded.view(*padded.shape[:2], kv_heads, -1, padded.size(-1))                           # [B, new, kv heads, group, columns]
    pos = (ctx - new)[:, None, None] + i[:, None]
    seen = key <= pos
    if c.get("window", 0):
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
    return o.flatten(2, 3)[at], lse[at]


def _plain(s):
    c = s["case"]
    if c["kind"] == "join":
        top = s["lses"].amax(0)
        top = torch.where(top == -math.inf, torch.zeros_like(top), top)
        share = torch.exp(s["lses"] - top)
        total = share.sum(0)
        out = (share[..., None] * s["outs"].float()).sum(0) / total.clamp(min=1e-30)[..., None]
        return {"out": out.to(s["outs"].dtype), "lse": top + total.log()}
    q, dim = s["q"], c["dim"]
    if c["kind"].startswith("shared"):
        out, lse = _plain_maps(s, q, slice(0, dim))
        return {"out": out.to(q.dtype), **({"lse": lse} if c["lse"] else {})}
    half = dim // 2
    out = _plain_maps(s, q[..., :half], slice(0, half))[0]
    out = out - s["lam"][..., None] * _plain_maps(s, q[..., half:], slice(half, dim))[0]
    if c["norm"]:
        out = out * torch.rsqrt((out * out).mean(-1, keepdim=True) + EPS) * s["norm_weight"].float()
    return {"out": out.to(q.dtype)}


def run(state):
    s = state
    c = s["case"]
    if not own:
        return _plain(s)
    from nanovllm_voxcpm_b200 import attention

    if c["kind"] == "join":
        out, lse = attention.join_attention(s["outs"], s["lses"], return_lse=True)
        return {"out": out, "lse": lse}
    cache = (s["q"], s["k_cache"], s["v_cache"], s["block_tables"], s["context_lens"])
    if c["kind"].startswith("shared"):
        if c["kind"] == "shared_decode":
            got = attention.shared_prefix_decode_attention(*cache, s["prefix_lens"], s["cu_groups"], scale=s["scale"], return_lse=c["lse"])
        else:
            got = attention.shared_prefix_prefill_attention(*cache, s["cu_seqlens"], s["prefix_lens"], s["cu_groups"], scale=s["scale"],
                                                            return_lse=c["lse"])
        return {"out": got[0], "lse": got[1]} if c["lse"] else {"out": got}
    how = dict(norm_weight=s["norm_weight"], eps=EPS, scale=s["scale"], window=c["window"], sinks=c["sinks"])
    if c["kind"] == "diff_decode":
        return {"out": attention.differential_decode_attention(*cache, s["lam"], **how)}
    return {"out": attention.differential_prefill_attention(*cache, s["cu_seqlens"], s["lam"], **how)}


# ----------------------------------------------------------------------------------------------------- 64 bits, by definition
def exact(case, seed):
    s = prepare(case, seed)
    if case["kind"] == "join":
        lse = torch.logsumexp(s["lses"].double(), dim=0)
        out = torch.zeros(s["outs"].shape[1:], dtype=torch.float64, device=lse.device)
        for o, part in zip(s["outs"], s["lses"].double()):
            out += torch.nan_to_num(torch.exp(part - lse), nan=0.0)[..., None] * o.double()
        return {"out": out, "lse": lse}
    new, ctx, _, _ = _lens(case)
    kv_heads, dim, page = case["kv_heads"], case["dim"], case["page"]
    group = case["heads"] // kv_heads
    two = case["kind"].startswith("diff")
    out = torch.zeros(s["q"].shape, dtype=torch.float64, device=s["q"].device)
    lse = torch.zeros(s["q"].shape[:2], dtype=torch.float64, device=s["q"].device)
    tables = s["block_tables"].tolist()
    if two:
        lam = s["lam"].double().expand(out.shape[:2])
    begin = 0
    for b, (n, c) in enumerate(zip(new, ctx)):
        first = _first_kept(case, n, c)
        keys = sorted(set(range(min(c, case.get("sinks", 0)))) | set(range(first, c)))
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
                if case.get("window", 0):
                    hidden |= (back >= case["window"]) & (key >= case["sinks"])
                for g in range(h * group, (h + 1) * group):
                    x = s["q"][rows, g].double()
                    for m, part in enumerate(torch.chunk(torch.arange(dim), 2) if two else [torch.arange(dim)]):
                        y = torch.matmul(x[:, part], k[:, part].T) * s["scale"]
                        y[hidden] = -math.inf
                        lse[rows, g] = torch.logsumexp(y, dim=-1)
                        weight = 1 if m == 0 else -lam[rows, g, None]
                        out[rows, g] += weight * torch.matmul(torch.exp(y - lse[rows, g, None]), v)
        begin += n
    if two and case["norm"]:
        out = out / (out.square().sum(-1, keepdim=True) / dim + EPS).sqrt() * s["norm_weight"].double()
    return {"out": out, **({"lse": lse} if case.get("lse") else {})}
