"""Random problems over a paged cache for the tests, and the bounds that follow from the kernels' roundings."""

import math
import random

import torch

from oracle import paged_oracle as PO


def make(heads, kv_heads, dim, page, contexts, new=None, *, dtype=torch.bfloat16, window=0, sinks=0, seed=0, poison=False, spare=2,
         interleaved=False, device="cuda", behind=0):
    """``new`` None: decode. ``poison``: every cache row that no token sees is NaN, blocks without a seen key are given back.
    ``interleaved``: k and v of a block in one tensor, heads ahead of positions. ``behind``: rows of q behind the last sequence."""
    gen = torch.Generator().manual_seed(seed)
    host = random.Random(seed)
    n_blocks = sum(-(-max(c, 0) // page) for c in contexts) + spare
    order = list(range(n_blocks))
    host.shuffle(order)
    width = max(1, max(-(-max(c, 0) // page) for c in contexts))
    tables = []
    seen_rows = torch.zeros(n_blocks, page, dtype=torch.bool)
    for i, c in enumerate(contexts):
        mine = [order.pop() for _ in range(-(-max(c, 0) // page))]
        n = 1 if new is None else new[i]
        seen = {j for t in range(n) for j in PO.visible_keys(c - 1 - t, window, sinks, len(mine) * page)}
        for j in seen:
            seen_rows[mine[j // page], j % page] = True
        kept = {j // page for j in seen}
        tables.append([b if not poison or x in kept else -1 for x, b in enumerate(mine)] + [-1 if poison else 0] * (width - len(mine)))
    T = (len(contexts) if new is None else sum(new)) + behind
    k = torch.randn(n_blocks, page, kv_heads, dim, generator=gen)
    v = torch.randn(n_blocks, page, kv_heads, dim, generator=gen)
    if poison:
        k[~seen_rows] = math.nan
        v[~seen_rows] = math.nan
    q = (torch.randn(T, heads, dim, generator=gen) * 2).to(dtype)
    k, v = k.to(dtype), v.to(dtype)
    cu = None
    if new is not None:
        cu = [0]
        for n in new:
            cu.append(cu[-1] + n)
    if interleaved:
        both = torch.empty(n_blocks, 2, kv_heads, page, dim, dtype=dtype)
        both[:, 0], both[:, 1] = k.transpose(1, 2), v.transpose(1, 2)
        both = both.to(device)
        kd, vd = both[:, 0].transpose(1, 2), both[:, 1].transpose(1, 2)
    else:
        kd, vd = k.to(device), v.to(device)
    as_int = lambda x: torch.tensor(x, dtype=torch.int32, device=device)  # noqa: E731
    return dict(q=q, k=k, v=v, tables=tables, contexts=contexts, cu=cu, window=window, sinks=sinks, scale=dim ** -0.5,
                args=(q.to(device), kd, vd, as_int(tables), as_int(contexts), *([] if cu is None else [as_int(cu)])))


def check(p, out, lse=None, what=""):
    """Bounds: the result is rounded once (u relative) and every probability once before its product with v (u relative, in fp16
    also half of the smallest step, 2^-25 against a largest probability of at least 1), while their sum is not: u (|out| + sum
    p |v|) + keys 2^-25 max |v|. Scores are sums of dim products in fp32: off by at most dim 2^-24 sum |q k| scale, which is also
    the relative error of a probability, twice with the denominator; exponentials and the running sums add 2^-18 and keys 2^-24."""
    q = p["q"]
    u = torch.finfo(q.dtype).eps / 2
    want, want_lse, size, count = PO.paged_attention(q, p["k"], p["v"], p["tables"], p["contexts"], p["cu"], p["scale"], p["window"], p["sinks"])
    rows = ~want_lse[:, 0].isnan()
    k_finite = p["k"].float().nan_to_num(0, 0, 0)
    score_err = q.size(-1) * 2.0 ** -24 * p["scale"] * float(q.float().norm(dim=-1).max()) * float(k_finite.norm(dim=-1).max())
    eps = 2 * score_err + 2.0 ** -18 + count.double()[:, None, None] * 2.0 ** -23
    top = float(p["v"].float().nan_to_num(0, 0, 0).abs().max())
    bound = u * want.abs() + (u * (1 + u) + eps) * size * (1 + u) + (count[:, None, None] * 2.0 ** -25 * top if q.dtype == torch.float16 else 0)
    got = out.double().cpu()
    err = (got - want).abs()[rows]
    assert not got[rows].isnan().any(), f"{what}: NaN"
    assert bool((err <= bound[rows] + 1e-30).all()), f"{what}: worst {float((err / (bound[rows] + 1e-30)).max()):.3g} of the bound"
    if lse is not None:
        got, want_lse = lse.double().cpu()[rows], want_lse[rows]
        empty = want_lse == -math.inf
        assert torch.equal(got == -math.inf, empty), f"{what}: lse of empty rows"
        tol = score_err + 2.0 ** -19 * (1 + want_lse.abs()) + count[rows].double()[:, None] * 2.0 ** -24
        assert bool(((got - want_lse).abs() <= tol)[~empty].all()), f"{what}: lse off by {float((got - want_lse)[~empty].abs().max()):.3g}"
