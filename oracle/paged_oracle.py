"""Plain 64-bit forms of the operators around the paged cache: head norms with rotation and store, causal attention over the
pages with window and first tokens. By the definitions, loops over requests; test infrastructure only."""

from __future__ import annotations

import math

import torch


def head_norm_rope(x: torch.Tensor, weight: torch.Tensor | None, eps: float, positions=None, cos=None, sin=None):
    """``x [T, heads, D]`` -> (result, size of the rotation's terms), both float64. ``cos`` / ``sin``: [max_pos, D] or [.., D / 2]."""
    x = x.double()
    if weight is not None:
        x = x / torch.sqrt((x * x).mean(-1, keepdim=True) + eps) * weight.double()
    if cos is None:
        return x, x.abs()
    half = x.size(-1) // 2
    pos = positions.clamp(0, cos.size(0) - 1)
    c, s = cos.double()[pos].unsqueeze(1), sin.double()[pos].unsqueeze(1)
    if c.size(-1) == half:
        c, s = torch.cat((c, c), -1), torch.cat((s, s), -1)
    turned = torch.cat((-x[..., half:], x[..., :half]), -1)
    return x * c + turned * s, (x * c).abs() + (turned * s).abs()


def visible_keys(pos: int, window: int, sinks: int, held: int) -> list[int]:
    """Keys that a token at position ``pos`` sees, of the first ``held`` of its sequence."""
    return [j for j in range(min(pos + 1, held)) if window == 0 or pos - j < window or j < sinks]


def paged_attention(q, k_cache, v_cache, tables, context_lens, cu_seqlens, scale, window, sinks):
    """(out, lse, mean of |v|, keys) per row and head, float64; rows of no sequence are NaN. ``cu_seqlens`` None: decode."""
    T, heads, dim = q.shape
    blocks, page, kv_heads, _ = k_cache.shape
    group = heads // kv_heads
    out = torch.full((T, heads, dim), math.nan, dtype=torch.float64)
    lse = torch.full((T, heads), math.nan, dtype=torch.float64)
    size = torch.zeros(T, heads, dim, dtype=torch.float64)
    count = torch.zeros(T, dtype=torch.int64)
    cu = list(range(len(context_lens) + 1)) if cu_seqlens is None else list(cu_seqlens)
    for r, ctx in enumerate(context_lens):
        rows = range(cu[r], cu[r + 1])
        if not rows:
            continue
        held = len(tables[r]) * page
        seen = [[j for j in visible_keys(ctx - 1 - (cu[r + 1] - 1 - row), window, sinks, held) if 0 <= tables[r][j // page] < blocks]
                for row in rows]
        keys = sorted(set().union(*map(set, seen)))
        at = {j: i for i, j in enumerate(keys)}
        place = [(tables[r][j // page], j % page) for j in keys]
        b, o = (torch.tensor([p[i] for p in place], dtype=torch.int64) for i in (0, 1))
        k = k_cache[b, o].double() if keys else torch.zeros(0, kv_heads, dim, dtype=torch.float64)
        v = v_cache[b, o].double() if keys else k
        hidden = torch.ones(len(rows), len(keys), dtype=torch.bool)
        for i, js in enumerate(seen):
            hidden[i, [at[j] for j in js]] = False
            count[rows[i]] = len(js)
        for h in range(heads):
            s = q[rows.start:rows.stop, h].double() @ k[:, h // group].T * scale
            s[hidden] = -math.inf
            total = torch.logsumexp(s, -1) if keys else torch.full((len(rows),), -math.inf, dtype=torch.float64)
            p = torch.exp(s - torch.where(total == -math.inf, torch.zeros_like(total), total)[:, None])
            # (a key that a row does not see has no part in it, whatever its value)
            vv = v[:, h // group]
            if vv.isfinite().all():
                out[rows.start:rows.stop, h], size[rows.start:rows.stop, h] = p @ vv, p @ vv.abs()
            else:
                for i in range(len(rows)):
                    mine = ~hidden[i]
                    out[rows[i], h], size[rows[i], h] = p[i, mine] @ vv[mine], p[i, mine] @ vv[mine].abs()
            lse[rows.start:rows.stop, h] = total
    return out, lse, size, count
