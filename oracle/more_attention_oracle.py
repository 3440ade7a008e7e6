"""Plain 64-bit forms of the attentions over the paged cache that are more than one softmax: the difference of two maps with its norm,
and the join of results over parts. By the definitions; test infrastructure only."""

from __future__ import annotations

import math

import torch

from .paged_oracle import paged_attention


def two_maps(q, k_cache, v_cache, tables, context_lens, cu_seqlens, scale, window, sinks):
    """((out, size) of the first map, of the second, keys a row), float64; rows of no sequence are NaN. ``size``: mean of |v|."""
    half = q.size(-1) // 2
    maps = []
    for m in range(2):
        cols = slice(m * half, (m + 1) * half)
        outs, sizes = [], []
        for part in range(2):  # (the columns of v are independent of one another)
            v = v_cache[..., part * half:(part + 1) * half]
            o, _, size, count = paged_attention(q[..., cols], k_cache[..., cols], v, tables, context_lens, cu_seqlens, scale, window, sinks)
            outs.append(o)
            sizes.append(size)
        maps.append((torch.cat(outs, -1), torch.cat(sizes, -1)))
    return maps[0], maps[1], count


def rms_norm(y, weight, eps):
    return y / (y.square().mean(-1, keepdim=True) + eps).sqrt() * weight.double()


def join(outs, lses):
    """``outs [parts, T, H, D]``, ``lses [parts, T, H]`` -> (out, lse, sum of |terms|), float64."""
    lses = lses.double()
    lse = torch.logsumexp(lses, 0)
    share = torch.exp(lses - torch.where(lse == -math.inf, torch.zeros_like(lse), lse))
    terms = torch.where((lses == -math.inf)[..., None], torch.zeros((), dtype=torch.float64, device=outs.device), share[..., None] * outs.double())
    return terms.sum(0), lse, terms.abs().sum(0)
