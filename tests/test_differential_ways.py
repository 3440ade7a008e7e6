"""How a differential call meets the GPU, said first and then run, so that a changed rule cannot leave a way without a test; and what values
that are not finite do by each of them."""

import math

import pytest
import torch

import test_differential_gpu as TD
from nanovllm_voxcpm_b200 import _native as N
from nanovllm_voxcpm_b200 import attention as A
from test_paged_ways import EIGHTS, FOURS, PAIRS, SHARES, WARPS4, WARPS8

BF16, FP16 = torch.bfloat16, torch.float16

# way, heads, contexts, keys that the table holds
DECODE = [
    (SHARES, (16, 2, 64), [6000], 23000), (SHARES, (3, 1, 128), [40], 12000), (SHARES, (16, 2, 64), [0], 23000),
    (SHARES, (16, 2, 64), [5000, 0, 1, 33] + [(97 * i) % 700 for i in range(80)] + [4200, 0], 5000),
    (SHARES, (8, 2, 128), [0, 0, 2600] + [(61 * i) % 300 for i in range(90)] + [17], 2600),
    (SHARES, (20, 2, 64), [4200, 7, 0, 640] * 11 + [50], 4200),  # (chunks of eight heads and of two)
    (EIGHTS, (16, 2, 64), [2000, 5], 2000), (EIGHTS, (16, 2, 128), [333, 0], 333), (FOURS, (8, 2, 64), [1000] * 10 + [3, 0], 1000),
    (FOURS, (20, 2, 128), [500, 900, 0, 320, 1, 33], 900), (PAIRS, (32, 8, 128), [1200, 800, 17, 0, 1100, 64], 1200),
    (WARPS8, (16, 2, 64), [1000, 30, 0, 500] * 10, 1000), (WARPS4, (16, 2, 128), [(37 * i) % 500 for i in range(90)], 500),
]
# heads, new tokens, contexts; whether items are cut along the keys and joined
PREFILL = [((16, 2, 64), [40, 90], [60, 90], False), ((16, 2, 128), [40, 90], [60, 90], False), ((16, 2, 64), [20], [2500], True),
           ((16, 2, 128), [20], [2500], True)]


def way(T, heads, kv_heads, dim, width, page, window=0, sinks=0):
    return N.lib().lora_b200_differential_way(T, heads, kv_heads, dim, width, page, window, sinks)


def test_the_rule():
    """Host code: every case of the list takes the way that it is there for, and shares alone take a workspace."""
    need = N.lib().lora_b200_differential_workspace_bytes
    for its, (heads, kv_heads, dim), contexts, keys in DECODE:
        n = len(contexts)
        assert way(n, heads, kv_heads, dim, -(-keys // 32), 32) == its, (its, heads, contexts[:4])
        assert (need(n, n, heads, kv_heads, dim, -(-keys // 32), 32, 0, 0, 0) > 0) == (its == SHARES)
    for (heads, kv_heads, dim), new, contexts, cut in PREFILL:
        assert (need(sum(new), len(new), heads, kv_heads, dim, -(-max(contexts) // 16), 16, 0, 0, 1) > 0) == cut
    assert way(1, 8, 0, 64, 100, 1) < 0 and way(1, 2, 4, 64, 100, 1) < 0
    assert way(64, 16, 2, 128, 750, 16, 1024, 4) == WARPS8  # (a window is what a row sees at most)


def _decode_problem(heads, contexts, keys, dtype=BF16, **kw):
    p = TD.make(*heads, 32, contexts, dtype=dtype, seed=len(contexts) + sum(heads), **kw)
    args = list(p["args"])
    args[3] = torch.nn.functional.pad(args[3], (0, max(0, -(-keys // 32) - args[3].size(1))), value=-1)
    p["args"] = tuple(args)
    return p


def _taken(p):
    q, k, _, tables = p["args"][:4]
    return way(q.size(0), q.size(1), k.size(2), q.size(2), tables.size(1), k.size(1), p["window"], p["sinks"])


@pytest.mark.gpu
@pytest.mark.parametrize("dtype,norm", [(BF16, True), (FP16, False)])
@pytest.mark.parametrize("its,heads,contexts,keys", DECODE)
def test_decode_by_each_way(its, heads, contexts, keys, dtype, norm):
    p = _decode_problem(heads, contexts, keys, dtype, norm=norm, poison=True)
    assert _taken(p) == its
    out = TD.call(p)
    TD.check(p, out)
    assert torch.equal(out, TD.call(p)) and N.device_status() == 0


def _with(p, **kw):
    """The call with other k, v, lam or weight on the GPU."""
    args = list(p["args"])
    for i, name in ((1, "k"), (2, "v")):
        args[i] = kw.get(name, args[i])
    f = A.differential_decode_attention if p["cu"] is None else A.differential_prefill_attention
    weight = kw.get("weight", None if p["weight"] is None else p["weight"].cuda())
    return f(*args, kw.get("lam", p["lam"].cuda()), norm_weight=weight, eps=TD.EPS, window=p["window"], sinks=p["sinks"])


def _poisoned(p, name, request, key, kv_head, column, value=math.nan):
    c = p["args"][1 if name == "k" else 2].clone()
    page = c.size(1)
    c[p["tables"][request][key // page], key % page, kv_head, column] = value
    return {name: c}


# (a request of 40 keys by each way: its last key is the one that is not finite)
@pytest.mark.gpu
@pytest.mark.parametrize("norm", [False, True])
@pytest.mark.parametrize("dim", [64, 128])
@pytest.mark.parametrize("its,n,keys", [(EIGHTS, 2, 2000), (FOURS, 16, 2000), (WARPS8, 40, 600), (WARPS4, 100, 300), (SHARES, 2, 23000)])
def test_decode_of_values_that_are_not_finite(its, n, keys, dim, norm):
    p = _decode_problem((4, 2, dim), [40] * n, keys, norm=norm)
    assert _taken(p) == its
    base = TD.call(p)
    touched, column = (0, slice(2, 4)), 5
    others = torch.ones(n, 4, dtype=torch.bool, device="cuda")
    others[0, 2:] = False
    # a value: its column of the heads that see it, of a normed head all of it
    for value in (math.nan, math.inf):
        out = _with(p, **_poisoned(p, "v", 0, 39, 1, column, value))
        assert torch.equal(out[others], base[others])
        bad = ~out[touched].isfinite()
        assert bool(bad[:, column].all())
        assert bool(bad.any(-1).all()) if norm else int(bad.sum()) == 2 and torch.equal(out[touched][~bad], base[touched][~bad])
    # a key: the map that has its column, with it the head
    for c in (column, dim - 3):
        out = _with(p, **_poisoned(p, "k", 0, 39, 1, c))
        assert torch.equal(out[others], base[others]) and bool(out[touched].isnan().all())
    # lam: of one head, in all requests; by requests, of one
    for value in (math.inf, math.nan):
        lam = p["lam"].cuda()
        lam[3] = value
        out = _with(p, lam=lam)
        assert torch.equal(out[:, :3], base[:, :3]) and not bool(out[:, 3].isfinite().all(-1).any())
        lam = p["lam"].cuda().expand(n, 4).clone()
        lam[n - 1, 3] = value
        out = _with(p, lam=lam)
        others = torch.ones_like(others)
        others[n - 1, 3] = False
        assert torch.equal(out[others], base[others]) and not bool(out[n - 1, 3].isfinite().all())
        others = torch.ones_like(others)
        others[0, 2:] = False
    if norm:
        weight = p["weight"].cuda().clone()
        weight[7] = math.inf
        out, kept = _with(p, weight=weight), [c for c in range(dim) if c != 7]
        assert torch.equal(out[..., kept], base[..., kept]) and not bool(out[..., 7].isfinite().any())
    assert N.device_status() == 0


@pytest.mark.gpu
@pytest.mark.parametrize("norm", [False, True])
@pytest.mark.parametrize("heads,new,contexts,cut", PREFILL)
def test_prefill_of_values_that_are_not_finite(heads, new, contexts, cut, norm):
    p = TD.make(*heads, 16, contexts, new, norm=norm, seed=sum(new))
    base = TD.call(p)
    dim, n, ctx = heads[2], new[0], contexts[0]
    key, seen_from = ctx - n // 2, n - n // 2  # the last n // 2 tokens of the first sequence see that key
    here = slice(0, n)
    for value in (math.nan, math.inf):
        out = _with(p, **_poisoned(p, "v", 0, key, 1, 5, value))
        assert torch.equal(out[:, :8], base[:, :8]) and torch.equal(out[n:], base[n:])  # (of another kv head, of another sequence)
        assert not bool(out[seen_from:n, 8:, 5].isfinite().any())
        if not norm:  # (in tokens ahead of the key, of the same block of rows, it may reach its column: zero times it)
            kept = [c for c in range(dim) if c != 5]
            assert torch.equal(out[here, 8:][..., kept], base[here, 8:][..., kept])
    for c in (5, dim - 3):
        out = _with(p, **_poisoned(p, "k", 0, key, 1, c))
        assert torch.equal(out[:, :8], base[:, :8]) and torch.equal(out[n:], base[n:])
        assert bool(out[seen_from:n, 8:].isnan().all()) and torch.equal(out[:seen_from], base[:seen_from])
    for value in (math.inf, math.nan):
        lam = p["lam"].cuda().expand(sum(new), heads[0]).clone()
        lam[3, 2] = value
        out = _with(p, lam=lam)
        others = torch.ones(out.shape[:2], dtype=torch.bool, device="cuda")
        others[3, 2] = False
        assert torch.equal(out[others], base[others]) and not bool(out[3, 2].isfinite().all())
        out = _with(p, lam=lam[3].contiguous())
        others[:] = True
        others[:, 2] = False
        assert torch.equal(out[others], base[others]) and not bool(out[:, 2].isfinite().all(-1).any())
    if norm:
        weight = p["weight"].cuda().clone()
        weight[7] = math.inf
        out, kept = _with(p, weight=weight), [c for c in range(dim) if c != 7]
        assert torch.equal(out[..., kept], base[..., kept]) and not bool(out[..., 7].isfinite().any())
    assert N.device_status() == 0
