"""Attention over the paged cache by each way that a call can meet the GPU, the way checked first, so that a changed rule cannot leave one
of them without a test; and what values that are not finite do. Bounds in ``paged_problem.check``."""

import math

import pytest
import torch

import paged_problem as PP
from nanovllm_voxcpm_b200 import _native as N
from nanovllm_voxcpm_b200 import attention as A
from test_paged_ways import EIGHTS, FOURS, PAIRS, SHARES, WARPS4, WARPS8

pytestmark = pytest.mark.gpu
BF16, FP16 = torch.bfloat16, torch.float16


def _widened(p, keys):
    """The problem's arguments with a block table of at least ``keys`` keys (its width is what tells how long contexts may be)."""
    page = p["k"].size(1)
    args = list(p["args"])
    args[3] = torch.nn.functional.pad(args[3], (0, max(0, -(-keys // page) - args[3].size(1))), value=-1)
    return args


def _how(p):
    return dict(scale=p["scale"], window=p["window"], sinks=p["sinks"])


def _way(p, args):
    q, k, _, tables = args[:4]
    return N.lib().lora_b200_paged_decode_way(q.size(0), q.size(1), k.size(2), q.size(2), tables.size(1), k.size(1), p["window"], p["sinks"])


def _again(call, args, how, out, lse, rows=slice(None)):
    for _ in range(3):
        a, b = call(*args, **how, return_lse=True)
        assert torch.equal(a[rows], out[rows]) and torch.equal(b[rows], lse[rows])


DECODE = [
    # equal shares: one request in hundreds of parts, few blocks for few CTAs, none at all
    (SHARES, (16, 2, 64), [6000], 23000), (SHARES, (12, 1, 128), [3000], 12000), (SHARES, (3, 1, 64), [40], 23000), (SHARES, (16, 2, 64), [0], 23000),
    (SHARES, (1, 1, 128), [1], 12000),
    # rows of every length, empty ones among them; several whole items in a share; more rows than threads sum up
    (SHARES, (16, 2, 64), [5000, 0, 1, 33] + [(97 * i) % 700 for i in range(80)] + [4200, 0], 5000),
    (SHARES, (8, 2, 128), [0, 0, 2600] + [(61 * i) % 300 for i in range(90)] + [17], 2600),
    (SHARES, (2, 1, 64), [(13 * i) % 90 for i in range(299)] + [4300], 4300),
    # two chunks of heads, the second one short
    (SHARES, (40, 2, 64), [4200, 7, 0, 640] * 11 + [50], 4200), (SHARES, (23, 1, 128), [2100, 700] * 38 + [40] * 4, 2200),
    # clusters and single CTAs
    (EIGHTS, (16, 2, 64), [2000, 5], 2000), (FOURS, (8, 2, 64), [1000] * 10 + [3, 0], 1000), (FOURS, (40, 2, 128), [500, 900, 0, 320, 1, 33], 900),
    (PAIRS, (32, 8, 128), [1200, 800, 17, 0, 1100, 64], 1200), (WARPS8, (16, 2, 64), [1000, 30, 0, 500] * 10, 1000),
    (WARPS4, (16, 2, 128), [(37 * i) % 500 for i in range(90)], 500),
]


@pytest.mark.parametrize("dtype", [BF16, FP16])
@pytest.mark.parametrize("way,heads,contexts,keys", DECODE)
def test_decode_by_each_way(way, heads, contexts, keys, dtype):
    p = PP.make(*heads, 32, contexts, dtype=dtype, seed=len(contexts) + sum(heads), poison=True)
    args = _widened(p, keys)
    assert _way(p, args) == way
    out, lse = A.paged_decode_attention(*args, **_how(p), return_lse=True)
    PP.check(p, out, lse)
    _again(A.paged_decode_attention, args, _how(p), out, lse)
    assert N.device_status() == 0


@pytest.mark.parametrize("dim,window,contexts", [(64, 4300, [9000, 4300, 4301, 5, 0] + [300] * 80), (128, 2100, [5000, 2099, 40] + [200] * 90)])
def test_decode_shares_of_windows(dim, window, contexts):
    p = PP.make(8, 2, dim, 16, contexts, window=window, sinks=7, seed=dim, poison=True)
    assert _way(p, p["args"]) == SHARES
    out, lse = A.paged_decode_attention(*p["args"], **_how(p), return_lse=True)
    PP.check(p, out, lse)
    _again(A.paged_decode_attention, p["args"], _how(p), out, lse)


@pytest.mark.parametrize("dim", [64, 128])
def test_shares_of_prefill_rows(dim):
    """Pages that the tile kernel does not take, rows of no sequence among the shares, and a call without any row of a sequence."""
    p = PP.make(4, 2, dim, 12, [900, 61, 0, 5], [30, 61, 0, 9], seed=dim, poison=True, behind=60)
    args = _widened(p, 5000)
    out = torch.full_like(args[0], 7.0)
    need = N.lib().lora_b200_paged_prefill_workspace_bytes(out.size(0), 4, 4, 2, dim, args[3].size(1), 12, 0)
    assert need > 0
    got, lse = A.paged_prefill_attention(*args, **_how(p), out=out, return_lse=True)
    PP.check(p, got, lse)
    assert bool((out[100:] == 7).all())
    _again(A.paged_prefill_attention, args, _how(p), out, lse, slice(0, 100))
    out.fill_(7.0)
    A.paged_prefill_attention(*args[:5], torch.full_like(args[5], 3), **_how(p), out=out)
    assert bool((out == 7).all()) and N.device_status() == 0


def _items(p):
    """Pieces of work of the tile kernel, and CTAs of a launch."""
    heads, dim = p["q"].shape[1:]
    group, tile = heads // p["k"].size(2), 1
    while tile < 16 and group % (2 * tile) == 0:
        tile *= 2
    span = (1 if dim == 64 else 2) * (128 // tile)
    return sum(-(-(b - a) // span) for a, b in zip(p["cu"], p["cu"][1:])) * (heads // tile), 296 if dim == 64 else 148


def _cuts(p, args):
    q, k = args[:2]
    return N.lib().lora_b200_paged_prefill_workspace_bytes(q.size(0), args[4].numel(), q.size(1), k.size(2), q.size(2), args[3].size(1), k.size(1),
                                                           p["window"]) > 0


@pytest.mark.parametrize("dtype", [BF16, FP16])
# whole items, then parts of others in the same CTA; a rest of more than half a wave, which stays whole
@pytest.mark.parametrize("heads,new,contexts,rest", [((64, 4, 128), [450, 0, 200, 50], [1600, 3, 900, 1500], (1, 74)), ((64, 4, 128), [500, 480], [2100, 600], (75, 147)),
                                                     ((64, 4, 64), [500, 3, 207], [1600, 1590, 207], (1, 148)), ((64, 4, 64), [1000], [2050], (149, 295))])
def test_prefill_whole_waves_and_a_rest(heads, new, contexts, rest, dtype):
    p = PP.make(*heads, 32, contexts, new, dtype=dtype, seed=len(new), poison=True, behind=2)
    items, ctas = _items(p)
    assert _cuts(p, p["args"]) and items > ctas and rest[0] <= items % ctas <= rest[1]
    out = torch.full_like(p["args"][0], 7.0)
    got, lse = A.paged_prefill_attention(*p["args"], **_how(p), out=out, return_lse=True)
    PP.check(p, got, lse)
    assert bool((out[sum(new):] == 7).all())
    _again(A.paged_prefill_attention, p["args"], _how(p), out, lse, slice(0, sum(new)))
    assert N.device_status() == 0


@pytest.mark.parametrize("dim", [64, 128])
@pytest.mark.parametrize("window,sinks", [(0, 0), (60, 3)])
@pytest.mark.parametrize("requests", [18, 45])
def test_prefill_many_items_a_cta(requests, window, sinks, dim):
    """Three pieces of work and more for a CTA, of unequal length, some without keys."""
    new = [(100, 83, 0, 131, 9)[i % 5] + (i % 3 if i % 5 != 2 else 0) for i in range(requests)]
    contexts = [n + (i % 4) * 70 if i % 7 else 0 for i, n in enumerate(new)]
    p = PP.make(64, 4, dim, 16, contexts, new, window=window, sinks=sinks, seed=requests, poison=True, behind=1)
    items, ctas = _items(p)
    assert items > (2 if requests == 18 else 4) * ctas
    out, lse = A.paged_prefill_attention(*p["args"], **_how(p), return_lse=True)
    PP.check(p, out, lse)
    rows = slice(0, sum(new))
    _again(A.paged_prefill_attention, p["args"], _how(p), out, lse, rows)
    assert N.device_status() == 0


@pytest.mark.parametrize("dtype", [BF16, FP16])
@pytest.mark.parametrize("dim", [64, 128])
@pytest.mark.parametrize("cut", [False, True])
@pytest.mark.parametrize("falls", [False, True])
def test_prefill_extreme_scores(falls, cut, dim, dtype):
    """Scores of hundreds of either sign: the maximum grows by far more than 2^8 from tile to tile, or the first tile outweighs all others;
    then scores that are all equal."""
    new, contexts = [300, 140], [700, 900]
    p = PP.make(8, 2, dim, 16, contexts, new, dtype=dtype, seed=2)
    args = _widened(p, 16 * new[0] if cut else 0)
    assert _cuts(p, args) == cut
    for row, n in zip(p["tables"], contexts):
        for j, b in enumerate(row[:-(-n // 16)]):
            p["k"][b] *= 0.1 + 15 * (1 - j * 16 / n if falls else j * 16 / n)
    args[1] = p["k"].cuda()
    PP.check(p, *A.paged_prefill_attention(*args, **_how(p), return_lse=True))
    p["k"] = torch.zeros_like(p["k"])
    args[1] = p["k"].cuda()
    PP.check(p, *A.paged_prefill_attention(*args, **_how(p), return_lse=True))


def _rows_that_see(p, request, key):
    first, last = p["cu"][request], p["cu"][request + 1]
    return [row for row in range(first, last) if p["contexts"][request] - (last - row) >= key]


@pytest.mark.parametrize("dtype", [BF16, FP16])
@pytest.mark.parametrize("dim", [64, 128])
@pytest.mark.parametrize("cut", [False, True])
@pytest.mark.parametrize("value", [math.nan, math.inf])
def test_prefill_keys_that_are_not_finite(value, cut, dim, dtype):
    """A key with a NaN gives NaN to the rows that see it, as does a score of +inf; one of -inf has no weight. No other row changes."""
    p = PP.make(8, 2, dim, 16, [300, 280], [200, 90], dtype=dtype, seed=dim)
    args = _widened(p, 4000 if cut else 0)
    assert _cuts(p, args) == cut
    how = _how(p)
    args[0] = p["q"].abs().add_(0.01).cuda()  # (so that the sign of an infinite score is that of the key)
    args[1] = p["k"].cuda()
    want, want_lse = A.paged_prefill_attention(*args, **how, return_lse=True)
    for request, key in ((0, 0), (0, 137), (0, 299), (1, 250)):
        bad = p["k"].clone()
        bad[p["tables"][request][key // 16], key % 16, 1, 5] = value  # (of the second kv head)
        args[1] = bad.cuda()
        out, lse = A.paged_prefill_attention(*args, **how, return_lse=True)
        hit = torch.zeros(290, 8, dtype=torch.bool)
        hit[_rows_that_see(p, request, key), 4:] = True
        assert bool(out.cpu()[hit].isnan().all()) and bool(lse.cpu()[hit].isnan().all())
        assert torch.equal(out.cpu()[~hit], want.cpu()[~hit]) and torch.equal(lse.cpu()[~hit], want_lse.cpu()[~hit])
        if value == math.inf:
            args[1] = torch.where(bad.isinf(), -bad, bad).cuda()
            q, p["q"] = p["q"], args[0].cpu()
            got = A.paged_prefill_attention(*args, **how, return_lse=True)
            k, p["k"] = p["k"], p["k"].clone()
            blk = p["tables"][request][key // 16]
            p["k"][blk, key % 16, 1] = -2.0 ** 15  # (far below any other score: no weight in 64 bits either)
            norm = p["k"].clone()
            check_k(p, got, norm, blk, key % 16)
            p["q"], p["k"] = q, k


def check_k(p, got, norm, blk, at):
    """``paged_problem.check`` with the bound of the scores taken from the other keys: the one at hand has no weight, and no error."""
    out, lse = got
    u = torch.finfo(p["q"].dtype).eps / 2
    want, want_lse, size, count = PP.PO.paged_attention(p["q"], norm, p["v"], p["tables"], p["contexts"], p["cu"], p["scale"], p["window"], p["sinks"])
    norm[blk, at] = 0
    score_err = p["q"].size(-1) * 2.0 ** -24 * p["scale"] * float(p["q"].float().norm(dim=-1).max()) * float(norm.float().norm(dim=-1).max())
    eps = 2 * score_err + 2.0 ** -18 + count.double()[:, None, None] * 2.0 ** -23
    top = float(p["v"].float().abs().max())
    bound = u * want.abs() + (u * (1 + u) + eps) * size * (1 + u) + (count[:, None, None] * 2.0 ** -25 * top if p["q"].dtype == FP16 else 0)
    err = (out.double().cpu() - want).abs()
    alone = want_lse < -1000  # (rows that see no other key)
    assert bool((err <= bound + 1e-30)[~alone].all()), float((err / bound)[~alone].max())
    tol = score_err + 2.0 ** -19 * (1 + want_lse.abs()) + count.double()[:, None] * 2.0 ** -24
    assert bool(((lse.double().cpu() - want_lse).abs() <= tol)[~alone].all())
    assert bool((lse.cpu()[alone] == -math.inf).all()) and bool((out.cpu()[alone] == 0).all())


@pytest.mark.parametrize("dim", [64, 128])
def test_prefill_values_that_are_not_finite(dim):
    """A value with an infinity reaches the rows that see it and at most the others of their block of tokens, in its column alone."""
    p = PP.make(8, 2, dim, 16, [300, 280], [200, 90], seed=dim)
    args = list(p["args"])
    want, want_lse = A.paged_prefill_attention(*args, **_how(p), return_lse=True)
    span = 32 * (1 if dim == 64 else 2)
    for request, key in ((0, 0), (0, 137), (0, 299), (1, 250)):
        bad = p["v"].clone()
        bad[p["tables"][request][key // 16], key % 16, 1, 5] = math.inf
        args[2] = bad.cuda()
        out, lse = A.paged_prefill_attention(*args, **_how(p), return_lse=True)
        assert torch.equal(lse, want_lse)
        rows = _rows_that_see(p, request, key)
        hit, may = torch.zeros(290, 8, dim, dtype=torch.bool), torch.zeros(290, 8, dim, dtype=torch.bool)
        hit[rows, 4:, 5] = True
        first = p["cu"][request]
        may[first + (rows[0] - first) // span * span:p["cu"][request + 1], 4:, 5] = True
        assert not bool(out.cpu()[hit].isfinite().any())
        assert torch.equal(out.cpu()[~may], want.cpu()[~may])


@pytest.mark.parametrize("heads,contexts", [((8, 2, 64), [300, 40]), ((8, 2, 128), [300, 40]), ((8, 2, 64), [6000, 40]), ((8, 2, 64), [700] * 40)])
def test_decode_values_that_are_not_finite(heads, contexts):
    """Of the row that sees them, and of no other."""
    p = PP.make(*heads, 32, contexts, seed=len(contexts))
    for keys in (0, 23000 if len(contexts) < 3 else 0):
        args = _widened(p, keys)
        want, want_lse = A.paged_decode_attention(*args, **_how(p), return_lse=True)
        for which in ("k", "v"):
            bad = p[which].clone()
            bad[p["tables"][0][4], 7, 1, 5] = math.nan  # key 135 of the first request, second kv head
            got, lse = A.paged_decode_attention(args[0], *(bad.cuda() if x == which else p[x].cuda() for x in "kv"), *args[3:], **_how(p), return_lse=True)
            hit = torch.zeros(got.shape, dtype=torch.bool)
            hit[0, 4:] = True
            if which == "v":
                hit[..., :5] = hit[..., 6:] = False
            assert bool(got.cpu()[hit].isnan().all()) and torch.equal(got.cpu()[~hit], want.cpu()[~hit])
            told = lse.cpu()
            assert bool(told[0, 4:].isnan().all()) if which == "k" else torch.equal(told, want_lse.cpu())
            assert torch.equal(told[1:], want_lse.cpu()[1:]) and torch.equal(told[0, :4], want_lse.cpu()[0, :4])


@pytest.mark.parametrize("dim", [64, 128])
@pytest.mark.parametrize("page", [16, 12])  # (the tile kernel, the decode kernel)
def test_prefill_ranges_that_do_not_count(page, dim):
    """Of each list of ranges: rows that a sequence with a range of its own has are served, rows of a refused range stay as they are."""
    p = PP.make(8, 2, dim, page, [40, 50, 60], [40, 50, 60], seed=6)
    q, k, v, tables, ctx, cu = p["args"]
    want = A.paged_prefill_attention(*p["args"], **_how(p))
    PP.check(p, want)
    backwards = [([200, 40, 90, 150], [(40, 150)], [(0, 40)]), ([0, 40, 30, 150], [(0, 30), (90, 150)], [])] if page == 16 else []
    for bad, served, stay in [([0, 40, 90, 10 ** 6], [(0, 90)], [(90, 150)]), ([-5, 40, 90, 150], [(40, 150)], [(0, 40)])] + backwards:
        out = torch.full_like(q, 7.0)
        A.paged_prefill_attention(q, k, v, tables, ctx, torch.tensor(bad, dtype=torch.int32, device="cuda"), **_how(p), out=out)
        for a, b in served:
            assert torch.equal(out[a:b], want[a:b]), bad
        for a, b in stay:
            assert bool((out[a:b] == 7).all()), bad
    assert N.device_status() == 0


@pytest.mark.parametrize("dim", [64, 128])
@pytest.mark.parametrize("heads_first", [False, True])
def test_prefill_expanded_and_transposed(heads_first, dim):
    """q with heads ahead of tokens; one query row, one kv head or one block that stands for many."""
    p = PP.make(8, 2, dim, 16, [90, 200], [40, 33], seed=dim)
    q, k, v, *rest = p["args"]
    if heads_first:
        q = q.transpose(0, 1).contiguous().transpose(0, 1)
    want = A.paged_prefill_attention(q, k, v, *rest, **_how(p))
    PP.check(p, want)
    one = k[:, :, :1].expand_as(k), v[:, :, :1].expand_as(v)
    q1 = q[:1].expand_as(q)
    for args, same in (((q, *one), (q, *(x.contiguous() for x in one))), ((q1, k, v), (q1.contiguous(), k, v)),
                       ((q, k[:1].expand_as(k), v), (q, k[:1].expand_as(k).contiguous(), v))):
        p["q"], p["k"], p["v"] = (x.cpu() for x in same)
        PP.check(p, A.paged_prefill_attention(*args, *rest, **_how(p)))
        PP.check(p, A.paged_prefill_attention(*same, *rest, **_how(p)))
    assert N.device_status() == 0


@pytest.mark.parametrize("heads,contexts,new,keys", [((16, 2, 64), [5000], None, 23000), ((16, 2, 64), [2000, 5], None, 0), ((32, 8, 128), [700] * 40, None, 0),
                                                     ((16, 2, 64), [70, 900, 33], [70, 300, 1], 0), ((16, 2, 128), [3000, 40], [20, 40], 9000), ((8, 2, 64), [90, 61], [90, 33], 0)])
def test_results_in_place_of_the_queries(heads, contexts, new, keys):
    p = PP.make(*heads, 32, contexts, new, seed=len(contexts), behind=0 if new is None else 1)
    args, call = _widened(p, keys), A.paged_decode_attention if new is None else A.paged_prefill_attention
    rows = slice(0, len(contexts) if new is None else sum(new))
    want, want_lse = call(*args, **_how(p), return_lse=True)
    for _ in range(5):
        q = args[0].clone()
        out, lse = call(q, *args[1:], **_how(p), out=q, return_lse=True)
        assert out is q and torch.equal(q[rows], want[rows]) and torch.equal(lse[rows], want_lse[rows])
        assert torch.equal(q[rows.stop:], args[0][rows.stop:])


def test_large_calls_on_two_streams():
    """Cut prefills, shares of decodes and stores next to one another, each with tensors of its own stream."""
    ps = [PP.make(16, 2, 64, 64, [7000, 900], [90, 33], seed=1), PP.make(16, 2, 64, 64, [23500, 40], seed=2), PP.make(16, 2, 128, 64, [9000], [300], seed=3)]
    calls = [A.paged_prefill_attention, A.paged_decode_attention, A.paged_prefill_attention]
    want = [c(*p["args"], **_how(p)) for c, p in zip(calls, ps)]
    streams = [torch.cuda.Stream() for _ in ps]
    torch.cuda.synchronize()
    got = [[] for _ in ps]
    for _ in range(10):
        for i, (c, p, s) in enumerate(zip(calls, ps, streams)):
            with torch.cuda.stream(s):
                got[i].append(c(*p["args"], **_how(p)))
    torch.cuda.synchronize()
    for w, gs in zip(want, got):
        assert all(torch.equal(g, w) for g in gs)
    assert N.device_status() == 0
