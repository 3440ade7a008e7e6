"""Attention of requests that begin alike against the 64-bit form of attention over each one's whole context; bounds in
``paged_problem.check`` (a sum in two or more pieces that are fp32 rounds no more than one in one piece: the pieces' references leave
with their sums)."""

import math
import random

import pytest
import torch

import paged_problem as PP
from nanovllm_voxcpm_b200 import _native as N
from nanovllm_voxcpm_b200 import attention as A

pytestmark = pytest.mark.gpu
BF16, FP16 = torch.bfloat16, torch.float16


def way(p):
    """1: the call is attended by group; 0: request by request."""
    q, k, _, tables, lens, *cu = p["args"]
    return N.lib().lora_b200_shared_prefix_way(q.size(0), lens.numel(), p["groups"][0].numel(), q.size(1), k.size(2), q.size(2), tables.size(1),
                                               k.size(1), bool(cu))


def make(heads, kv_heads, dim, page, groups, new=None, *, seed=0, loose=0, wide=True, **kw):
    """``wide``: tables with as many (missing) blocks behind the contexts as make the call one that is attended by group. ``groups``: [(prefix, [own tokens of each request])]; own tokens count the new ones. Whole blocks of a prefix are the group's, the
    block it ends in is a copy of each request. ``loose``: requests behind the last group, which share nothing."""
    contexts = [p + n for p, own in groups for n in own] + [20 + 7 * i for i in range(loose)]
    p = PP.make(heads, kv_heads, dim, page, contexts, new, seed=seed, **kw)
    tables, k, v = p["tables"], p["k"], p["v"]
    first = 0
    for prefix, own in groups:
        for r in range(first + 1, first + len(own)):
            full = prefix // page
            for x in range(-(-prefix // page)):
                if x < full:
                    tables[r][x] = tables[first][x]
                elif contexts[r] > x * page and contexts[first] > x * page:
                    n = min(prefix - x * page, contexts[r] - x * page, contexts[first] - x * page)
                    k[tables[r][x], :n], v[tables[r][x], :n] = k[tables[first][x], :n], v[tables[first][x], :n]
        first += len(own)
    cu = [0]
    for _, own in groups:
        cu.append(cu[-1] + len(own))
    as_int = lambda x: torch.tensor(x, dtype=torch.int32, device="cuda")  # noqa: E731
    args = list(p["args"])
    if not kw.get("interleaved"):
        args[1], args[2] = k.cuda(), v.cuda()
    args[3] = as_int(tables)
    p["args"] = tuple(args)
    p["groups"] = (as_int([g[0] for g in groups]), as_int(cu))
    if wide and page % 8 == 0 and len(contexts) > len(groups):
        widen(p)
    return p


def widen(p):
    args = list(p["args"])
    for _ in range(40):
        if way(p):
            return
        args[3] = torch.nn.functional.pad(args[3], (0, args[3].size(1)), value=-1)
        p["args"] = tuple(args)
    assert way(p)


def call(p, **kw):
    f = A.shared_prefix_decode_attention if p["cu"] is None else A.shared_prefix_prefill_attention
    return f(*p["args"], *p["groups"], scale=p["scale"], **kw)


HEADS = [(16, 2, 64), (16, 2, 128), (32, 8, 128), (4, 4, 64), (3, 1, 128), (14, 2, 64), (12, 1, 64), (16, 1, 128), (40, 2, 64), (1, 1, 128)]


@pytest.mark.parametrize("dtype", [BF16, FP16])
@pytest.mark.parametrize("heads", HEADS)
def test_decode_heads(heads, dtype):
    p = make(*heads, 16, [(100, [1, 2, 17, 40]), (129, [1]), (300, [5, 60, 1, 130, 3])], dtype=dtype, seed=sum(heads))
    PP.check(p, *call(p, return_lse=True), f"{heads}")


@pytest.mark.parametrize("prefix", [0, 1, 7, 8, 15, 16, 17, 127, 128, 129, 255, 256, 257, 1000])
@pytest.mark.parametrize("dim", [64, 128])
def test_decode_prefixes(prefix, dim):
    p = make(16, 2, dim, 16, [(prefix, [1, 30, 2, 1, 64])], seed=prefix)
    PP.check(p, *call(p, return_lse=True), f"prefix of {prefix}")


@pytest.mark.parametrize("page", [1, 3, 8, 12, 24, 48, 64, 256])
def test_decode_pages(page):
    p = make(16, 2, 64, page, [(77, [1, 20, 3]), (300, [1, 2])], seed=page)
    PP.check(p, *call(p, return_lse=True), f"pages of {page}")


@pytest.mark.parametrize("dim", [64, 128])
@pytest.mark.parametrize("n,groups,prefix,own", [(2, 1, 5000, 3), (3, 1, 700, 3000), (40, 2, 400, 90), (90, 1, 200, 40), (200, 5, 150, 30), (80, 40, 60, 20),
                                                 (130, 65, 33, 5), (5, 5, 100, 9), (64, 1, 4000, 1)])
def test_decode_sizes(n, groups, prefix, own, dim):
    """Many and few requests, groups of one among them, more groups than a warp has lanes; one long prefix in many parts."""
    rng = random.Random(n)
    each = [n // groups + (i < n % groups) for i in range(groups)]
    p = make(16, 2, dim, 16, [(rng.randint(prefix // 2, prefix), [rng.randint(1, own) for _ in range(m)]) for m in each], seed=n)
    out, lse = call(p, return_lse=True)
    PP.check(p, out, lse, f"{n} requests")
    again = call(p)
    assert torch.equal(out, again)  # the same bits from run to run
    assert N.device_status() == 0


@pytest.mark.parametrize("n,groups", [(513, 3), (600, 300), (511, 40)])
def test_decode_many_requests(n, groups):
    """More rows than are put in order, more groups than a warp has lanes."""
    each = [n // groups + (i < n % groups) for i in range(groups)]
    p = make(4, 2, 64, 8, [(9 + 5 * i % 40, [1 + (i + j) % 7 for j in range(m)]) for i, m in enumerate(each)], seed=n, loose=2)
    out, lse = call(p, return_lse=True)
    PP.check(p, out, lse, f"{n} requests")
    assert torch.equal(out, call(p)) and N.device_status() == 0


def test_decode_requests_of_no_group():
    p = make(16, 2, 64, 16, [(64, [1, 5, 9])], loose=4)
    PP.check(p, *call(p, return_lse=True))
    lens, cu = p["groups"]
    for bad in ([2, 9], [-1, 3], [3, 1], [0, 0], [7, 7], [0, 8], [6, 100]):  # groups that leave the requests, or have none: nobody shares
        p["groups"] = (lens, torch.tensor(bad, dtype=torch.int32, device="cuda"))
        PP.check(p, *call(p, return_lse=True), f"{bad}")
    p["groups"] = (torch.tensor([-5], dtype=torch.int32, device="cuda"), cu)  # a prefix of less than none
    PP.check(p, *call(p, return_lse=True))
    p["groups"] = (lens[:0].contiguous(), cu[:1].contiguous())
    PP.check(p, *call(p, return_lse=True), "no groups")


@pytest.mark.parametrize("dim", [64, 128])
def test_decode_contexts_inside_the_prefix(dim):
    """Requests that are shorter than what they would share see no more than they have; of no key at all zeros."""
    p = make(16, 2, dim, 16, [(200, [10, 1, 30, 2])], seed=2)
    p["contexts"] = [210, 90, 0, 200]
    args = list(p["args"])
    args[4] = torch.tensor(p["contexts"], dtype=torch.int32, device="cuda")
    p["args"] = tuple(args)
    out, lse = call(p, return_lse=True)
    PP.check(p, out, lse)
    assert bool((out[2] == 0).all()) and bool((lse[2] == -math.inf).all())
    args[4] = torch.tensor([-1, 0, -7, 0], dtype=torch.int32, device="cuda")
    p["args"] = tuple(args)
    assert bool((call(p) == 0).all())


def test_stale_rows_do_not_count():
    """NaN in every cache row that no request sees, behind the prefix's keys of a block too."""
    p = make(16, 2, 64, 32, [(70, [1, 3, 9]), (33, [31, 1])], seed=6, poison=True)
    for name in ("k", "v"):  # (the shared blocks' rows behind the prefix, and the copies' unused first blocks, are nobody's)
        c = p[name]
        used = torch.zeros(c.shape[:2], dtype=torch.bool)
        for r, ctx in enumerate(p["contexts"]):
            for j in range(ctx):
                used[p["tables"][r][j // 32], j % 32] = True
        c[~used] = math.nan
        assert not c[used].isnan().any()
    args = list(p["args"])
    args[1], args[2] = p["k"].cuda(), p["v"].cuda()
    p["args"] = tuple(args)
    PP.check(p, *call(p, return_lse=True))


def test_missing_blocks_and_tables_that_end():
    p = make(16, 2, 64, 16, [(160, [5, 40, 9])], seed=7)
    width = p["args"][3].size(1)
    for r in range(3):
        p["tables"][r][3] = -1
        p["tables"][r][7] = p["k"].size(0)
    p["contexts"] = [165, 2 ** 31 - 1, 169]
    args = list(p["args"])
    padded = lambda: torch.tensor([t + [-1] * (width - len(t)) for t in p["tables"]], dtype=torch.int32, device="cuda")  # noqa: E731
    args[3] = padded()
    args[4] = torch.tensor(p["contexts"], dtype=torch.int32, device="cuda")
    p["args"] = tuple(args)
    p["contexts"] = [165, len(p["tables"][1]) * 16, 169]
    PP.check(p, *call(p, return_lse=True))
    p["groups"] = (torch.tensor([2 ** 31 - 1], dtype=torch.int32, device="cuda"), p["groups"][1])  # a prefix behind the table's end
    for r in (1, 2):
        p["tables"][r] = list(p["tables"][0])
    args[3] = padded()
    p["args"] = tuple(args)
    assert way(p) == 1
    PP.check(p, *call(p, return_lse=True))


@pytest.mark.parametrize("dtype", [BF16, FP16])
@pytest.mark.parametrize("heads", [(16, 2, 64), (16, 2, 128), (32, 8, 128), (3, 1, 128), (14, 2, 64), (40, 2, 64), (8, 8, 64)])
def test_prefill(heads, dtype):
    groups = [(100, [1, 12, 30]), (257, [40, 3]), (64, [20])]
    p = make(*heads, 16, groups, [1, 5, 30, 17, 3, 20], dtype=dtype, seed=sum(heads), behind=3, loose=0)
    out = torch.full_like(p["args"][0], 7.0)
    got, lse = call(p, out=out, return_lse=True)
    assert got is out
    PP.check(p, out, lse, f"{heads}")
    assert bool((out[-3:] == 7).all())


@pytest.mark.parametrize("dim", [64, 128])
@pytest.mark.parametrize("n,prefix,own,new", [(2, 3000, 4000, 40), (24, 1500, 60, 12), (5, 129, 300, 300), (3, 8000, 16, 16), (70, 64, 9, 4)])
def test_prefill_sizes(n, prefix, own, new, dim):
    rng = random.Random(n)
    news = [rng.randint(1, new) for _ in range(n)]
    owns = [rng.randint(m, max(m, own)) for m in news]
    cut = n // 2
    p = make(16, 2, dim, 16, [(prefix, owns[:cut]), (prefix // 2, owns[cut:])], news, seed=n)
    out, lse = call(p, return_lse=True)
    PP.check(p, out, lse, f"{n} requests")
    assert torch.equal(out, call(p))
    assert N.device_status() == 0


def test_prefill_many_requests():
    """Packed: 700 tokens of 140 requests in 70 groups, some without new tokens, some rows of no sequence."""
    new = [(3 * i) % 11 for i in range(140)]
    p = make(8, 2, 64, 16, [(20 + 3 * i % 90, [new[2 * i] + 1, new[2 * i + 1] + 4]) for i in range(70)], new, seed=1, behind=5)
    out = torch.full_like(p["args"][0], 7.0)
    _, lse = call(p, out=out, return_lse=True)
    PP.check(p, out, lse)
    assert bool((out[-5:] == 7).all()) and N.device_status() == 0


@pytest.mark.parametrize("page", [8, 12, 24, 256])
def test_prefill_pages(page):
    p = make(16, 2, 64, page, [(130, [9, 20]), (77, [5, 6, 100])], [9, 3, 5, 1, 70], seed=page)
    PP.check(p, *call(p, return_lse=True), f"pages of {page}")


@pytest.mark.parametrize("dim", [64, 128])
def test_prefill_tokens_inside_the_prefix(dim):
    """The request that brings the prefix, in the same batch: its tokens see it up to themselves. And requests without new tokens."""
    p = make(16, 2, dim, 16, [(150, [10, 1, 30, 2])], [160, 1, 0, 60], seed=2)
    PP.check(p, *call(p, return_lse=True))


@pytest.mark.parametrize("prefill", [False, True])
def test_strided(prefill):
    p = make(16, 2, 128, 32, [(96, [70, 1, 33])], [7, 1, 20] if prefill else None, seed=5)
    q, k, v, *rest = p["args"]
    both = torch.empty(k.size(0), 2, 2, 32, 128, dtype=BF16, device="cuda")  # k and v of a block in one tensor, heads ahead of positions
    both[:, 0], both[:, 1] = k.transpose(1, 2), v.transpose(1, 2)
    T = q.size(0)
    packed = torch.randn(T, 20 * 128 + 8, device="cuda").to(BF16)
    packed[:, 8:8 + 16 * 128] = q.view(T, -1)
    q = packed[:, 8:8 + 16 * 128].view(T, 16, 128)
    p["args"] = (q, both[:, 0].transpose(1, 2), both[:, 1].transpose(1, 2), *rest)
    wide = torch.full((T, 24, 128), 3.0, device="cuda", dtype=BF16)
    call(p, out=wide[:, 4:20])
    PP.check(p, wide[:, 4:20])
    assert bool((wide[:, :4] == 3).all()) and bool((wide[:, 20:] == 3).all())
    want = wide[:, 4:20].clone()
    q1 = q[:, :1].expand(T, 16, 128)  # strides of zero, which a tensor map refuses: request by request
    p["q"] = q1.cpu()
    p["args"] = (q1, *p["args"][1:])
    PP.check(p, call(p))
    p["args"] = (q, *p["args"][1:])
    call(p, out=q)  # in place: what the second launch reads of q lies ahead of what it writes
    assert torch.equal(q, want)


@pytest.mark.parametrize("prefill", [False, True])
def test_graphs_and_streams(prefill):
    p = make(16, 2, 64, 16, [(2500, [9, 40, 3]), (300, [1, 2])], [9, 4, 3, 1, 2] if prefill else None, seed=8)
    want = call(p)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        got = call(p)
    side.synchronize()
    assert torch.equal(got, want)
    graphs, outs = [], []
    for _ in range(2):  # two graphs, each with a workspace of its own
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            outs.append(call(p))
        graphs.append(g)
    streams = [torch.cuda.Stream() for _ in graphs]
    for _ in range(5):
        for g, s in zip(graphs, streams):
            with torch.cuda.stream(s):
                g.replay()
    torch.cuda.synchronize()
    assert all(torch.equal(o, want) for o in outs)
    # replayed over other lengths, prefixes and queries
    q, lens, (prefix, cu) = p["args"][0], p["args"][4], p["groups"]
    q.mul_(0.5)
    p["q"] = q.cpu()
    prefix.copy_(torch.tensor([2000, 0], dtype=torch.int32))
    for g in graphs:
        g.replay()
    torch.cuda.synchronize()
    for o in outs:
        PP.check(p, o)


def test_queries_and_rows_of_the_launch_ahead():
    """What writes q and the newest rows runs right ahead of the call, again and again: neither launch may read them early."""
    p = make(16, 2, 64, 16, [(500, [9, 40, 3, 80])], seed=3)
    q, k, v, tables, lens = p["args"]
    qs = [torch.randn_like(q) for _ in range(4)]
    news = [torch.randn(4, 2, 64, device="cuda").to(BF16) for _ in range(4)]
    at = lens.long() - 1
    rows = tables.long()[torch.arange(4, device="cuda"), at // 16], at % 16
    outs = []
    for r in range(200):
        q.copy_(qs[r % 4])
        k[rows] = news[r % 4]
        v[rows] = news[(r + 1) % 4]
        outs.append(call(p))
    torch.cuda.synchronize()
    assert all(torch.equal(outs[r], outs[r % 4]) for r in range(200))
    assert not torch.equal(outs[0], outs[1])
    q.copy_(qs[3])
    p["q"], p["k"], p["v"] = q.cpu(), k.cpu(), v.cpu()
    PP.check(p, outs[199])


@pytest.mark.parametrize("prefill", [False, True])
def test_narrow_tables_go_request_by_request(prefill):
    """Where a second launch would not pay: the other calls' result, bit for bit."""
    p = make(16, 2, 64, 16, [(100, [9, 40, 3])], [9, 4, 3] if prefill else None, wide=False)
    assert way(p) == 0
    f = A.paged_prefill_attention if prefill else A.paged_decode_attention
    assert torch.equal(call(p), f(*p["args"]))


def test_ways():
    """Both launches of a call: items by clusters and by CTAs as they come, in either head size; the rule's line."""
    for dim, n in ((64, 4), (64, 200), (128, 4), (128, 200)):
        p = make(16, 2, dim, 64, [(700, [5 + i % 90 for i in range(n)])], seed=n)
        assert way(p) == 1
        PP.check(p, *call(p, return_lse=True), f"{n} requests, heads of {dim}")
    ask = N.lib().lora_b200_shared_prefix_way
    assert ask(64, 64, 1, 32, 8, 128, 512, 16, 0) == 1 and ask(64, 64, 1, 16, 2, 64, 10, 256, 0) == 0
    assert ask(64, 64, 64, 32, 8, 128, 512, 16, 0) == 0 and ask(64, 64, 1, 32, 8, 128, 512, 12, 0) == 0 and ask(64, 64, 0, 32, 8, 128, 512, 16, 0) == 0


def test_same_as_request_by_request():
    """Against the calls that know of no groups: what differs is the order of sums."""
    p = make(16, 2, 64, 16, [(700, [9, 40, 3, 80, 1])], seed=13)
    one, lse = A.paged_decode_attention(*p["args"], return_lse=True)
    two, lse2 = call(p, return_lse=True)
    assert float((one.float() - two.float()).abs().max()) <= 4 * 2.0 ** -8 * float(p["v"].float().abs().max())
    assert float((lse - lse2).abs().max()) <= 1e-5 * float(lse.abs().max()) + 1e-5
