"""Differential attention over the paged cache against the 64-bit form."""

import math

import pytest
import torch

import paged_problem as PP
from nanovllm_voxcpm_b200 import _native as N
from nanovllm_voxcpm_b200 import attention as A
from oracle import more_attention_oracle as MO

pytestmark = pytest.mark.gpu
BF16, FP16 = torch.bfloat16, torch.float16
EPS = 1e-5


def make(heads, kv_heads, dim, page, contexts, new=None, *, per_token=False, norm=True, seed=0, **kw):
    p = PP.make(heads, kv_heads, dim, page, contexts, new, seed=seed, **kw)
    gen = torch.Generator().manual_seed(seed + 77)
    T = p["q"].size(0)
    p["lam"] = torch.sigmoid(torch.randn(*((T, heads) if per_token else (heads,)), generator=gen))
    p["weight"] = (0.8 + 0.2 * torch.randn(dim, generator=gen)).to(p["q"].dtype) if norm else None
    p["scale"] = (dim // 2) ** -0.5
    return p


def call(p, **kw):
    how = dict(norm_weight=None if p["weight"] is None else p["weight"].cuda(), eps=EPS, window=p["window"], sinks=p["sinks"], **kw)
    f = A.differential_decode_attention if p["cu"] is None else A.differential_prefill_attention
    return f(*p["args"], p["lam"].cuda(), **how)


def check(p, out, what=""):
    """A map's result before its rounding is off by (u (1 + u) + eps) size (+ keys 2^-25 max |v| in fp16), as ``paged_problem.check``
    derives it with half of the columns in a score; the difference of two by the sum e of both, the second times lam, and four fp32
    roundings. The root of the mean square n of a head is 1-Lipschitz in that of the errors E, so that y / n is off by at most
    (e + |y| E / n) / (n - E), n - E no less than sqrt(eps); the sum of the squares of D terms in fp32 adds D 2^-24. Then one rounding u."""
    q, dim = p["q"], p["q"].size(-1)
    u = torch.finfo(q.dtype).eps / 2
    one, two, count = MO.two_maps(q, p["k"], p["v"], p["tables"], p["contexts"], p["cu"], p["scale"], p["window"], p["sinks"])
    lam = p["lam"].double().expand(q.shape[:2])[..., None]
    k_finite = p["k"].float().nan_to_num(0, 0, 0)
    top = float(p["v"].float().nan_to_num(0, 0, 0).abs().max())
    half = dim // 2
    err = 0
    for m, (_, size) in enumerate((one, two)):
        cols = slice(m * half, (m + 1) * half)
        score_err = half * 2.0 ** -24 * p["scale"] * float(q[..., cols].float().norm(dim=-1).max()) * float(k_finite[..., cols].norm(dim=-1).max())
        eps = 2 * score_err + 2.0 ** -18 + count.double()[:, None, None] * 2.0 ** -23
        mine = (u * (1 + u) + eps) * size + (count[:, None, None] * 2.0 ** -25 * top if q.dtype == FP16 else 0)
        err = err + (mine if m == 0 else lam * mine)
    y = one[0] - lam * two[0]
    err = err + 2.0 ** -22 * (one[1] + lam * two[1])
    if p["weight"] is not None:
        eps = p.get("eps", EPS)
        n = (y.square().mean(-1, keepdim=True) + eps).sqrt()
        E = err.square().mean(-1, keepdim=True).sqrt()
        w = p["weight"].double()
        want = MO.rms_norm(y, w, eps)
        bound = w.abs() * (err + y.abs() * E / n) / torch.clamp(n - E, min=eps ** 0.5) + (dim + 16) * 2.0 ** -24 * want.abs()
    else:
        want, bound = y, err
    bound = u * want.abs() + (1 + u) * bound + (2.0 ** -25 if q.dtype == FP16 else 0)
    rows = ~one[0][:, 0, 0].isnan()
    got = out.double().cpu()
    assert not got[rows].isnan().any(), f"{what}: NaN"
    off = (got - want).abs()[rows]
    assert bool((off <= bound[rows] + 1e-30).all()), f"{what}: worst {float((off / (bound[rows] + 1e-30)).max()):.3g} of the bound"


HEADS = [(16, 2, 64), (16, 2, 128), (32, 8, 128), (4, 4, 64), (3, 1, 128), (14, 2, 64), (12, 1, 64), (16, 1, 128), (40, 2, 64), (1, 1, 128)]


@pytest.mark.parametrize("norm", [False, True])
@pytest.mark.parametrize("dtype", [BF16, FP16])
@pytest.mark.parametrize("heads", HEADS)
def test_decode_heads(heads, dtype, norm):
    p = make(*heads, 16, [1, 2, 15, 16, 17, 31, 32, 33, 127, 128, 129, 300], dtype=dtype, norm=norm, seed=sum(heads))
    check(p, call(p), f"{heads}")


@pytest.mark.parametrize("page", [1, 3, 7, 8, 16, 24, 48, 100, 256])
def test_decode_pages(page):
    p = make(16, 2, 64, page, [1, 50, 257, 513], seed=page, poison=True, per_token=True)
    check(p, call(p), f"pages of {page}")


@pytest.mark.parametrize("dim", [64, 128])
@pytest.mark.parametrize("window,sinks", [(1, 0), (1, 1), (7, 3), (64, 4), (100, 129), (256, 0), (1000, 4), (2 ** 31 - 1, 5)])
def test_decode_window_and_sinks(window, sinks, dim):
    p = make(16, 2, dim, 16, [1, 2, 7, 8, 64, 65, 130, 400, 777], window=window, sinks=sinks, seed=window % 97, poison=True, norm=False)
    check(p, call(p), f"window {window}, {sinks} sinks")


@pytest.mark.parametrize("dim", [64, 128])
@pytest.mark.parametrize("n,context,width", [(1, 333, 0), (1, 20000, 0), (2, 5000, 0), (7, 3000, 0), (40, 700, 0), (160, 100, 0), (24, 2500, 4000)])
def test_decode_ways(n, context, width, dim):
    """Items by one CTA each, by clusters of two to eight, by equal shares of all blocks with a join; the last by the table's width."""
    p = make(16, 2, dim, 16, [context - 7 * i % context for i in range(n)], seed=n, norm=dim == 64)
    args = list(p["args"])
    if width:
        args[3] = torch.nn.functional.pad(args[3], (0, width - args[3].size(1)), value=-1)
        p["args"] = tuple(args)
    out = call(p)
    check(p, out, f"{n} of {context}")
    assert torch.equal(out, call(p))


def test_no_keys_are_zeros():
    p = make(8, 2, 64, 16, [0, 5, 0, 40, 0], poison=True)
    out = call(p)
    check(p, out)
    assert bool((out[[0, 2, 4]] == 0).all())


@pytest.mark.parametrize("dim", [64, 128])
def test_equal_maps_cancel(dim):
    """Maps that are the same, lam = 1: the difference is exactly zero, and so is its norm."""
    p = make(8, 2, dim, 16, [1, 17, 300], seed=4)
    q, k = p["args"][0], p["args"][1]
    q[..., dim // 2:] = q[..., :dim // 2]
    k[..., dim // 2:] = k[..., :dim // 2]
    p["lam"] = torch.ones(8)
    assert bool((call(p) == 0).all())
    p["lam"] = torch.zeros(8)  # and none of the second map: the plain attention of the first half
    p["weight"] = None
    p["q"], p["k"] = q.cpu(), k.cpu()
    check(p, call(p))


@pytest.mark.parametrize("new,contexts", [([1], [1]), ([5, 1, 40], [5, 100, 40]), ([129, 16, 17], [129, 500, 17]), ([300], [700]), ([0, 3, 0, 2], [9, 3, 0, 50]),
                                          ([64] * 9, [64 + 37 * i for i in range(9)])])
@pytest.mark.parametrize("heads", [(16, 2, 64), (16, 2, 128), (3, 1, 128), (8, 8, 64), (14, 2, 64)])
def test_prefill(heads, new, contexts):
    p = make(*heads, 16, contexts, new, seed=len(new), poison=True, behind=3, per_token=len(new) % 2 == 0)
    out = torch.full_like(p["args"][0], 7.0)
    assert call(p, out=out) is out
    check(p, out, f"{heads} {new}")
    assert bool((out[sum(new):] == 7).all())


@pytest.mark.parametrize("dtype", [BF16, FP16])
@pytest.mark.parametrize("dim", [64, 128])
@pytest.mark.parametrize("window,sinks", [(1, 0), (5, 2), (100, 0), (128, 4), (300, 40), (2 ** 31 - 1, 1)])
def test_prefill_window(window, sinks, dim, dtype):
    p = make(16, 2, dim, 16, [260, 700, 1], [260, 130, 1], window=window, sinks=sinks, seed=3, poison=True, dtype=dtype)
    check(p, call(p), f"window {window}, {sinks} sinks")


@pytest.mark.parametrize("page", [8, 12, 24, 64, 256])
@pytest.mark.parametrize("dim", [64, 128])
def test_prefill_pages(page, dim):
    p = make(16, 2, dim, page, [300, 140], [100, 140], seed=page, poison=True)
    check(p, call(p), f"pages of {page}")


@pytest.mark.parametrize("new,context", [(16, 8000), (200, 6000), (1000, 1500)])
@pytest.mark.parametrize("heads", [(16, 2, 64), (16, 2, 128)])
def test_prefill_behind_long_contexts(heads, new, context):
    """Items that are cut along the keys and joined."""
    p = make(*heads, 64, [context], [new], seed=new)
    out = call(p)
    check(p, out)
    assert torch.equal(out, call(p))


@pytest.mark.parametrize("prefill", [False, True])
def test_strided(prefill):
    """q as columns of packed rows, out as columns of a wider buffer, heads-first cache, lam by token with strides, in place."""
    p = make(16, 2, 128, 32, [70, 1, 333], [7, 1, 50] if prefill else None, interleaved=True, seed=5, per_token=True)
    q = p["args"][0]
    T = q.size(0)
    packed = torch.randn(T, 20 * 128 + 8, device="cuda").to(BF16)
    packed[:, 8:8 + 16 * 128] = q.view(T, -1)
    q = packed[:, 8:8 + 16 * 128].view(T, 16, 128)
    p["args"] = (q, *p["args"][1:])
    p["lam"] = p["lam"].t().contiguous().t()
    wide = torch.full((T, 24, 128), 3.0, device="cuda", dtype=BF16)
    call(p, out=wide[:, 4:20])
    check(p, wide[:, 4:20])
    assert bool((wide[:, :4] == 3).all()) and bool((wide[:, 20:] == 3).all())
    want = wide[:, 4:20].clone()
    call(p, out=q)  # (a row of q is read before it is written)
    assert torch.equal(q, want)


def test_scalar_lam_by_strides():
    """One lam for all heads and tokens: a [1] tensor, expanded."""
    p = make(8, 2, 64, 16, [9, 100])
    one = torch.full((1,), 0.37, device="cuda")
    a = A.differential_decode_attention(*p["args"], one.expand(8))
    b = A.differential_decode_attention(*p["args"], one.expand(2, 8))
    c = A.differential_decode_attention(*p["args"], torch.full((2, 8), 0.37, device="cuda"))
    assert torch.equal(a, b) and torch.equal(a, c)
    p["lam"], p["weight"] = torch.full((8,), 0.37), None
    check(p, a)


@pytest.mark.parametrize("prefill", [False, True])
def test_graph_and_streams(prefill):
    p = make(16, 2, 64, 16, [2500, 40], [20, 40] if prefill else None, seed=8)
    want = call(p)
    lam, weight = p["lam"].cuda(), p["weight"].cuda()
    f = A.differential_prefill_attention if prefill else A.differential_decode_attention
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        got = f(*p["args"], lam, norm_weight=weight, eps=EPS)
    side.synchronize()
    assert torch.equal(got, want)
    graphs, outs = [], []
    for _ in range(2):  # two graphs, each with a workspace of its own
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            outs.append(f(*p["args"], lam, norm_weight=weight, eps=EPS))
        graphs.append(g)
    streams = [torch.cuda.Stream() for _ in graphs]
    for _ in range(3):
        for g, s in zip(graphs, streams):
            with torch.cuda.stream(s):
                g.replay()
    torch.cuda.synchronize()
    assert all(torch.equal(o, want) for o in outs)
    assert N.device_status() == 0


def test_values_that_are_not_finite():
    """A NaN in a key or a value reaches the heads and requests that see it, and no others; an infinite lam gives no surprise elsewhere."""
    p = make(4, 2, 64, 16, [40, 40], norm=False)
    base = call(p)
    k = p["args"][1].clone()
    k[p["tables"][0][0], 3, 1, 5] = math.nan  # first half of kv head 1: map 1 of heads 2 and 3 of request 0
    got = A.differential_decode_attention(p["args"][0], k, *p["args"][2:], p["lam"].cuda())
    assert bool(got[0, 2:].isnan().all())
    assert torch.equal(got[0, :2], base[0, :2]) and torch.equal(got[1], base[1])
