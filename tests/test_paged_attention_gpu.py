"""Decode and prefill attention over the paged cache against the 64-bit form; bounds in ``paged_problem.check``."""

import pytest
import torch

import paged_problem as PP
from nanovllm_voxcpm_b200 import _native as N
from nanovllm_voxcpm_b200 import attention as A

pytestmark = pytest.mark.gpu
BF16, FP16 = torch.bfloat16, torch.float16


def _decode(p, **kw):
    return A.paged_decode_attention(*p["args"], scale=p["scale"], window=p["window"], sinks=p["sinks"], **kw)


def _prefill(p, **kw):
    return A.paged_prefill_attention(*p["args"], scale=p["scale"], window=p["window"], sinks=p["sinks"], **kw)


HEADS = [(16, 2, 64), (16, 2, 128), (32, 8, 128), (4, 4, 64), (3, 1, 128), (14, 2, 64), (12, 1, 64), (16, 1, 128), (40, 2, 64), (1, 1, 128)]


@pytest.mark.parametrize("dtype", [BF16, FP16])
@pytest.mark.parametrize("heads", HEADS)
def test_decode_heads(heads, dtype):
    p = PP.make(*heads, 16, [1, 2, 15, 16, 17, 31, 32, 33, 127, 128, 129, 300], dtype=dtype, seed=sum(heads))
    PP.check(p, *_decode(p, return_lse=True), f"{heads}")


@pytest.mark.parametrize("page", [1, 3, 7, 8, 16, 24, 48, 100, 256])
def test_decode_pages(page):
    p = PP.make(16, 2, 64, page, [1, 50, 257, 513], seed=page, poison=True)
    PP.check(p, *_decode(p, return_lse=True), f"pages of {page}")


@pytest.mark.parametrize("dtype", [BF16, FP16])
@pytest.mark.parametrize("dim", [64, 128])
@pytest.mark.parametrize("window,sinks", [(1, 0), (1, 1), (7, 3), (64, 4), (100, 129), (256, 0), (1000, 4), (2 ** 31 - 1, 5)])
def test_decode_window_and_sinks(window, sinks, dim, dtype):
    p = PP.make(16, 2, dim, 16, [1, 2, 7, 8, 64, 65, 130, 400, 777], window=window, sinks=sinks, dtype=dtype, seed=window % 97, poison=True)
    PP.check(p, *_decode(p, return_lse=True), f"window {window}, {sinks} sinks")


def test_decode_requests_without_keys():
    """Contexts of zero (and below): zeros, -inf; their table entries are not used."""
    p = PP.make(8, 2, 64, 16, [0, 5, 0, 40, 0], poison=True)
    out, lse = _decode(p, return_lse=True)
    PP.check(p, out, lse)
    assert bool((out[[0, 2, 4]] == 0).all()) and bool((lse[[0, 2, 4]] == -float("inf")).all())
    args = list(p["args"])
    args[4] = torch.tensor([-3, 0, 0, 0, 0], dtype=torch.int32, device="cuda")
    assert bool((A.paged_decode_attention(*args) == 0).all())
    assert bool((A.paged_decode_attention(*args[:3], args[3][:, :0], p["args"][4]) == 0).all())


def test_decode_entries_outside_the_cache():
    """Missing blocks, blocks behind the cache and contexts behind the table: such keys are left out."""
    p = PP.make(16, 2, 64, 16, [200, 100, 90], seed=3)
    p["tables"][0][2], p["tables"][0][5], p["tables"][1][0] = -1, 2 ** 31 - 1, p["k"].size(0)
    p["tables"][2] = [-7] * len(p["tables"][2])
    args = list(p["args"])
    args[3] = torch.tensor(p["tables"], dtype=torch.int32, device="cuda")
    out, lse = A.paged_decode_attention(*args, return_lse=True)
    PP.check(p, out, lse)
    assert bool((out[2] == 0).all())
    p["contexts"] = [10 ** 9, 2 ** 31 - 1, 90]
    args[4] = torch.tensor(p["contexts"], dtype=torch.int32, device="cuda")
    p["contexts"] = [len(p["tables"][0]) * 16] * 2 + [90]  # without a window the same keys
    PP.check(p, *A.paged_decode_attention(*args, return_lse=True))


@pytest.mark.parametrize("dtype", [BF16, FP16])
def test_decode_strided(dtype):
    """q as columns of packed rows, out as columns of a wider buffer, k and v of a block in one tensor with heads first."""
    p = PP.make(16, 2, 128, 32, [70, 1, 333], dtype=dtype, interleaved=True, seed=5)
    q, *rest = p["args"]
    packed = torch.randn(3, 20 * 128 + 8, device="cuda").to(dtype)
    packed[:, 8:8 + 16 * 128] = q.view(3, -1)
    wide = torch.full((3, 16, 136 + 8), 7.0, device="cuda", dtype=dtype)
    view = packed[:, 8:8 + 16 * 128].view(3, 16, 128)
    out = A.paged_decode_attention(view, *rest, scale=p["scale"], out=wide[:, :, 8:136])
    assert out.data_ptr() == wide[:, :, 8:].data_ptr()
    PP.check(p, out)
    assert bool((wide[:, :, :8] == 7).all()) and bool((wide[:, :, 136:] == 7).all())


@pytest.mark.parametrize("heads,contexts", [((16, 2, 128), [2500]), ((32, 8, 128), [700]), ((16, 2, 64), [900, 3, 0, 1024]), ((12, 1, 128), [1500] * 3),
                                            ((40, 2, 64), [2100, 1]), ((16, 2, 64), [1000] * 40), ((16, 2, 64), [300] * 200), ((8, 8, 64), [5] * 60)])
def test_decode_ways(heads, contexts):
    """One CTA an item, clusters of them, with four and with eight warps; run to run the same."""
    p = PP.make(*heads, 32, contexts, seed=len(contexts), poison=True)
    out, lse = _decode(p, return_lse=True)
    PP.check(p, out, lse)
    for _ in range(3):
        again, lse2 = _decode(p, return_lse=True)
        assert torch.equal(again, out) and torch.equal(lse2, lse)


@pytest.mark.parametrize("contexts", [[5000], [9000, 1, 30], [40] * 700, [3000] * 20, list(range(0, 640, 5))])
def test_decode_shares_of_the_work(contexts):
    """One long request over many CTAs, many short ones over few, shares that begin and end inside requests; run to run the same."""
    p = PP.make(8, 2, 64, 64, contexts, seed=len(contexts))
    out, lse = _decode(p, return_lse=True)
    PP.check(p, out, lse)
    for _ in range(5):
        again, lse2 = _decode(p, return_lse=True)
        assert torch.equal(again, out) and torch.equal(lse2, lse)


def test_decode_far_offsets():
    """A cache whose last block lies past 2^31 elements."""
    far = 2 ** 31 + 4096
    store = torch.zeros(far + 4 * 16 * 2 * 64, dtype=BF16, device="cuda")
    p = PP.make(4, 2, 64, 16, [30], seed=9, spare=0)
    order = p["tables"][0]
    k = store.as_strided((2, 16, 2, 64), (far, 256, 64, 1))
    v = store.as_strided((2, 16, 2, 64), (far, 256, 64, 1), 128)
    k.copy_(p["k"].cuda())
    v.copy_(p["v"].cuda())
    assert sorted(order) == [0, 1]
    PP.check(p, A.paged_decode_attention(p["args"][0], k, v, *p["args"][3:], scale=p["scale"]))


def test_decode_extreme_scores():
    """Scores of hundreds, all equal, and a maximum that grows block by block."""
    p = PP.make(8, 2, 64, 16, [500, 300], seed=2)
    p["k"] = p["k"] * torch.linspace(0.1, 30, p["k"].size(0)).view(-1, 1, 1, 1).to(BF16)
    args = list(p["args"])
    args[1] = p["k"].cuda()
    PP.check(p, *A.paged_decode_attention(*args, scale=p["scale"], return_lse=True))
    p["k"] = torch.zeros_like(p["k"])
    args[1] = p["k"].cuda()
    PP.check(p, *A.paged_decode_attention(*args, scale=p["scale"], return_lse=True))


PREFILL = [([1], [1]), ([37], [37]), ([128], [128]), ([129, 1, 5], [129, 1, 5]), ([300, 0, 17], [300, 9, 17]), ([16], [700]), ([1, 1, 1], [1, 300, 77]),
           ([200, 31], [500, 31]), ([0, 0], [4, 0])]


@pytest.mark.parametrize("dtype", [BF16, FP16])
@pytest.mark.parametrize("heads", [(16, 2, 64), (8, 2, 128), (3, 1, 64), (2, 2, 128), (12, 1, 128)])
@pytest.mark.parametrize("new,contexts", PREFILL)
def test_prefill(new, contexts, heads, dtype):
    p = PP.make(*heads, 16, contexts, new, dtype=dtype, seed=len(new) + sum(heads), poison=True, behind=3)
    out = torch.full_like(p["args"][0], 7.0)
    got, lse = _prefill(p, out=out, return_lse=True)
    PP.check(p, got, lse, f"{new} {contexts}")
    assert bool((out[sum(new):] == 7).all())


@pytest.mark.parametrize("page", [8, 16, 24, 48, 64, 128, 136, 256])
@pytest.mark.parametrize("window,sinks", [(0, 0), (1, 1), (50, 4), (128, 0), (200, 140)])
def test_prefill_pages_and_windows(page, window, sinks):
    p = PP.make(8, 1, 64, page, [333, 520, 40], [333, 120, 3], window=window, sinks=sinks, seed=page + window, poison=True)
    PP.check(p, *_prefill(p, return_lse=True), f"pages of {page}, window {window}, {sinks} sinks")


@pytest.mark.parametrize("page", [1, 7, 12, 100])
def test_prefill_pages_that_the_tile_kernel_does_not_take(page):
    p = PP.make(8, 2, 64, page, [130, 61], [30, 61], window=40, sinks=3, seed=page, poison=True)
    PP.check(p, *_prefill(p, return_lse=True), f"pages of {page}")


@pytest.mark.parametrize("heads", [(16, 2, 64), (8, 2, 128)])
@pytest.mark.parametrize("n", [31, 32, 33, 70])
def test_prefill_many_requests(n, heads):
    """More requests than a warp has lanes, empty ones and prompts of several blocks among them, some behind a context."""
    new = [(7 * i) % 41 if i % 9 else 150 + i for i in range(n)]
    p = PP.make(*heads, 16, [x + (i % 3) * 60 for i, x in enumerate(new)], new, seed=n, poison=True, behind=1)
    PP.check(p, *_prefill(p, return_lse=True), f"{n} requests")


def test_prefill_ranges_outside_the_rows():
    """Ranges that leave the rows of q, or run backwards, count as none; the others are served."""
    p = PP.make(8, 2, 64, 16, [40, 50, 60], [40, 50, 60], seed=6)
    q, k, v, tables, ctx, cu = p["args"]
    want = _prefill(p)
    for bad in ([0, 40, 90, 10 ** 6], [-5, 40, 90, 150], [0, 40, 30, 150], [200, 40, 90, 150]):
        out = torch.full_like(q, 7.0)
        A.paged_prefill_attention(q, k, v, tables, ctx, torch.tensor(bad, dtype=torch.int32, device="cuda"), scale=p["scale"], out=out)
        torch.cuda.synchronize()
        assert torch.equal(out[40:90], want[40:90]) or bad[2] == 30
    assert N.device_status() == 0


def test_prefill_tokens_ahead_of_their_context():
    """More new tokens than the context holds: the first ones have no position, see nothing and give zeros."""
    p = PP.make(8, 2, 64, 16, [5], [9], seed=4)
    out, lse = _prefill(p, return_lse=True)
    PP.check(p, out, lse)
    assert bool((out[:4] == 0).all()) and bool((lse[:4] == -float("inf")).all())


@pytest.mark.parametrize("dim", [64, 128])
@pytest.mark.parametrize("new,contexts,window,sinks", [([16], [6000], 0, 0), ([3, 1, 70], [4000, 9000, 3500], 0, 0), ([600], [4200], 0, 0),
                                                       ([40, 0, 5], [50, 7000, 4000], 3500, 200), ([1], [20000], 0, 0), ([9], [5], 0, 0)])
def test_prefill_shares_of_long_contexts(new, contexts, window, sinks, dim):
    """Few tokens behind long contexts: the keys of a block are shared out over the CTAs and joined; run to run the same."""
    p = PP.make(16, 2, dim, 64, contexts, new, window=window, sinks=sinks, seed=dim + len(new), poison=True, behind=2)
    pad = max(0, 4096 // 64 - p["args"][3].size(1))  # (the table's width is what tells how long contexts may be)
    args = list(p["args"])
    args[3] = torch.nn.functional.pad(args[3], (0, pad), value=-1)
    out = torch.full_like(args[0], 7.0)
    got, lse = A.paged_prefill_attention(*args, scale=p["scale"], window=window, sinks=sinks, out=out, return_lse=True)
    PP.check(p, got, lse, f"{new} {contexts}")
    assert bool((out[sum(new):] == 7).all())
    again, lse2 = A.paged_prefill_attention(*args, scale=p["scale"], window=window, sinks=sinks, return_lse=True)
    assert torch.equal(again[:sum(new)], got[:sum(new)]) and torch.equal(lse2[:sum(new)], lse[:sum(new)])


def test_prefill_rows_around_the_sequences():
    """cu_seqlens that begin behind row 0: rows ahead of the first and behind the last sequence stay as they are."""
    p = PP.make(8, 2, 128, 16, [40, 90], [40, 20], seed=8)
    q, k, v, tables, ctx, cu = p["args"]
    padded = torch.full((70, 8, 128), float("nan"), dtype=BF16, device="cuda")
    padded[6:66] = q
    out = torch.full_like(padded, 7.0)
    A.paged_prefill_attention(padded, k, v, tables, ctx, cu + 6, scale=p["scale"], out=out)
    PP.check(p, out[6:66])
    assert bool((out[:6] == 7).all()) and bool((out[66:] == 7).all())


def test_prefill_strided():
    p = PP.make(16, 2, 128, 32, [70, 300], [70, 61], dtype=FP16, interleaved=True, seed=5)
    q, *rest = p["args"]
    T = q.size(0)
    packed = torch.randn(T, 20 * 128 + 8, device="cuda").to(FP16)
    packed[:, 8:8 + 16 * 128] = q.view(T, -1)
    wide = torch.full((T, 16, 136 + 8), 7.0, device="cuda", dtype=FP16)
    out = A.paged_prefill_attention(packed[:, 8:8 + 16 * 128].view(T, 16, 128), *rest, scale=p["scale"], out=wide[:, :, 8:136])
    PP.check(p, out)
    assert bool((wide[:, :, :8] == 7).all()) and bool((wide[:, :, 136:] == 7).all())


@pytest.mark.parametrize("prefill", [False, True])
def test_graphs_and_streams(prefill):
    """Two graphs captured and replayed on two streams at once, new lengths and queries between replays, next to eager calls."""
    ps = [PP.make(16, 2, 64, 16, [900, 40, 300], [7, 40, 90] if prefill else None, seed=s) for s in (1, 2)]
    call = _prefill if prefill else _decode
    want = [call(p) for p in ps]
    streams = [torch.cuda.Stream() for _ in ps]
    graphs, outs = [], []
    for p, s in zip(ps, streams):
        s.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(s):
            call(p)
            s.synchronize()
            g = torch.cuda.CUDAGraph()
            with torch.cuda.graph(g, stream=s):
                outs.append(call(p))
        graphs.append(g)
    torch.cuda.synchronize()
    for _ in range(20):
        for g, s in zip(graphs, streams):
            with torch.cuda.stream(s):
                g.replay()
        eager = call(ps[0])
    torch.cuda.synchronize()
    assert torch.equal(eager, want[0]) and all(torch.equal(a, b) for a, b in zip(outs, want))
    short = [30, 40, 299] if not prefill else [800, 40, 91]
    ps[0]["args"][4].copy_(torch.tensor(short, dtype=torch.int32))
    ps[0]["contexts"] = short
    graphs[0].replay()
    torch.cuda.synchronize()
    PP.check(ps[0], outs[0])
    assert torch.equal(outs[0], call(ps[0]))


def test_two_parts_of_a_context_join():
    """What the log sums are for: attention over a window joined with attention over what lies ahead of it."""
    p = PP.make(8, 2, 64, 16, [320], seed=1)
    q, k, v, tables, ctx = p["args"]
    whole = A.paged_decode_attention(q, k, v, tables, ctx, scale=p["scale"])
    a, la = A.paged_decode_attention(q, k, v, tables, ctx, scale=p["scale"], window=64, return_lse=True)
    b, lb = A.paged_decode_attention(q, k, v, tables, ctx - 64, scale=p["scale"], return_lse=True)
    top = torch.logaddexp(la, lb)
    both = a.float() * (la - top).exp()[..., None] + b.float() * (lb - top).exp()[..., None]
    # two results rounded to bf16 instead of one
    assert bool(((both - whole.float()).abs() <= 2.0 ** -7 * (a.float().abs() + b.float().abs() + 1)).all())


def test_refusals_leave_the_device_healthy():
    p = PP.make(8, 2, 64, 16, [20])
    q, k, v, tables, ctx = p["args"]
    with pytest.raises(ValueError):
        A.paged_decode_attention(q, k, v, tables, ctx, sinks=2)
    with pytest.raises(ValueError):
        A.paged_decode_attention(q, k, v, tables, ctx, window=-1)
    with pytest.raises(ValueError):
        A.paged_decode_attention(q, k, v, tables, ctx, scale=float("nan"))
    with pytest.raises(ValueError):
        A.paged_decode_attention(q, k, v, tables.long(), ctx)
    with pytest.raises(ValueError):
        A.paged_decode_attention(q, k, v, tables, ctx.repeat(2))
    with pytest.raises(ValueError):
        A.paged_decode_attention(q, k[:, :, :, :32], v[:, :, :, :32], tables, ctx)
    with pytest.raises(ValueError):
        A.paged_decode_attention(q, k.half(), v.half(), tables, ctx)
    with pytest.raises(ValueError):
        A.paged_decode_attention(q[:, :7], k, v, tables, ctx)
    with pytest.raises(RuntimeError):
        A.paged_decode_attention(q.float(), k.float(), v.float(), tables, ctx)
    with pytest.raises(RuntimeError):
        A.paged_decode_attention(q.cpu(), k, v, tables, ctx)
    with pytest.raises(ValueError):
        A.paged_decode_attention(q, k, v, tables, ctx, out=torch.empty_like(q[:, :4]))
    assert N.device_status() == 0
    PP.check(p, _decode(p))
    assert A.paged_decode_attention(q[:0], k, v, tables[:0], ctx[:0]).shape == (0, 8, 64)


@pytest.mark.parametrize("dim", [64, 128])
@pytest.mark.parametrize("window,sinks", [(64, 4), (1, 40), (2 ** 31 - 21, 0), (2 ** 31 - 21, 9), (2 ** 31 - 1, 3)])
def test_positions_next_to_two_to_the_31(window, sinks, dim):
    """Contexts of 2^31 - 1 behind a short table: the first tokens alone, or a window whose begin lies inside the table for the last rows
    and ahead of it for the others."""
    last = 2 ** 31 - 1
    for page in (8, 16):
        p = PP.make(8, 2, dim, page, [64, 64], [150, 3], window=window, sinks=sinks, seed=dim + sinks)
        p["contexts"] = [last, last - 40]
        args = list(p["args"])
        args[4] = torch.tensor(p["contexts"], dtype=torch.int32, device="cuda")
        how = dict(scale=p["scale"], window=window, sinks=sinks, return_lse=True)
        out, lse = A.paged_prefill_attention(*args, **how)
        assert N.device_status() == 0
        PP.check(p, out, lse)
        p["q"], p["cu"] = p["q"][[149, 152]], None  # the last token of each
        out, lse = A.paged_decode_attention(args[0][[149, 152]], *args[1:5], **how)
        PP.check(p, out, lse)


@pytest.mark.parametrize("dim", [64, 128])
@pytest.mark.parametrize("window", [0, 100])
def test_tables_of_two_to_the_31_keys(window, dim):
    """The last pages of a table of 2^31 keys, the others missing: what the same pages give alone."""
    blocks, page, tail = 2 ** 23, 256, 3
    near = 2 ** 31 - 1 - (blocks - tail) * page
    p = PP.make(2, 1, dim, page, [near], [5], window=window, seed=dim)
    q, k, v, tables, _, cu = p["args"]
    wide = torch.full((1, blocks), -1, dtype=torch.int32, device="cuda")
    wide[:, blocks - tail:] = tables
    ctx = torch.tensor([2 ** 31 - 1], dtype=torch.int32, device="cuda")
    how = dict(scale=p["scale"], window=window, return_lse=True)
    if window:  # (without one every row walks the whole table)
        out, lse = A.paged_prefill_attention(q, k, v, wide, ctx, cu, **how)
        PP.check(p, out, lse)
    p["q"], p["cu"] = p["q"][4:], None
    out, lse = A.paged_decode_attention(q[4:], k, v, wide, ctx, **how)
    PP.check(p, out, lse)
    assert N.device_status() == 0


@pytest.mark.parametrize("prefill", [False, True])
@pytest.mark.parametrize("dim", [64, 128])
@pytest.mark.parametrize("spread", [0.0, 3.0])
def test_one_key_outweighs_a_long_context(spread, dim, prefill):
    """One key with 2^25 to 2^26 times the weight of any other of 60000, and a value of zero: the result is what the others add up to.
    Roundings in fp16: u of every probability (those from 2^-21 of the largest on are normal numbers) or, below that, 2^-32 of the largest;
    their sum is not rounded, the result once. The rest as in ``paged_problem.check``: scores are one product here (2^-24 of at most 20,
    twice), exponentials and running sums 2^-18 and keys 2^-23."""
    n = 60000
    p = PP.make(2, 1, dim, 64, [n], [2] if prefill else None, dtype=FP16, seed=3)
    flat = torch.tensor(p["tables"][0])
    k, v = torch.zeros_like(p["k"]), torch.rand(p["v"].shape, generator=torch.Generator().manual_seed(1)).add_(0.5).to(FP16)
    k[..., 1] = (torch.rand(k.shape[:3], generator=torch.Generator().manual_seed(2)) * -spread).to(FP16)
    k[flat[0], 0, 0, 0], k[flat[0], 0, 0, 1], v[flat[0], 0] = 8.0, 0.0, 0.0
    q = torch.zeros_like(p["q"])
    q[..., 0] = 17.5 / 8 / p["scale"]
    q[..., 1] = 0.25 / p["scale"]
    p.update(q=q, k=k, v=v)
    args = [q.cuda(), k.cuda(), v.cuda(), *p["args"][3:]]
    out, lse = (A.paged_prefill_attention if prefill else A.paged_decode_attention)(*args, scale=p["scale"], return_lse=True)
    want, want_lse, size, _ = PP.PO.paged_attention(q, k, v, p["tables"], p["contexts"], p["cu"], p["scale"], 0, 0)
    assert float(want.min()) > 5e-4
    u = 2.0 ** -11
    eps = 2 * 20 * 2.0 ** -24 + 2.0 ** -18 + n * 2.0 ** -23
    bound = u * want + (u * (1 + u) + eps) * size + n * 2.0 ** -32 * 1.5
    err = (out.double().cpu() - want).abs()
    assert bool((err <= bound).all()), f"worst {float((err / bound).max()):.3g} of the bound, {float((err / want).max()):.3g} of the result"
    assert bool(((lse.double().cpu() - want_lse).abs() <= 20 * 2.0 ** -24 + 2.0 ** -19 * 20 + n * 2.0 ** -24).all())
