"""Head norms with rotation and cache store against the 64-bit form.

Bounds: a result is rounded once, u = eps / 2 relative to it; the two products of the rotation and their sum are fp32, as are the
statistics (a sum of head_dim squares), so 2^-20 of the sizes of the two products covers them."""

import pytest
import torch

from nanovllm_voxcpm_b200 import _native as N
from nanovllm_voxcpm_b200 import glue as G
from oracle import paged_oracle as PO

pytestmark = pytest.mark.gpu
BF16, FP16 = torch.bfloat16, torch.float16


def _make(T, hq, hk, d, page, dtype, *, max_pos=600, half_table=True, table_dtype=torch.float32, seed=0, pad=0):
    gen = torch.Generator().manual_seed(seed)
    wide = (torch.randn(T, (hq + 2 * hk) * d + pad, generator=gen) * torch.exp(2 * torch.randn(T, 1, generator=gen))).to(dtype)
    qw, kw = ((1 + 0.3 * torch.randn(d, generator=gen)).to(dtype) for _ in range(2))
    angle = torch.randn(max_pos, d // 2 if half_table else d, generator=gen) * 3
    cos, sin = angle.cos().to(table_dtype), angle.sin().to(table_dtype)
    pos = torch.randint(0, max_pos, (T,), generator=gen)
    n_blocks = -(-T // page) + 2
    slots = torch.randperm(n_blocks * page, generator=gen)[:T].to(torch.int32)
    caches = [torch.randn(n_blocks, page, hk, d, generator=gen).to(dtype) for _ in range(2)]
    return wide, qw, kw, cos, sin, pos, slots, caches


def _near(got, want, size, dtype, what):
    got = got.double().cpu()
    bound = torch.finfo(dtype).eps / 2 * want.abs() + 2.0 ** -20 * size + (2.0 ** -25 if dtype == FP16 else 0)
    assert bool(((got - want).abs() <= bound).all()), f"{what}: worst {float(((got - want).abs() / bound).max()):.3g} of the bound"


@pytest.mark.parametrize("dtype", [BF16, FP16])
# (from 8 MB of rows on they come by bulk copies: the first seven; rows of more than a stage do not)
@pytest.mark.parametrize("T,hq,hk,d,page", [(701, 32, 8, 128, 16), (5001, 16, 2, 64, 64), (2300, 7, 7, 96, 24), (4800, 3, 1, 192, 16), (3700, 5, 3, 112, 8),
                                            (23011, 1, 1, 64, 256), (160, 90, 10, 256, 16), (1, 16, 2, 64, 256), (37, 16, 2, 128, 16), (300, 32, 8, 128, 16), (5, 3, 1, 80, 7), (9, 4, 4, 256, 3),
                                            (2, 1, 1, 16, 1), (65, 7, 7, 96, 24), (1000, 8, 2, 64, 64)])
@pytest.mark.parametrize("separate", [False, True])
def test_against_64_bits(T, hq, hk, d, page, dtype, separate):
    wide, qw, kw, cos, sin, pos, slots, (kc, vc) = _make(T, hq, hk, d, page, dtype, seed=T + d, pad=8, half_table=T % 2 == 1)
    slots[T // 2] = -1
    x = wide[:, 8:].view(T, hq + 2 * hk, d) if T else None
    q, q_size = PO.head_norm_rope(x[:, :hq], qw, 1e-6, pos, cos, sin)
    k, k_size = PO.head_norm_rope(x[:, hq:hq + hk], kw, 1e-6, pos, cos, sin)
    dev = wide.cuda()
    kd, vd = kc.cuda(), vc.cuda()
    out = torch.full((T, hq + 1, d), 7.0, dtype=dtype, device="cuda")[:, :hq] if separate else None
    got_q, got_k, got_v = G.qk_norm_rope_kv_store(dev[:, 8:], hq, hk, d, qw.cuda(), kw.cuda(), 1e-6, positions=pos.cuda(), cos=cos.cuda(),
                                                  sin=sin.cuda(), k_cache=kd, v_cache=vd, slot_mapping=slots.cuda(), q_out=out)
    _near(got_q, q, q_size, dtype, "q")
    if separate:
        assert got_k is None and torch.equal(dev.cpu(), wide) and got_q.data_ptr() == out.data_ptr()
    else:
        _near(got_k, k, k_size, dtype, "k")
        assert got_q.data_ptr() == dev[:, 8:].data_ptr() and torch.equal(dev[:, :8].cpu(), wide[:, :8])
    assert torch.equal(got_v.cpu(), x[:, hq + hk:])
    kept = slots >= 0
    at = slots[kept].long()
    _near(kd.view(-1, hk, d)[at.cuda()], k[kept], k_size[kept], dtype, "k cache")
    assert torch.equal(vd.view(-1, hk, d)[at.cuda()].cpu(), x[kept, hq + hk:])
    others = torch.ones(kc.size(0) * page, dtype=torch.bool)
    others[at] = False
    assert torch.equal(kd.cpu().view(-1, hk, d)[others], kc.view(-1, hk, d)[others])
    assert torch.equal(vd.cpu().view(-1, hk, d)[others], vc.view(-1, hk, d)[others])


@pytest.mark.parametrize("table_dtype", [BF16, FP16, torch.float32])
@pytest.mark.parametrize("rotate,store", [(True, False), (False, True), (False, False)])
def test_forms(rotate, store, table_dtype):
    """Without rotation, without a cache; tables of each type; positions outside the table count as its ends."""
    T, hq, hk, d = 21, 8, 2, 64
    wide, qw, kw, cos, sin, pos, slots, (kc, vc) = _make(T, hq, hk, d, 8, BF16, table_dtype=table_dtype)
    pos[0], pos[1] = -5, 10 ** 12
    x = wide.view(T, -1, d)
    turn = (pos, cos, sin) if rotate else ()
    q, q_size = PO.head_norm_rope(x[:, :hq], qw, 1e-5, *turn)
    k, k_size = PO.head_norm_rope(x[:, hq:hq + hk], kw, 1e-5, *turn)
    kw_args = dict(zip(("positions", "cos", "sin"), (t.cuda() for t in (pos, cos, sin)))) if rotate else {}
    kd, vd = kc.cuda(), vc.cuda()
    if store:
        kw_args.update(k_cache=kd, v_cache=vd, slot_mapping=slots.cuda())
    got_q, got_k, _ = G.qk_norm_rope_kv_store(wide.cuda(), hq, hk, d, qw.cuda(), kw.cuda(), 1e-5, **kw_args)
    _near(got_q, q, q_size, BF16, "q")
    _near(got_k, k, k_size, BF16, "k")
    if store:
        _near(kd.view(-1, hk, d)[slots.long().cuda()], k, k_size, BF16, "cache")
    else:
        assert torch.equal(kd.cpu(), kc)


def test_strided_caches_and_slots_outside():
    """k and v of a block in one tensor, heads ahead of positions; slots at and behind the cache's end are skipped."""
    T, hq, hk, d, page = 40, 8, 2, 128, 16
    wide, qw, kw, cos, sin, pos, slots, _ = _make(T, hq, hk, d, page, FP16, seed=3)
    both = torch.full((5, 2, hk, page, d), 7.0, dtype=FP16, device="cuda")
    kd, vd = both[:, 0].transpose(1, 2), both[:, 1].transpose(1, 2)
    slots = slots.clone()
    slots[3], slots[4], slots[5] = 5 * page, 2 ** 31 - 1, -2 ** 31
    G.qk_norm_rope_kv_store(wide.cuda(), hq, hk, d, qw.cuda(), kw.cuda(), 1e-6, positions=pos.cuda(), cos=cos.cuda(), sin=sin.cuda(),
                            k_cache=kd, v_cache=vd, slot_mapping=slots.cuda())
    x = wide.view(T, -1, d)
    k, k_size = PO.head_norm_rope(x[:, hq:hq + hk], kw, 1e-6, pos, cos, sin)
    written = torch.zeros(5 * page, dtype=torch.bool)
    for t in range(T):
        if 0 <= slots[t] < 5 * page:
            b, o = int(slots[t]) // page, int(slots[t]) % page
            _near(kd[b, o], k[t], k_size[t], FP16, "k")
            assert torch.equal(vd[b, o].cpu(), x[t, hq + hk:])
            written[int(slots[t])] = True
    assert bool((kd.cpu().reshape(-1, hk, d)[~written] == 7).all()) and bool((vd.cpu().reshape(-1, hk, d)[~written] == 7).all())


def test_rows_of_zeros_and_of_infinities():
    wide = torch.zeros(3, 6 * 64, dtype=BF16, device="cuda")
    wide[1, 5] = float("inf")
    wide[2] = 3.0e38
    one = torch.ones(64, dtype=BF16, device="cuda")
    q, k, v = G.qk_norm_rope_kv_store(wide.clone(), 4, 1, 64, one, one, 1e-6)
    assert bool((q[0] == 0).all()) and bool((k[0] == 0).all())
    assert bool(q[1, 0, 5].isnan()) and bool((q[1, 1:] == 0).all())
    assert bool((q[2] == 0).all())  # the sum of squares is infinite, as in any fp32 norm


@pytest.mark.parametrize("T", [3, 24000])  # (a thread a piece; rows by bulk copies)
@pytest.mark.parametrize("rotate", [False, True])
def test_heads_of_an_infinite_sum_of_squares(rotate, T):
    """Their factor is 0 (the sum is fp32), and 0 times an element, its weight and its angle is 0 for finite elements whatever the order
    of the products gives on the way; only the infinite element is NaN, with a rotation its opposite column too."""
    hq, hk, d = 2, 1, 64
    wide = torch.zeros(T, hq + 2 * hk, d, dtype=BF16)
    wide[0, 0, 5] = float("inf")
    wide[0, 0, 6:] = 3.0
    wide[0, 2, 40] = -float("inf")
    wide[1] = 3.0e38
    wide[2, :, ::2], wide[2, :, 1::2] = -3.0e38, 2.0e38
    wide[-1, 1, 3] = float("inf")
    weight = torch.linspace(1.5, 40.0, d).to(BF16)
    angle = torch.linspace(0.1, 3.0, d // 2).expand(8, -1)
    turn = dict(positions=(torch.arange(T) % 8).cuda(), cos=angle.cos().contiguous().cuda(), sin=angle.sin().contiguous().cuda()) if rotate else {}
    q, k, v = G.qk_norm_rope_kv_store(wide.cuda().view(T, -1), hq, hk, d, weight.cuda(), weight.cuda(), 1e-6, **turn)
    for got, head, at in ((q, 0, (0, 5)), (k, 2, (0, 40)), (q, 1, (T - 1, 3))):
        row = got[at[0], head if got is q else 0].cpu()
        nan = torch.zeros(d, dtype=torch.bool)
        nan[at[1]] = True
        if rotate:
            nan[(at[1] + d // 2) % d] = True
        assert torch.equal(row.isnan(), nan) and bool((row[~nan] == 0).all()), (head, row)
    assert bool((q[1] == 0).all()) and bool((k[1] == 0).all())
    if T > 3:
        assert bool((q[2] == 0).all()) and bool((k[2] == 0).all())
    else:
        assert bool((q[2, 0] == 0).all()) and bool((k[2] == 0).all())
    assert torch.equal(v.cpu(), wide[:, hq + hk:])


def test_graph_and_empty_batch():
    T, hq, hk, d = 12, 16, 2, 64
    wide, qw, kw, cos, sin, pos, slots, (kc, vc) = (t.cuda() if torch.is_tensor(t) else [c.cuda() for c in t] for t in _make(T, hq, hk, d, 16, BF16))
    out = torch.empty(T, hq, d, dtype=BF16, device="cuda")
    call = lambda w, p, s, o: G.qk_norm_rope_kv_store(w, hq, hk, d, qw, kw, 1e-6, positions=p, cos=cos, sin=sin, k_cache=kc, v_cache=vc,  # noqa: E731
                                                      slot_mapping=s, q_out=o)
    call(wide, pos, slots, out)
    want, want_k = out.clone(), kc.clone()
    stream = torch.cuda.Stream()
    stream.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(stream):
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g, stream=stream):
            call(wide, pos, slots, out)
        out.zero_()
        kc.zero_()
        g.replay()
    stream.synchronize()
    assert torch.equal(out, want) and torch.equal(kc.view(-1, hk, d)[slots.long()], want_k.view(-1, hk, d)[slots.long()])
    call(wide[:0], pos[:0], slots[:0], out[:0])
    assert N.device_status() == 0
