"""Join of attention results over parts of a context against the 64-bit form."""

import math

import pytest
import torch

import paged_problem as PP
from nanovllm_voxcpm_b200 import attention as A
from oracle import more_attention_oracle as MO

pytestmark = pytest.mark.gpu


def parts_of(n, T, heads, dim, dtype, seed=0, none=0.2):
    gen = torch.Generator().manual_seed(seed)
    outs = torch.randn(n, T, heads, dim, generator=gen).to(dtype)
    lses = torch.randn(n, T, heads, generator=gen) * 3 + 5
    lses[torch.rand(n, T, heads, generator=gen) < none] = -math.inf
    return outs, lses


def check(outs, lses, out, lse):
    """A weight is exp of a difference of two fp32 numbers, of which the largest is one of them: off by 2^-24 of the difference and 2^-21
    relative for the exponential of up to 88 in units of log2 (88 * 1.45 * 2^-24, and 2 ulp); sums of n terms in fp32; one rounding."""
    want, want_lse, size = MO.join(outs, lses)
    n = outs.size(0)
    eps = 2 * (2.0 ** -16 + (n + 6) * 2.0 ** -24)
    u = torch.finfo(outs.dtype).eps / 2
    bound = u * want.abs() + (1 + u) * eps * size + (2.0 ** -25 if outs.dtype == torch.float16 else 0)
    got = out.double().cpu()
    assert not got.isnan().any()
    assert bool(((got - want).abs() <= bound + 1e-30).all())
    if lse is not None:
        lse = lse.double().cpu()
        empty = want_lse == -math.inf
        assert torch.equal(lse == -math.inf, empty) and bool((got[empty] == 0).all())
        assert bool(((lse - want_lse).abs() <= eps + 2.0 ** -22 * (1 + want_lse.abs()))[~empty].all())


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16, torch.float32])
@pytest.mark.parametrize("n", [1, 2, 3, 4, 5, 8, 9, 64])
@pytest.mark.parametrize("T,heads,dim", [(1, 1, 8), (3, 5, 64), (17, 16, 128), (2, 3, 72), (40, 7, 256)])
def test_parts(n, T, heads, dim, dtype):
    outs, lses = parts_of(n, T, heads, dim, dtype, seed=n)
    out, lse = A.join_attention(outs.cuda(), lses.cuda(), return_lse=True)
    check(outs, lses, out, lse)
    assert torch.equal(out, A.join_attention(list(outs.cuda()), list(lses.cuda())))


def test_values_of_parts_without_keys_do_not_count():
    outs, lses = parts_of(4, 6, 4, 64, torch.bfloat16, none=0.5)
    clean = A.join_attention(outs.cuda(), lses.cuda())
    outs[(lses == -math.inf)] = math.nan
    got, lse = A.join_attention(outs.cuda(), lses.cuda(), return_lse=True)
    assert torch.equal(got, clean)
    outs[2, 1, 1], lses[2, 1, 1] = 1.0, math.nan
    got, lse = A.join_attention(outs.cuda(), lses.cuda(), return_lse=True)
    assert bool(got[1, 1].isnan().all()) and bool(lse[1, 1].isnan()) and int(got.isnan().sum()) == 64


def test_far_apart():
    """Logarithms next to the ends of fp32 and far from one another: no overflow, the larger part alone."""
    outs, lses = parts_of(3, 2, 2, 64, torch.float32, none=0)
    lses[0], lses[1], lses[2] = 3e38, -3e38, 0
    out, lse = A.join_attention(outs.cuda(), lses.cuda(), return_lse=True)
    assert torch.equal(out.cpu(), outs[0]) and bool((lse == 3e38).all())


def test_strides_and_in_place():
    outs, lses = parts_of(2, 9, 6, 64, torch.bfloat16)
    wide = [torch.zeros(9, 8, 80, dtype=torch.bfloat16, device="cuda") for _ in range(2)]
    logs = [torch.zeros(6, 9, device="cuda") for _ in range(2)]
    for i in range(2):
        wide[i][:, 1:7, 8:72] = outs[i].cuda()
        logs[i].copy_(lses[i].t())
    views = [w[:, 1:7, 8:72] for w in wide]
    out, lse = A.join_attention(views, [x.t() for x in logs], return_lse=True)
    check(outs, lses, out, lse)
    assert A.join_attention(views, [x.t() for x in logs], out=views[1]) is views[1]
    assert torch.equal(views[1], out) and bool((wide[1][:, 0] == 0).all()) and bool((wide[1][:, :, :8] == 0).all())


def test_empty_and_graph():
    assert A.join_attention(torch.zeros(2, 0, 4, 64, device="cuda"), torch.zeros(2, 0, 4, device="cuda")).shape == (0, 4, 64)
    outs, lses = parts_of(3, 50, 16, 64, torch.bfloat16)
    o, x = outs.cuda(), lses.cuda()
    want = A.join_attention(o, x)
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        got = A.join_attention(o, x)
    o[0] += 1
    g.replay()
    assert not torch.equal(got, want) and torch.equal(got, A.join_attention(o, x))


@pytest.mark.parametrize("cut", [1, 100, 257, 1023])
def test_a_context_in_two_pieces(cut):
    """What the logarithms are for: a context attended as two, joined, against the whole of it."""
    p = PP.make(16, 2, 64, 1, [1024], seed=cut)
    q, k, v, tables, _ = p["args"]
    lens = [torch.tensor([n], dtype=torch.int32, device="cuda") for n in (cut, 1024 - cut)]
    first = A.paged_decode_attention(q, k, v, tables, lens[0], return_lse=True)
    second = A.paged_decode_attention(q, k, v, tables[:, cut:].contiguous(), lens[1], return_lse=True)
    out, lse = A.join_attention((first[0], second[0]), (first[1], second[1]), return_lse=True)
    whole, whole_lse = A.paged_decode_attention(*p["args"], return_lse=True)
    # (each piece and the join round once more: three roundings of at most the sum of |p v|, which is at most max |v|)
    u = torch.finfo(torch.bfloat16).eps / 2
    assert float((out.float() - whole.float()).abs().max()) <= 5 * u * float(v.float().abs().max())
    assert float((lse - whole_lse).abs().max()) <= 1e-4
