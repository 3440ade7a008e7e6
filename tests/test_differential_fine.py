"""The bits of differential attention's probabilities: maps that nearly cancel, held to a bound that a kernel passes only if every
probability enters the product with v as two 16-bit numbers. The bound is shown to refuse the same result with one number a
probability, or with two for the first 64 keys of each 128 alone (host code, the mistake planted in the 64-bit form)."""

import pytest
import torch

import paged_problem as PP
from nanovllm_voxcpm_b200 import attention as A
from oracle import more_attention_oracle as MO

BF16, FP16 = torch.bfloat16, torch.float16


def make(heads, kv_heads, dim, contexts, new=None, *, dtype=BF16, seed=0, page=16, device="cuda"):
    """The second map's columns are the first's but for a fiftieth of their spread, lam next to 1, scores of spread 1 to 2."""
    p = PP.make(heads, kv_heads, dim, page, contexts, new, seed=seed, dtype=dtype, device="cpu")
    gen, half = torch.Generator().manual_seed(seed + 5), dim // 2
    for name, spread in (("q", 0.7), ("k", 1.0)):
        x = torch.randn(p[name].shape, generator=gen) * spread
        x[..., half:] = x[..., :half] + 0.02 * spread * torch.randn(*x.shape[:-1], half, generator=gen)
        p[name] = x.to(dtype)
    p["lam"] = 1 - 0.02 * torch.rand(heads, generator=gen)
    p["scale"] = half ** -0.5
    if device != "cpu":
        p["args"] = tuple(x.to(device) for x in (p["q"], p["k"], p["v"], *p["args"][3:]))
    return p


def check(p, out, what=""):
    """What a map's result is off by before its rounding, relative to sum p |v| ("size"):
    a probability as two numbers, in bf16 both truncated (the first leaves less than 2^-7 of its power of two, of which the second keeps
    8 bits: 2^-15), in fp16 both rounded (2^-11, then 2^-12 of that: 2^-23; and what lies below 2^-24 is lost, 2^-25 of a largest
    probability that is 2^7 or more, since that is where the reference of the exponentials is laid down: 2^-32 of it a key);
    scores, sums of dim / 2 products in fp32: dim / 2 * 2^-24 sum |q k| scale, twice with the denominator; the exponentials and the
    running sums as ``paged_problem.check``: 2^-18 and keys 2^-23. The difference is off by the sum of both, the second times lam, and
    2^-22 of both for its own products, then rounded once."""
    q, dim = p["q"], p["q"].size(-1)
    half, u = dim // 2, torch.finfo(q.dtype).eps / 2
    one, two, count = MO.two_maps(q, p["k"], p["v"], p["tables"], p["contexts"], p["cu"], p["scale"], 0, 0)
    lam = p["lam"].double()[None, :, None]
    top = float(p["v"].float().abs().max())
    spread = torch.stack([(q[..., m * half:(m + 1) * half].double().norm(dim=-1) * p["k"][..., m * half:(m + 1) * half].double().norm(dim=-1).max())
                          for m in range(2)])  # (Cauchy: sum |q k| of a row and any key)
    err = 0
    for m, (_, size) in enumerate((one, two)):
        eps = 2 * half * 2.0 ** -24 * p["scale"] * spread[m][..., None] + 2.0 ** -18 + count.double()[:, None, None] * 2.0 ** -23
        mine = (eps + (2.0 ** -15 if q.dtype == BF16 else 2.0 ** -23)) * size
        mine = mine + (count[:, None, None] * 2.0 ** -32 * top if q.dtype == FP16 else 0)
        err = err + (mine if m == 0 else lam * mine)
    err = err + 2.0 ** -22 * (one[1] + lam * two[1])
    want = one[0] - lam * two[0]
    bound = u * want.abs() + (1 + u) * err + (2.0 ** -25 if q.dtype == FP16 else 0)
    off = (out.double().cpu() - want).abs() / bound
    assert not off.isnan().any() and float(off.max()) <= 1, f"{what}: worst {float(off.max()):.3g} of the bound"


def rounded(p, kept):
    """The 64-bit form with each probability rounded to one 16-bit number ahead of its product with v, but for the ``kept`` keys."""
    q, k, v = p["q"].double(), p["k"].double(), p["v"].double()
    dim, page = q.size(-1), k.size(1)
    half, group = dim // 2, q.size(1) // k.size(2)
    out = torch.zeros_like(q)
    cu = p["cu"] or list(range(len(p["contexts"]) + 1))
    for r, ctx in enumerate(p["contexts"]):
        for row in range(cu[r], cu[r + 1]):
            n = ctx - (cu[r + 1] - 1 - row)
            place = [(p["tables"][r][j // page], j % page) for j in range(n)]
            b, o = (torch.tensor([x[i] for x in place]) for i in range(2))
            for m, sign in ((0, 1.0), (1, -p["lam"].double())):
                cols = slice(m * half, (m + 1) * half)
                s = torch.einsum("hd,jhd->hj", q[row][:, cols], k[b, o][..., cols].repeat_interleave(group, 1)) * p["scale"]
                e = torch.exp(s - s.amax(-1, keepdim=True))
                coarse = torch.where(kept(torch.arange(n)), e, e.to(p["q"].dtype).double())
                got = torch.einsum("hj,jhd->hd", coarse, v[b, o].repeat_interleave(group, 1)) / e.sum(-1, keepdim=True)
                out[row] += got * (sign if m == 0 else sign[:, None])
    return out.to(p["q"].dtype)


CONTEXTS = {BF16: [2, 5, 17, 70, 100, 128, 300], FP16: [2, 3, 5, 9, 17, 30]}


@pytest.mark.parametrize("dtype", [BF16, FP16])
@pytest.mark.parametrize("dim", [64, 128])
def test_the_bound_refuses_one_number(dim, dtype):
    p = make(4, 2, dim, CONTEXTS[dtype], dtype=dtype, seed=dim, device="cpu")
    check(p, rounded(p, lambda j: j >= 0), "both numbers")
    with pytest.raises(AssertionError, match="of the bound"):
        check(p, rounded(p, lambda j: j < 0), "one number")


@pytest.mark.parametrize("contexts", [[70, 100, 128], [200, 300]])
def test_the_bound_refuses_two_numbers_for_half_of_the_keys(contexts):
    p = make(4, 2, 128, contexts, [3] * len(contexts), seed=1, device="cpu")
    with pytest.raises(AssertionError, match="of the bound"):
        check(p, rounded(p, lambda j: j % 128 < 64), "half of the keys")


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [BF16, FP16])
@pytest.mark.parametrize("heads", [(4, 2, 64), (4, 2, 128), (16, 2, 64), (16, 2, 128), (32, 8, 128), (3, 1, 128)])
def test_decode(heads, dtype):
    for contexts in (CONTEXTS[dtype], [900, 2000], [64] * 100):  # (items by one CTA or a cluster)
        p = make(*heads, contexts, dtype=dtype, seed=sum(heads))
        check(p, A.differential_decode_attention(*p["args"], p["lam"].cuda()), f"{heads} {contexts[:4]}")


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [BF16, FP16])
@pytest.mark.parametrize("heads", [(4, 2, 64), (4, 2, 128), (16, 2, 64), (16, 2, 128), (32, 8, 128), (3, 1, 128)])
@pytest.mark.parametrize("page", [16, 12])
def test_prefill(heads, dtype, page):
    """Whole items and, behind longer contexts, items that are cut and joined; blocks that the tile kernel does not take."""
    for new, contexts in (([1, 3, 17, 70], [1, 3, 17, 100]), ([5], [300]), ([16], [1500])):
        p = make(*heads, contexts, new, dtype=dtype, seed=sum(heads), page=page)
        check(p, A.differential_prefill_attention(*p["args"], p["lam"].cuda()), f"{heads} {new}")


@pytest.mark.gpu
@pytest.mark.parametrize("dim", [64, 128])
def test_a_token_is_as_exact_wherever_its_keys_lie(dim):
    """The same token by prefill and by decode, its weight on one key that moves through a tile: either within the bound."""
    for at in (0, 40, 63, 64, 65, 100, 126):
        p = make(4, 2, dim, [128], [1], seed=at)
        row = p["tables"][0][at // 16], at % 16
        for m in range(2):
            cols = slice(m * dim // 2, (m + 1) * dim // 2)
            p["k"][row][:, cols] = p["q"][0, ::2, cols] * (1.5 if m == 0 else 1.48)
        args = (p["q"].cuda(), p["k"].cuda(), p["v"].cuda(), *p["args"][3:])
        check(p, A.differential_prefill_attention(*args, p["lam"].cuda()), f"prefill, key {at}")
        check(p, A.differential_decode_attention(*args[:5], p["lam"].cuda()), f"decode, key {at}")


def test_two_numbers_keep_what_the_bound_says():
    """The split itself over a dense range: bf16 by truncation 2^-15, by rounding 2^-17; fp16 by rounding 2^-23 and, below its normal
    numbers, half of the smallest step."""
    x = torch.exp2(torch.linspace(-12, 0, 200001, dtype=torch.float64)).float()
    cut = lambda t: (t.view(torch.int32) & -65536).view(torch.float32)  # noqa: E731
    for least, y, split in ((2.0 ** -15, x, cut), (2.0 ** -17, x, lambda t: t.to(BF16).float()), (2.0 ** -23, 128 * x, lambda t: t.to(FP16).float())):
        hi = split(y)
        left = (hi.double() + split(y - hi).double() - y.double()).abs()
        assert bool((left <= least * y.double() + (2.0 ** -25 if least == 2.0 ** -23 else 0)).all())
