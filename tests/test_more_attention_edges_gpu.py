"""Sizes and layouts at the ends of what attention behind shared prefixes, differential attention and the join take: none and one of a
thing, tables and parts by a stride of zero, caches and rows whose offsets pass 32 bits, calls side by side."""

import math

import pytest
import torch

import paged_problem as PP
import test_differential_gpu as TD
import test_shared_prefix_gpu as SP
from nanovllm_voxcpm_b200 import _native as N
from nanovllm_voxcpm_b200 import attention as A
from oracle import more_attention_oracle as MO

pytestmark = pytest.mark.gpu
BF16 = torch.bfloat16


@pytest.fixture(autouse=True)
def _clean():
    yield
    torch.cuda.synchronize()
    assert N.device_status() == 0


def _ints(*values):
    return torch.tensor(values, dtype=torch.int32, device="cuda")


def _differential(packed):
    return TD.make(16, 2, 64, 16, [300, 40, 77], [30, 1, 40] if packed else None, seed=3, per_token=True)


def _shared(packed):
    return SP.make(16, 2, 64, 16, [(500, [9, 40, 30]), (130, [20])], [9, 4, 30, 1] if packed else None, seed=8)


@pytest.mark.parametrize("packed", [False, True])
def test_no_rows_and_no_requests(packed):
    cache, none, start = torch.zeros(4, 16, 2, 64, device="cuda", dtype=BF16), _ints(), _ints(0)
    tables, weight = torch.zeros(0, 7, dtype=torch.int32, device="cuda"), torch.ones(64, device="cuda", dtype=BF16)
    for T in (0, 3) if packed else (0,):  # (rows of no sequence stay as they are)
        q = torch.zeros(T, 16, 64, device="cuda", dtype=BF16)
        base = (q, cache, cache, tables, none, *([start] if packed else []))
        out = torch.full_like(q, 7.0)
        f = A.differential_prefill_attention if packed else A.differential_decode_attention
        assert f(*base, torch.zeros(16, device="cuda"), norm_weight=weight, out=out) is out
        f = A.shared_prefix_prefill_attention if packed else A.shared_prefix_decode_attention
        assert f(*base, none, start, out=out) is out
        _, lse = f(*base, _ints(5), _ints(0, 0), out=out, return_lse=True)
        assert lse.shape == (T, 16) and bool((out == 7).all())
    # requests without a new token
    if packed:
        q = torch.zeros(0, 16, 64, device="cuda", dtype=BF16)
        base = (q, cache, cache, torch.zeros(3, 7, dtype=torch.int32, device="cuda"), _ints(5, 0, 9), _ints(0, 0, 0, 0))
        assert A.shared_prefix_prefill_attention(*base, _ints(16), _ints(0, 3)).shape == (0, 16, 64)
        assert A.differential_prefill_attention(*base, torch.zeros(16, device="cuda")).shape == (0, 16, 64)


@pytest.mark.parametrize("packed", [False, True])
def test_tables_of_no_blocks(packed):
    """Tables without a column: nobody has a key, and zeros are what is left."""
    q, cache = torch.randn(3, 16, 64, device="cuda").to(BF16), torch.zeros(4, 16, 2, 64, device="cuda", dtype=BF16)
    base = (q, cache, cache, torch.zeros(3, 0, dtype=torch.int32, device="cuda"), _ints(5, 0, 9), *([_ints(0, 1, 2, 3)] if packed else []))
    f = A.differential_prefill_attention if packed else A.differential_decode_attention
    assert bool((f(*base, torch.full((16,), 0.3, device="cuda")) == 0).all())
    f = A.shared_prefix_prefill_attention if packed else A.shared_prefix_decode_attention
    out, lse = f(*base, _ints(16), _ints(0, 3), return_lse=True)
    assert bool((out == 0).all()) and bool((lse == -math.inf).all())


@pytest.mark.parametrize("packed", [False, True])
def test_one_table_for_all_by_a_stride_of_zero(packed):
    """Requests that are the same but for their queries: the same table for each, not copied."""
    n, context = 24, 700
    for kind in ("differential", "shared"):
        new = [1 + i % 5 for i in range(n)] if packed else None
        p = (TD if kind == "differential" else PP).make(16, 2, 64, 16, [context] * n, new, seed=4)
        p["tables"] = [p["tables"][0]] * n
        args = list(p["args"])
        one = args[3][:1]
        if kind == "shared":
            p["groups"] = (_ints(640), _ints(0, n))  # (whole blocks; the rest of each context is the same, too)
            args[3] = torch.nn.functional.pad(one, (0, 4000 - one.size(1)), value=-1)
        else:
            args[3] = one
        args[3] = args[3].expand(n, -1)
        assert args[3].stride(0) == 0
        p["args"] = tuple(args)
        if kind == "shared":
            assert SP.way(p) == 1
            PP.check(p, *SP.call(p, return_lse=True))
        else:
            TD.check(p, TD.call(p))


@pytest.mark.parametrize("packed", [False, True])
@pytest.mark.parametrize("kind", ["differential", "shared"])
def test_blocks_whose_offsets_pass_32_bits(kind, packed):
    """The blocks of a small problem at the end of a cache of more than 2^31 elements: the same bits."""
    p = (_differential if kind == "differential" else _shared)(packed)
    call = (TD if kind == "differential" else SP).call
    want = call(p)
    q, k, v, tables, *rest = p["args"]
    blocks = 2 ** 31 // k[0].numel() + 2 * k.size(0)
    caches = []
    for c in (k, v):
        big = torch.empty(blocks, *c.shape[1:], dtype=c.dtype, device="cuda")
        big[-c.size(0):] = c
        caches.append(big)
    moved = torch.where(tables >= 0, tables + (blocks - k.size(0)), tables)
    p["args"] = (q, *caches, moved, *rest)
    if kind == "shared":
        assert SP.way(p) == 1
    assert torch.equal(call(p), want)


@pytest.mark.parametrize("packed", [False, True])
@pytest.mark.parametrize("kind", ["differential", "shared"])
def test_rows_whose_offsets_pass_32_bits(kind, packed):
    """q and out as rows so far apart that the last one begins behind 2^31 elements."""
    p = (_differential if kind == "differential" else _shared)(packed)
    call = (TD if kind == "differential" else SP).call
    want = call(p)
    q = p["args"][0]
    T, far = q.size(0), 2 ** 31 // (q.size(0) - 1) // 8 * 8 + 1024 * 8
    wide = [torch.empty((T - 1) * far + 1024, dtype=BF16, device="cuda").as_strided((T, 16, 64), (far, 64, 1)) for _ in range(2)]
    wide[0].copy_(q)
    p["args"] = (wide[0], *p["args"][1:])
    call(p, out=wide[1])
    assert torch.equal(wide[1], want)


def test_a_long_prefix_in_all_its_parts():
    """150000 keys that three requests share, cut into as many parts as there are at most."""
    p = SP.make(2, 1, 64, 256, [(150000, [3, 700, 40])], seed=2)
    out, lse = SP.call(p, return_lse=True)
    PP.check(p, out, lse)


def test_calls_side_by_side():
    """Calls of either kind on two streams at once, each with a workspace of its own."""
    problems = [(_differential(True), TD.call), (_shared(False), SP.call), (_differential(False), TD.call), (_shared(True), SP.call)]
    wants = [f(p) for p, f in problems]
    streams = [torch.cuda.Stream() for _ in range(2)]
    torch.cuda.synchronize()
    outs = []
    for i in range(24):
        with torch.cuda.stream(streams[i % 2]):
            p, f = problems[(i // 2 + i) % 4]
            outs.append(((i // 2 + i) % 4, f(p)))
    torch.cuda.synchronize()
    assert all(torch.equal(o, wants[i]) for i, o in outs)


def test_a_join_of_more_rows_than_32_bit_indexes_take():
    """2^30 pieces of 16 bytes, parts by strides of zero: few rows again and again, so that every one of them is known."""
    rows, heads, dim = 2 ** 21 + 3, 32, 128
    gen = torch.Generator().manual_seed(1)
    outs, lses = torch.randn(2, 1, heads, dim, generator=gen).to(BF16), torch.randn(2, 1, heads, generator=gen)
    lses[0, 0, 5] = -math.inf
    parts, logs = [o.cuda().expand(rows, -1, -1) for o in outs], [x.cuda().expand(rows, -1) for x in lses]
    out, lse = A.join_attention(parts, logs, return_lse=True)
    few = A.join_attention([o[:1].contiguous() for o in parts], [x[:1].contiguous() for x in logs], return_lse=True)
    want, _, size = MO.join(outs, lses)
    assert bool(((few[0].double().cpu() - want).abs() <= 2.0 ** -8 * want.abs() + 2.0 ** -14 * size).all())
    for at in range(0, rows, 2 ** 18):
        assert bool((out[at:at + 2 ** 18] == few[0]).all()) and bool((lse[at:at + 2 ** 18] == few[1]).all())
