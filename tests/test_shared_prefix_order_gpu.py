"""The two launches of attention behind a shared prefix: the same bits in strict stream order as with the second one beside the first, and
whatever lies in the workspace before the call."""

import pytest
import torch

import paged_problem as PP
import test_shared_prefix_gpu as SP
from nanovllm_voxcpm_b200 import _native as N

pytestmark = pytest.mark.gpu


@pytest.fixture(autouse=True)
def _restored():
    yield
    N.set_option(N.OPT_PDL, 1)
    assert N.device_status() == 0


# (requests: items by clusters of CTAs; by CTAs that take them from the counter, in order and, from 513 on, as they are)
CASES = [(2, False), (60, False), (513, False), (3, True), (40, True)]


def _problem(n, packed, dim):
    groups = [(300 + 7 * dim, [9 + 13 * i % 50 for i in range(n - n // 3)])] + ([(130, [9 + i % 40 for i in range(n // 3)])] if n >= 3 else [])
    return SP.make(16, 2, dim, 16, groups, [1 + i % 9 for i in range(n)] if packed else None, seed=n)


@pytest.mark.parametrize("dim", [64, 128])
@pytest.mark.parametrize("n,packed", CASES)
def test_strict_stream_order_gives_the_same(n, packed, dim):
    p = _problem(n, packed, dim)
    assert SP.way(p) == 1
    out, lse = SP.call(p, return_lse=True)
    N.set_option(N.OPT_PDL, 0)
    again, lse_again = SP.call(p, return_lse=True)
    assert torch.equal(out, again) and torch.equal(lse, lse_again)
    PP.check(p, again, lse_again, f"{n} requests")


@pytest.mark.parametrize("n,packed", CASES)
def test_whatever_lies_in_the_workspace(n, packed):
    """Counter, order and parts of an earlier life of the workspace are not read: words that say there are no items left, then others."""
    p = _problem(n, packed, 64)
    want = SP.call(p)
    q, k, tables, lens = p["args"][0], p["args"][1], p["args"][3], p["args"][4]
    need = N.lib().lora_b200_shared_prefix_workspace_bytes(q.size(0), lens.numel(), p["groups"][0].numel(), q.size(1), k.size(2), q.size(2),
                                                           tables.size(1), k.size(1), packed)
    out = torch.empty_like(want)
    for word in (2 ** 31 - 1, 0, -1, 1, 10 ** 6):
        for _ in range(20):
            torch.full((-(-need // 4),), word, dtype=torch.int32, device="cuda")  # (given back at once: the call's workspace is these bytes)
            SP.call(p, out=out)
            assert torch.equal(out, want), f"words of {word}"
