"""Attention behind a shared prefix at the ends of what a length can be."""

import math

import pytest
import torch

import paged_problem as PP
import test_shared_prefix_gpu as SP
from nanovllm_voxcpm_b200 import _native as N

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("n", [4, 60])  # (items by clusters, and from the counter)
def test_contexts_of_less_than_no_key(n):
    """A context of -2^31 has no key either, in either launch; the others of the group are as they were."""
    p = SP.make(16, 2, 64, 16, [(700, [5 + i % 40 for i in range(n)])], seed=n)
    base, base_lse = SP.call(p, return_lse=True)
    args = list(p["args"])
    for least in (-2 ** 31, -2 ** 31 + 1, -1, 0):
        lens = args[4].clone()
        lens[1::3] = least
        p["args"] = (*args[:4], lens)
        assert SP.way(p) == 1
        out, lse = SP.call(p, return_lse=True)
        assert bool((out[1::3] == 0).all()) and bool((lse[1::3] == -math.inf).all()), f"{least}"
        kept = [i for i in range(n) if i % 3 != 1]
        p["contexts"] = lens.tolist()
        PP.check(p, out, lse, f"contexts of {least}")
        assert torch.equal(lse[kept] == -math.inf, base_lse[kept] == -math.inf)
    assert N.device_status() == 0


def test_packed_contexts_of_less_than_their_new_tokens():
    """New tokens ahead of position 0 have no key; a context of -2^31 none at all."""
    p = SP.make(16, 2, 64, 16, [(300, [20, 9, 30, 4])], [3, 2, 5, 4], seed=2)
    args = list(p["args"])
    lens = args[4].clone()
    lens[1], lens[2] = -2 ** 31, 3
    p["args"] = (*args[:4], lens, args[5])
    p["contexts"] = lens.tolist()
    assert SP.way(p) == 1
    out, lse = SP.call(p, return_lse=True)
    PP.check(p, out, lse)
    assert bool((out[3:7] == 0).all()) and bool((lse[3:7] == -math.inf).all())
    assert N.device_status() == 0
