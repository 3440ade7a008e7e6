"""How a paged decode call meets the GPU (host code only): the rule takes the way that measured fastest where it says so, and the GPU
tests' cases for each way reach it."""

import pytest

from nanovllm_voxcpm_b200 import _native as N

SHARES, WARPS4, WARPS8, PAIRS, FOURS, EIGHTS = 0, 16 + 4, 16 + 8, 32 + 8, 64 + 8, 128 + 8


def way(T, heads, kv_heads, dim, keys, window=0, sinks=0, page=1):
    return N.lib().lora_b200_paged_decode_way(T, heads, kv_heads, dim, -(-keys // page), page, window, sinks)


# requests, heads, kv heads, head dim, longest context; us by ways, measured on a B200 (None: not measured)
MEASURED = [
    (1, 16, 2, 64, 700, (8.2, 7.1, 7.4, 6.6, 6.3, 10.9)),
    (1, 16, 2, 64, 8000, (48, 33, 22, 15, 10.9, 15.9)),
    (1, 16, 2, 64, 32000, (210, 125, 69, 39, 23.4, 21.4)),
    (64, 16, 2, 64, 1000, (11.9, 10.0, 16.5, 35, 66, 16.7)),
    (64, 16, 2, 64, 8000, (64, 48, 53, 84, 128, 52)),
    (8, 32, 8, 128, 300, (7.9, 7.4, 8.4, 12.5, 30, 13.1)),
    (8, 32, 8, 128, 2000, (30, 22, 18.9, 24, 42, 22)),
    (128, 16, 2, 128, 1000, (27.2, 29.2, 42, 97, 158, 34)),
    (48, 32, 8, 128, 8192, (203, 179, 166, 273, 368, 138)),
    (16, 32, 8, 128, 16000, (208, 138, 147, 146, 210, 109)),
]


@pytest.mark.parametrize("T,heads,kv_heads,dim,keys,us", MEASURED)
def test_chosen_way_is_the_one_that_measured_fastest(T, heads, kv_heads, dim, keys, us):
    took = us[(WARPS4, WARPS8, PAIRS, FOURS, EIGHTS, SHARES).index(way(T, heads, kv_heads, dim, keys))]
    assert took <= 1.02 * min(us)


@pytest.mark.parametrize("args", [(1, 16, 2, 64, 32000), (48, 32, 8, 128, 8192), (200, 40, 2, 64, 5000), (1, 1, 1, 128, 2 ** 31 - 256)])
def test_shares_come_with_a_workspace_and_the_others_without(args):
    T, heads, kv_heads, dim, keys = args
    need = lambda width: N.lib().lora_b200_paged_decode_workspace_bytes(T, heads, kv_heads, dim, width, 1, 0, 0)  # noqa: E731
    assert way(*args) == SHARES and need(keys) > 0
    assert way(T, heads, kv_heads, dim, 100) != SHARES and need(100) == 0
    assert way(*args, window=100) != SHARES


def test_refused_forms():
    assert way(1, 8, 0, 64, 100) < 0 and way(1, 2, 4, 64, 100) < 0
