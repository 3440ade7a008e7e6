"""What attention behind a shared prefix and differential attention cannot do without is named where it is missing."""

import pytest
import torch

from nanovllm_voxcpm_b200 import attention as A


def _args(packed):
    q, cache, ints = torch.zeros(2, 16, 64), torch.zeros(4, 16, 2, 64), torch.zeros(2, 1, dtype=torch.int32)
    lens = torch.ones(2, dtype=torch.int32)
    return q, cache, cache, ints, lens, *([torch.tensor([0, 1, 2], dtype=torch.int32)] if packed else [])


@pytest.mark.parametrize("packed", [False, True])
def test_groups_that_are_missing(packed):
    f = A.shared_prefix_prefill_attention if packed else A.shared_prefix_decode_attention
    lens, groups = torch.ones(1, dtype=torch.int32), torch.tensor([0, 2], dtype=torch.int32)
    for prefix, cu in ((None, groups), (lens, None), (None, None)):
        with pytest.raises(ValueError, match="prefix_lens and cu_groups"):
            f(*_args(packed), prefix, cu)


@pytest.mark.parametrize("packed", [False, True])
def test_lam_that_is_missing(packed):
    f = A.differential_prefill_attention if packed else A.differential_decode_attention
    with pytest.raises(ValueError, match="lam"):
        f(*_args(packed), None)
