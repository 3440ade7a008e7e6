"""Parts of a join whose dimensions of one entry have strides of their own, which mean nothing: single tokens and single heads out of
buffers of different layouts, by the compiled path and by the one behind it."""

import pytest
import torch

from nanovllm_voxcpm_b200 import _native as N
from nanovllm_voxcpm_b200 import attention as A
from test_join_attention_gpu import check, parts_of

pytestmark = pytest.mark.gpu


class _NotHandled:
    @staticmethod
    def join_attention(*_):
        return None


@pytest.mark.parametrize("compiled", [True, False])
@pytest.mark.parametrize("T,heads", [(1, 6), (5, 1), (1, 1)])
def test_strides_of_single_entries(T, heads, compiled, monkeypatch):
    outs, lses = parts_of(3, T, heads, 64, torch.bfloat16, seed=T + heads, none=0)
    o, x = outs.cuda(), lses.cuda()
    # strides that a part of several tokens or heads could not have: of the single entries alone
    strides, log_strides = (67 if T == 1 else heads * 64, 69 if heads == 1 else 64, 1), (99 if T == 1 else heads, 77 if heads == 1 else 1)
    like = lambda t, how: torch.zeros_like(t).flatten().as_strided(t.shape, how).copy_(t)  # noqa: E731
    parts, its = [o[0], like(o[1], strides), o[2]], [x[0], x[1], like(x[2], log_strides)]
    if not compiled:
        monkeypatch.setattr(N, "native", lambda: _NotHandled)
    target = like(torch.zeros_like(o[0]), strides)
    out, lse = A.join_attention(parts, its, out=target, return_lse=True)
    assert out is target
    check(outs, lses, out, lse)


@pytest.mark.parametrize("compiled", [True, False])
def test_strides_of_several_entries_still_have_to_agree(compiled, monkeypatch):
    outs, lses = parts_of(2, 3, 4, 64, torch.bfloat16)
    o, x = outs.cuda(), lses.cuda()
    if not compiled:
        monkeypatch.setattr(N, "native", lambda: _NotHandled)
    heads_first = o[1].transpose(0, 1).contiguous().transpose(0, 1)
    with pytest.raises(ValueError, match="strides"):
        A.join_attention([o[0], heads_first], list(x))
    with pytest.raises(ValueError, match="strides"):
        A.join_attention(list(o), [x[0], x[1].t().contiguous().t()])
