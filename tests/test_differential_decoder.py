"""The weight of a differential decoder's second maps: fp32, as the attention takes it, whatever type the model is given."""

import pytest
import torch

from nanovllm_voxcpm_b200 import attention as A
from nanovllm_voxcpm_b200 import backbone as BB


def _attention(**kw):
    cfg = BB.DecoderConfig(hidden_size=64, num_heads=4, num_kv_heads=2, head_dim=64, intermediate_size=64, num_layers=1, max_loras=2, max_lora_rank=8,
                           max_position=64, **kw)
    return BB.DecoderAttention(cfg)


@pytest.mark.parametrize("change", [lambda m: m.to(torch.bfloat16), lambda m: m.half(), lambda m: m.to("cpu", torch.bfloat16), lambda m: m.double()])
def test_lam_keeps_its_bits(change):
    module = torch.nn.Sequential(_attention(differential=True))
    lam = torch.rand(4)
    with torch.no_grad():
        module[0].lam.copy_(lam)
    parameter = module[0].lam
    change(module)
    assert module[0].diff_norm.dtype != torch.float32 and module[0].qkv_proj.weight.dtype == module[0].diff_norm.dtype
    assert module[0].lam is parameter and module[0].lam.dtype == torch.float32 and torch.equal(module[0].lam.data, lam)
    assert [n for n, _ in module.named_parameters()].count("0.lam") == 1


def test_a_state_of_another_type_is_taken():
    one, two = _attention(differential=True).to(torch.bfloat16), _attention(differential=True).to(torch.bfloat16)
    state = {k: v.to(torch.bfloat16) if k == "lam" else v for k, v in one.state_dict().items()}
    two.load_state_dict(state)
    assert two.lam.dtype == torch.float32 and torch.equal(two.lam.data, torch.full((4,), 0.5))


def test_a_decoder_without_maps_has_none():
    assert not hasattr(_attention().to(torch.bfloat16), "lam")


@pytest.mark.parametrize("packed", [False, True])
def test_the_attention_is_given_the_parameter_itself(packed, monkeypatch):
    """No cast of its own in a step: what the call takes is what the module holds."""
    given = []
    for name in ("differential_decode_attention", "differential_prefill_attention"):
        monkeypatch.setattr(A, name, lambda *args, **kw: given.append(args[6 if packed else 5]))
    module = _attention(differential=True).to(torch.bfloat16)
    ints = torch.zeros(2, dtype=torch.int32)
    step = BB.AttentionStep(is_prefill=packed, cu_seqlens=torch.tensor([0, 1, 2], dtype=torch.int32), context_lens=ints, block_tables=ints[:, None],
                            prefill_context_lens=ints, prefill_block_tables=ints[:, None], slot_mapping=None)
    module._attend_paged(torch.zeros(2, 4, 64, dtype=torch.bfloat16), step)
    assert len(given) == 1 and given[0] is module.lam
