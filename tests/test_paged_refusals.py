"""What the operators around the paged cache refuse before any launch: in Python on CPU tensors, and behind the C ABI with
addresses that are never read."""

import ctypes

import pytest
import torch

from nanovllm_voxcpm_b200 import _native as N
from nanovllm_voxcpm_b200 import attention as A
from nanovllm_voxcpm_b200 import glue as G

AT = 1 << 20  # a well-aligned address


def _cache(**kw):
    c = dict(k=AT, v=AT, num_blocks=4, block_size=16, k_block=2048, k_token=128, k_head=64, v_block=2048, v_token=128, v_head=64)
    c.update(kw)
    return N.PagedCache(**c)


def _decode(**kw):
    a = dict(out=AT, ot=1024, oh=64, lse=None, q=AT, qt=1024, qh=64, T=2, heads=16, kv=2, dim=64, cache=_cache(), tables=AT, ld=4, width=4,
             ctx=AT, scale=0.125, window=0, sinks=0, dtype=N.DT_BF16, ws=AT, bytes=1 << 30, stream=None)
    a.update(kw)
    a["cache"] = ctypes.byref(a["cache"]) if a["cache"] is not None else None
    return N.lib().lora_b200_paged_decode_attention(*a.values())


def _prefill(**kw):
    a = dict(out=AT, ot=1024, oh=64, lse=None, q=AT, qt=1024, qh=64, T=20, heads=16, kv=2, dim=64, cache=_cache(), tables=AT, ld=4, width=4,
             ctx=AT, cu=AT, n=2, scale=0.125, window=0, sinks=0, dtype=N.DT_BF16, ws=AT, bytes=1 << 30, stream=None)
    a.update(kw)
    a["cache"] = ctypes.byref(a["cache"]) if a["cache"] is not None else None
    return N.lib().lora_b200_paged_prefill_attention(*a.values())


BAD = [
    (dict(T=-1), N.E_INVAL), (dict(window=-1), N.E_INVAL), (dict(sinks=-1), N.E_INVAL), (dict(width=-1), N.E_INVAL), (dict(kv=0), N.E_INVAL),
    (dict(heads=15), N.E_INVAL), (dict(heads=0), N.E_INVAL), (dict(scale=0.0), N.E_INVAL), (dict(scale=-1.0), N.E_INVAL),
    (dict(scale=float("inf")), N.E_INVAL), (dict(scale=float("nan")), N.E_INVAL), (dict(dtype=N.DT_F32), N.E_UNSUPPORTED),
    (dict(dtype=9), N.E_UNSUPPORTED), (dict(dim=96), N.E_UNSUPPORTED), (dict(out=None), N.E_INVAL), (dict(q=None), N.E_INVAL),
    (dict(tables=None), N.E_INVAL), (dict(ctx=None), N.E_INVAL), (dict(cache=None), N.E_INVAL), (dict(cache=_cache(k=None)), N.E_INVAL),
    (dict(cache=_cache(v=None)), N.E_INVAL), (dict(cache=_cache(num_blocks=0)), N.E_INVAL), (dict(cache=_cache(block_size=0)), N.E_INVAL),
    (dict(cache=_cache(k=AT + 8)), N.E_UNSUPPORTED), (dict(cache=_cache(v_token=132)), N.E_UNSUPPORTED), (dict(q=AT + 2), N.E_UNSUPPORTED),
    (dict(qh=68), N.E_UNSUPPORTED), (dict(ot=1028), N.E_UNSUPPORTED), (dict(width=1 << 16, ws=None), N.E_WORKSPACE), (dict(width=1 << 16, bytes=16), N.E_WORKSPACE),
    (dict(ws=AT + 4), N.E_UNSUPPORTED),
]


@pytest.mark.parametrize("kw,code", BAD)
def test_attention_statuses(kw, code):
    assert _decode(**kw) == code and N.lib().lora_b200_last_error()
    assert _prefill(**kw) == code


def test_prefill_needs_cu_seqlens_and_takes_empty_calls():
    assert _prefill(cu=None) == N.E_INVAL and _prefill(n=-1) == N.E_INVAL
    assert _prefill(T=0) == 0 and _prefill(n=0) == 0 and _decode(T=0) == 0


def _store(**kw):
    a = dict(qkv=AT, ld=1280, T=2, hq=16, hk=2, d=64, qw=AT, kw=AT, eps=1e-6, pos=AT, cos=AT, sin=AT, dim=32, tdt=N.DT_F32, max=64, out=None,
             out_ld=0, cache=_cache(), slots=AT, dtype=N.DT_BF16, stream=None)
    a.update(kw)
    a["cache"] = ctypes.byref(a["cache"]) if a["cache"] is not None else None
    return N.lib().lora_b200_glue_qk_norm_rope_kv_store(*a.values())


@pytest.mark.parametrize("kw,code", [
    (dict(T=-1), N.E_INVAL), (dict(hq=-1), N.E_INVAL), (dict(d=0), N.E_INVAL), (dict(d=72), N.E_UNSUPPORTED), (dict(d=272), N.E_UNSUPPORTED),
    (dict(dtype=N.DT_F32), N.E_UNSUPPORTED), (dict(qkv=None), N.E_INVAL), (dict(qw=None), N.E_INVAL), (dict(kw=None), N.E_INVAL),
    (dict(ld=1272), N.E_INVAL), (dict(ld=1284), N.E_UNSUPPORTED), (dict(qkv=AT + 8), N.E_UNSUPPORTED), (dict(qw=AT + 2), N.E_UNSUPPORTED),
    (dict(pos=None), N.E_INVAL), (dict(sin=None), N.E_INVAL), (dict(max=0), N.E_INVAL), (dict(dim=48), N.E_INVAL), (dict(tdt=7), N.E_INVAL),
    (dict(slots=None), N.E_INVAL), (dict(cache=_cache(v=None)), N.E_INVAL), (dict(cache=_cache(k=None)), N.E_INVAL),
    (dict(cache=_cache(k_head=4)), N.E_UNSUPPORTED), (dict(out=AT, out_ld=1024, cache=None), N.E_INVAL), (dict(out=AT, out_ld=1016), N.E_INVAL),
    (dict(out=AT + 8, out_ld=1024), N.E_UNSUPPORTED), (dict(out=AT, out_ld=1028), N.E_UNSUPPORTED),
])
def test_store_statuses(kw, code):
    assert _store(**kw) == code and N.lib().lora_b200_last_error()
    assert _store(T=0) == 0


def test_cpu_tensors_are_refused():
    q, k = torch.zeros(1, 16, 64, dtype=torch.bfloat16), torch.zeros(4, 16, 2, 64, dtype=torch.bfloat16)
    tables, ctx = torch.zeros(1, 4, dtype=torch.int32), torch.ones(1, dtype=torch.int32)
    with pytest.raises(RuntimeError, match="CUDA"):
        A.paged_decode_attention(q, k, k, tables, ctx)
    with pytest.raises(RuntimeError, match="CUDA"):
        A.paged_prefill_attention(q, k, k, tables, ctx, torch.tensor([0, 1], dtype=torch.int32))
    one = torch.ones(64, dtype=torch.bfloat16)
    with pytest.raises(RuntimeError, match="CUDA"):
        G.qk_norm_rope_kv_store(torch.zeros(1, 1280, dtype=torch.bfloat16), 16, 2, 64, one, one, 1e-6)


def test_oracle_agrees_with_masked_softmax():
    """The oracle's own arithmetic, on a case small enough to write out as one masked softmax."""
    import paged_problem as PP
    from oracle import paged_oracle as PO

    p = PP.make(4, 2, 64, 8, [20, 9], [6, 9], window=5, sinks=2, device="cpu")
    out, lse, _, count = PO.paged_attention(p["q"], p["k"], p["v"], p["tables"], p["contexts"], p["cu"], p["scale"], 5, 2)
    row = 0
    for r, (n, c) in enumerate(zip([6, 9], [20, 9])):
        flat = [p["tables"][r][j // 8] * 8 + j % 8 for j in range(c)]
        k, v = (x.reshape(-1, 2, 64)[flat].double().repeat_interleave(2, 1) for x in (p["k"], p["v"]))
        s = torch.einsum("ihd,jhd->hij", p["q"][row:row + n].double(), k) * p["scale"]
        i, j = torch.arange(c - n, c)[:, None], torch.arange(c)[None]
        s = s.masked_fill(~((j <= i) & ((i - j < 5) | (j < 2))), float("-inf"))
        torch.testing.assert_close(out[row:row + n], torch.einsum("hij,jhd->ihd", s.softmax(-1), v))
        torch.testing.assert_close(lse[row:row + n], s.logsumexp(-1).T)
        assert count[row:row + n].tolist() == [int(x) for x in (s[0] > float("-inf")).sum(-1)]
        row += n


def test_decoder_config_refuses_what_attention_does():
    from nanovllm_voxcpm_b200.backbone import DecoderConfig

    assert DecoderConfig(sliding_window=64, sink_tokens=2).paged_attention and not DecoderConfig().paged_attention
    for kw in (dict(sliding_window=-1), dict(sink_tokens=-1, sliding_window=4), dict(sink_tokens=2)):
        with pytest.raises(ValueError):
            DecoderConfig(**kw)


def test_prefill_without_cu_seqlens_is_refused_by_name():
    """As many rows as requests would pass for a decode batch otherwise."""
    q, k = torch.zeros(2, 16, 64, dtype=torch.bfloat16), torch.zeros(4, 16, 2, 64, dtype=torch.bfloat16)
    with pytest.raises(ValueError, match="cu_seqlens"):
        A.paged_prefill_attention(q, k, k, torch.zeros(2, 4, dtype=torch.int32), torch.ones(2, dtype=torch.int32), None)


@pytest.mark.parametrize("missing", ["prefill_context_lens", "prefill_block_tables", "cu_seqlens", "context_lens", "block_tables"])
def test_steps_without_what_paged_attention_needs(missing):
    from nanovllm_voxcpm_b200 import backbone as BB

    cfg = BB.DecoderConfig(hidden_size=128, num_heads=2, num_kv_heads=1, head_dim=64, intermediate_size=128, num_layers=1, max_loras=2,
                           max_lora_rank=16, max_position=64, sliding_window=8)
    layer = BB.DecoderAttention(cfg)
    ints = torch.ones(1, dtype=torch.int32)
    step = BB.AttentionStep(True, torch.arange(3), cu_seqlens=torch.tensor([0, 2], dtype=torch.int32), max_seqlen=2, context_lens=ints,
                            block_tables=ints.view(1, 1), n_decode=1, prefill_context_lens=2 * ints, prefill_block_tables=ints.view(1, 1))
    setattr(step, missing, None)
    with pytest.raises(ValueError, match=missing):
        layer._attend_paged(torch.zeros(3, 2, 64, dtype=torch.bfloat16), step)
    if missing in ("context_lens", "block_tables"):
        with pytest.raises(ValueError, match=missing):
            layer._attend_paged(torch.zeros(1, 2, 64, dtype=torch.bfloat16), BB.AttentionStep(False, torch.arange(1), **{
                "context_lens": ints, "block_tables": ints.view(1, 1), missing: None}))


@pytest.mark.parametrize("call", [_decode, _prefill])
def test_scales_that_overflow_in_units_of_log2(call):
    """Scores are kept in units of log2: a scale that is finite, but not times log2(e), would turn scores of zero into NaN."""
    assert call(scale=2.9e38) == N.E_INVAL and call(scale=2.4e38) == N.E_INVAL and b"log2" in N.lib().lora_b200_last_error()
    assert call(scale=2.3e38, T=0) == 0
