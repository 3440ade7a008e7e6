"""The operators around the paged cache together, as a decoder calls them: head norms + rotation + store, prefill attention, decode
attention, with a sliding window and first tokens, in prefill steps, graph-replayed decode steps and steps that mix both. Against the
same decoder with the plain torch glue and dense masked attention in fp32; the bound is that of the other tests of this stack (two
bf16 layers, each rounding a handful of intermediates to 2^-8: 6e-2)."""

import pytest
import torch

from nanovllm_voxcpm_b200 import _native as N
from nanovllm_voxcpm_b200 import backbone as BB
from nanovllm_voxcpm_b200 import context as CTX

pytestmark = pytest.mark.gpu


@pytest.fixture(autouse=True)
def _clean():
    CTX.reset_lora_context()
    yield
    CTX.reset_lora_context()
    assert N.device_status() == 0


def _dense(q, k_cache, v_cache, tables, contexts, new, window, sinks):
    outs, row = [], 0
    page = k_cache.size(1)
    for i, (n, c) in enumerate(zip(new, contexts)):
        j = torch.arange(c, device=q.device)
        place = tables[i].long()[j // page], j % page
        k, v = (x[place].float().repeat_interleave(q.size(1) // x.size(2), 1) for x in (k_cache, v_cache))
        s = torch.einsum("ihd,jhd->hij", q[row:row + n].float(), k) * q.size(-1) ** -0.5
        p = torch.arange(c - n, c, device=q.device)[:, None]
        seen = j <= p
        if window:
            seen &= (p - j < window) | (j < sinks)
        outs.append(torch.einsum("hij,jhd->ihd", s.masked_fill(~seen, float("-inf")).softmax(-1), v).to(q.dtype))
        row += n
    return torch.cat(outs)


def _dense_attend(self, q, step):
    cfg, outs = self.cfg, []
    nd = step.n_decode if step.is_prefill else q.size(0)
    if nd:
        outs.append(_dense(q[:nd], self.k_cache, self.v_cache, step.block_tables, step.context_lens.tolist(), [1] * nd, cfg.sliding_window, cfg.sink_tokens))
    if step.is_prefill:
        new = (step.cu_seqlens[1:] - step.cu_seqlens[:-1]).tolist()
        outs.append(_dense(q[nd:], self.k_cache, self.v_cache, step.prefill_block_tables, step.prefill_context_lens.tolist(), new, cfg.sliding_window,
                           cfg.sink_tokens))
    return torch.cat(outs)


def _model(**kw):
    cfg = BB.DecoderConfig(hidden_size=256, num_heads=8, num_kv_heads=2, head_dim=64, intermediate_size=512, num_layers=2, max_loras=8,
                           max_lora_rank=32, max_position=1024, kv_block_size=64, **kw)
    with torch.device("cuda"):
        model = BB.Decoder(cfg).to(torch.bfloat16)
    model.init_random_(0, std=0.05)
    model.fill_adapter_slots_(8, 32, seed=1, std=0.05)
    if cfg.qk_norm:
        gen = torch.Generator(device="cuda").manual_seed(2)
        with torch.no_grad():
            for layer in model.layers:
                for w in (layer.self_attn.q_norm, layer.self_attn.k_norm):
                    w.copy_(1 + 0.3 * torch.randn(64, device="cuda", generator=gen))
    return model


def _plain(monkeypatch, model):
    monkeypatch.setattr(BB.DecoderAttention, "_attend_paged", _dense_attend)
    model.fused_glue = False


FORMS = [dict(qk_norm=True, sliding_window=50, sink_tokens=3), dict(qk_norm=True, paged_attention=True), dict(sliding_window=128),
         dict(paged_attention=True)]


@pytest.mark.parametrize("form", FORMS)
def test_prefill_and_decode(form, monkeypatch):
    model = _model(**form)
    model.fused_glue = True
    work = BB.BackboneWorkload([200, 17, 264, 5, 114], [0, 3, -1, 3, 7], decode_steps=3)
    got = []
    for graph in (True, False):
        run = BB.BackboneRunner(model, work)
        run.prefill()
        got.append(run.last_output.float())
        run.decode(3, use_graph=graph)
        got.append(run.last_output.float())
    assert torch.equal(got[0], got[2]) and torch.equal(got[1], got[3]), "graph replay and eager launches differ"
    _plain(monkeypatch, model)
    ref = BB.BackboneRunner(model, work)
    ref.prefill()
    torch.testing.assert_close(got[0], ref.last_output.float(), atol=6e-2, rtol=6e-2)
    ref.decode(3, use_graph=False)
    torch.testing.assert_close(got[1], ref.last_output.float(), atol=6e-2, rtol=6e-2)


@pytest.mark.parametrize("form", FORMS[:2])
def test_mixed_step(form, monkeypatch):
    model = _model(**form)
    model.fused_glue = True
    lens = [130, 70, 300]
    args = (model, 24, lens, [i % 8 for i in range(24)], [2, -1, 5])
    _, _, out = BB.time_mixed_step(*args, context_len=90, iters=1, warmup=0)
    _plain(monkeypatch, model)
    _, _, ref = BB.time_mixed_step(*args, context_len=90, iters=1, warmup=0)
    torch.testing.assert_close(out.float(), ref.float(), atol=6e-2, rtol=6e-2)


@torch.inference_mode()
def test_prompt_in_chunks():
    """A prompt in three chunks, each behind those before it in the cache, gives what it gives in one."""
    model = _model(qk_norm=True, sliding_window=70, sink_tokens=4)
    model.fused_glue = True
    n = 333
    model.allocate_kv_cache(8)
    tables = torch.tensor([[5, 0, 7, 2, 1, 6]], dtype=torch.int32, device="cuda")
    embeds = torch.randn(n, 256, device="cuda", generator=torch.Generator(device="cuda").manual_seed(3)).to(torch.bfloat16)
    pos = torch.arange(n, device="cuda")
    slots = tables[0].long()[pos // 64] * 64 + pos % 64

    def step(a, b):
        s = BB.AttentionStep(True, slots[a:b], cu_seqlens=torch.tensor([0, b - a], dtype=torch.int32, device="cuda"), max_seqlen=b - a,
                             prefill_context_lens=torch.tensor([b], dtype=torch.int32, device="cuda"), prefill_block_tables=tables)
        return model(embeds[a:b], pos[a:b], s).float()

    whole = step(0, n)
    parts = torch.cat([step(0, 100), step(100, 101), step(101, n)])
    torch.testing.assert_close(parts, whole, atol=6e-2, rtol=6e-2)
