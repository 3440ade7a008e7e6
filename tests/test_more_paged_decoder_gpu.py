"""Differential heads and shared prefixes in a decoder: head norms and rotation of the halves, store, attention of prompts, decode rows and
both, replayed from graphs. Against the same decoder with the plain torch glue and dense masked attention in fp32, or without the
groups; the bound is that of the other tests of this stack (two bf16 layers, each rounding a handful of intermediates to 2^-8: 6e-2)."""

import pytest
import torch

import test_differential_gpu as TD
from nanovllm_voxcpm_b200 import _native as N
from nanovllm_voxcpm_b200 import attention as A
from nanovllm_voxcpm_b200 import backbone as BB
from nanovllm_voxcpm_b200 import context as CTX

pytestmark = pytest.mark.gpu


@pytest.fixture(autouse=True)
def _clean():
    CTX.reset_lora_context()
    yield
    CTX.reset_lora_context()
    assert N.device_status() == 0


def _model(dim=64, **kw):
    cfg = BB.DecoderConfig(hidden_size=256, num_heads=8, num_kv_heads=2, head_dim=dim, intermediate_size=512, num_layers=2, max_loras=8,
                           max_lora_rank=32, max_position=8192, kv_block_size=64, **kw)
    with torch.device("cuda"):
        model = BB.Decoder(cfg).to(torch.bfloat16)
    model.init_random_(0, std=0.05)
    model.fill_adapter_slots_(8, 32, seed=1, std=0.05)
    gen = torch.Generator(device="cuda").manual_seed(2)
    with torch.no_grad():
        for layer in model.layers:
            a = layer.self_attn
            for w in ([a.q_norm, a.k_norm] if cfg.qk_norm else []) + ([a.diff_norm] if cfg.differential else []):
                w.copy_(1 + 0.3 * torch.randn(w.numel(), device="cuda", generator=gen))
            if cfg.differential:
                a.lam.copy_(torch.rand(a.lam.numel(), device="cuda", generator=gen))
    return model


def _dense(self, q, tables, contexts, new):
    cfg, outs, row = self.cfg, [], 0
    half, page = cfg.head_dim // 2, self.k_cache.size(1)
    for i, (n, c) in enumerate(zip(new, contexts)):
        j = torch.arange(c, device=q.device)
        place = tables[i].long()[j // page], j % page
        k, v = (x[place].float().repeat_interleave(q.size(1) // x.size(2), 1) for x in (self.k_cache, self.v_cache))
        p = torch.arange(c - n, c, device=q.device)[:, None]
        seen = j <= p
        if cfg.sliding_window:
            seen &= (p - j < cfg.sliding_window) | (j < cfg.sink_tokens)
        x = q[row:row + n].float()
        maps = [(torch.einsum("ihd,jhd->hij", x[..., m:m + half], k[..., m:m + half]) * half ** -0.5).masked_fill(~seen, float("-inf")).softmax(-1)
                for m in (0, half)]
        y = torch.einsum("hij,jhd->ihd", maps[0] - self.lam.float()[:, None, None] * maps[1], v)
        y = y * torch.rsqrt(y.square().mean(-1, keepdim=True) + cfg.rms_norm_eps) * self.diff_norm.float()
        outs.append(y.to(q.dtype))
        row += n
    return torch.cat(outs)


def _dense_attend(self, q, step):
    outs = []
    nd = step.n_decode if step.is_prefill else q.size(0)
    if nd:
        outs.append(_dense(self, q[:nd], step.block_tables, step.context_lens.tolist(), [1] * nd))
    if step.is_prefill:
        new = (step.cu_seqlens[1:] - step.cu_seqlens[:-1]).tolist()
        outs.append(_dense(self, q[nd:], step.prefill_block_tables, step.prefill_context_lens.tolist(), new))
    return torch.cat(outs)


FORMS = [dict(qk_norm=True, differential=True), dict(differential=True, dim=128), dict(qk_norm=True, differential=True, sliding_window=50, sink_tokens=3)]


@pytest.mark.parametrize("form", FORMS)
def test_differential_prefill_and_decode(form, monkeypatch):
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
    monkeypatch.setattr(BB.DecoderAttention, "_attend_paged", _dense_attend)
    model.fused_glue = False
    ref = BB.BackboneRunner(model, work)
    ref.prefill()
    torch.testing.assert_close(got[0], ref.last_output.float(), atol=6e-2, rtol=6e-2)
    ref.decode(3, use_graph=False)
    torch.testing.assert_close(got[1], ref.last_output.float(), atol=6e-2, rtol=6e-2)


def test_differential_mixed_step(monkeypatch):
    """Decode rows behind empty caches and a chunk of prompts in one step, every attention call of it against the 64-bit form of its own
    inputs. (Two decoders that round q and k differently cannot be held against one another here. A decode row sees 89 zero keys with
    zero values and its own: a head is y = (p1 - lam p2) v, which the norm makes v / rms(v) times the sign of p1 - lam p2, whatever is
    left of it. Errors d of p1 and p2 are errors (1 + lam) d / |p1 - lam p2| of the result, without bound where p1 = lam p2; those of the
    same inputs are bounded in ``test_differential_gpu.check``, which divides by what is left.)"""
    model = _model(**FORMS[0])
    model.fused_glue = True
    real, calls = BB.DecoderAttention._attend_paged, []

    def attend(self, q, step):
        out = real(self, q, step)
        cfg, nd = self.cfg, step.n_decode
        same = dict(k=self.k_cache.cpu(), v=self.v_cache.cpu(), window=cfg.sliding_window, sinks=cfg.sink_tokens, scale=cfg.rotary_dim ** -0.5,
                    lam=self.lam.float().detach().cpu(), weight=self.diff_norm.detach().cpu(), eps=cfg.rms_norm_eps)
        TD.check(dict(same, q=q[:nd].cpu(), tables=step.block_tables.tolist(), contexts=step.context_lens.tolist(), cu=None), out[:nd], "decode rows")
        TD.check(dict(same, q=q[nd:].cpu(), tables=step.prefill_block_tables.tolist(), contexts=step.prefill_context_lens.tolist(),
                      cu=step.cu_seqlens.tolist()), out[nd:], "prompts")
        calls.append(q.size(0))
        return out

    monkeypatch.setattr(BB.DecoderAttention, "_attend_paged", attend)
    _, _, out = BB.time_mixed_step(model, 24, [130, 70, 300], [i % 8 for i in range(24)], [2, -1, 5], context_len=90, iters=1, warmup=0)
    assert bool(out.isfinite().all()) and calls and set(calls) == {524}


@torch.inference_mode()
@pytest.mark.parametrize("mixed", [False, True])
def test_shared_prefix_steps(mixed):
    """A voice prompt of one request, prefilled once; then texts of all behind it as packed tokens, then decode steps from a graph, with
    groups and without."""
    model = _model(paged_attention=True, qk_norm=True)
    model.fused_glue = True
    n, prefix, width = 40, 1000, 100  # (tables wide enough for both calls to go by group)
    assert all(N.lib().lora_b200_shared_prefix_way(t, n, 1, 8, 2, 64, width, 64, packed) for t, packed in ((n, 0), (136, 1)))
    gen = torch.Generator(device="cuda").manual_seed(4)
    rand = lambda t: torch.randn(t, 256, device="cuda", generator=gen).to(torch.bfloat16)  # noqa: E731
    ints = lambda x: torch.tensor(x, dtype=torch.int32, device="cuda")  # noqa: E731
    full = prefix // 64
    tables = torch.full((n, width), -1, dtype=torch.int32)
    tables[:, :full] = torch.arange(full)
    tables[:, full:full + 2] = full + torch.arange(2 * n).view(n, 2)  # the block that the prefix ends in, copied, and one more
    tables = tables.cuda()
    text = [1 + 7 * i % 6 for i in range(n)]
    assert sum(text) == 136
    prompt, texts, rows = rand(prefix), rand(sum(text)), [rand(n) for _ in range(3)]
    groups = ints([prefix]), ints([0, n])

    def run(by_group):
        model.allocate_kv_cache(full + 2 * n)
        at = lambda r, p: tables[r].long()[p // 64] * 64 + p % 64  # noqa: E731
        pos = torch.arange(prefix, device="cuda")
        model(prompt, pos, BB.AttentionStep(True, at(0, pos), cu_seqlens=ints([0, prefix]), max_seqlen=prefix, prefill_context_lens=ints([prefix]),
                                            prefill_block_tables=tables[:1]))
        for layer in model.layers:
            for c in (layer.self_attn.k_cache, layer.self_attn.v_cache):
                c[tables[1:, full].long()] = c[tables[0, full].long()].clone()
        cu = [0]
        for t in text:
            cu.append(cu[-1] + t)
        pos = torch.cat([torch.arange(prefix, prefix + t, device="cuda") for t in text])
        slots = torch.cat([at(i, torch.arange(prefix, prefix + t, device="cuda")) for i, t in enumerate(text)])
        kw = dict(prefill_prefix_lens=groups[0], prefill_cu_groups=groups[1]) if by_group else {}
        outs = [model(texts, pos, BB.AttentionStep(True, slots, cu_seqlens=ints(cu), max_seqlen=max(text), prefill_context_lens=ints([prefix + t for t in text]),
                                                   prefill_block_tables=tables, **kw))]
        kw = dict(prefix_lens=groups[0], cu_groups=groups[1]) if by_group else {}
        lens = ints([prefix + t for t in text])
        embeds, pos, slots = rows[0].clone(), lens.long(), torch.empty(n, dtype=torch.int64, device="cuda")
        step = BB.AttentionStep(False, slots, context_lens=lens, block_tables=tables, **kw)
        graph = None
        for k in range(3):
            embeds.copy_(rows[k])
            pos.copy_(lens)
            slots.copy_(tables.long()[torch.arange(n, device="cuda"), pos // 64] * 64 + pos % 64)
            lens += 1
            if mixed:  # eager
                outs.append(model(embeds, pos, step))
                continue
            if graph is None:
                model(embeds, pos, step)
                torch.cuda.synchronize()
                graph = torch.cuda.CUDAGraph()
                with torch.cuda.graph(graph):
                    held = model(embeds, pos, step)
            graph.replay()
            outs.append(held.clone())
        return [o.float() for o in outs]

    for one, two in zip(run(True), run(False)):
        torch.testing.assert_close(one, two, atol=6e-2, rtol=6e-2)


@torch.inference_mode()
def test_steps_that_lack_or_mix_what_they_need():
    model = _model(paged_attention=True, sliding_window=64)
    model.fused_glue = True
    model.allocate_kv_cache(4)
    ints = lambda x: torch.tensor(x, dtype=torch.int32, device="cuda")  # noqa: E731
    embeds, pos, slots = torch.zeros(2, 256, device="cuda", dtype=torch.bfloat16), torch.zeros(2, dtype=torch.int64, device="cuda"), torch.arange(2, device="cuda") * 64
    step = BB.AttentionStep(False, slots, context_lens=ints([1, 1]), block_tables=ints([[0], [1]]), prefix_lens=ints([1]), cu_groups=ints([0, 2]))
    with pytest.raises(ValueError, match="by one map"):
        model(embeds, pos, step)
    step.cu_groups = None
    with pytest.raises(ValueError, match="come together"):
        model(embeds, pos, step)
    with pytest.raises(ValueError, match="64 or 128"):
        BB.DecoderConfig(differential=True, head_dim=96)


@pytest.mark.parametrize("heads", [(16, 2, 64), (32, 8, 128)])
def test_a_context_in_places_of_its_own(heads):
    """Several calls over parts of a context as they would be used side by side: a shared prefix, a part behind it, joined; and all of it by
    group in one call."""
    Hq, Hk, D = heads
    gen = torch.Generator(device="cuda").manual_seed(1)
    B, page, prefix, own = 24, 16, 4096, 64
    blocks = prefix // page + B * own // page
    k, v = (torch.randn(blocks, page, Hk, D, device="cuda", generator=gen).to(torch.bfloat16) for _ in range(2))
    q = torch.randn(B, Hq, D, device="cuda", generator=gen).to(torch.bfloat16)
    shared = torch.arange(prefix // page, device="cuda", dtype=torch.int32)
    mine = (prefix // page + torch.arange(B * own // page, device="cuda", dtype=torch.int32)).view(B, -1)
    lens = torch.arange(B, device="cuda", dtype=torch.int32) + 1
    ints = lambda x: torch.tensor(x, dtype=torch.int32, device="cuda")  # noqa: E731
    one = A.paged_decode_attention(q, k, v, shared.expand(B, -1), ints([prefix]).expand(B).contiguous(), return_lse=True)
    two = A.paged_decode_attention(q, k, v, mine, lens, return_lse=True)
    joined, lse = A.join_attention((one[0], two[0]), (one[1], two[1]), return_lse=True)
    tables = torch.cat((shared.expand(B, -1), mine, mine.new_full((B, 4096), -1)), 1)
    got, got_lse = A.shared_prefix_decode_attention(q, k, v, tables, lens + prefix, ints([prefix]), ints([0, B]), return_lse=True)
    u = 2.0 ** -8  # (the parts, the join and the one call round, each and in their products, by half a step of values up to max |v|)
    assert float((got.float() - joined.float()).abs().max()) <= 6 * u * float(v.float().abs().max())
    assert float((got_lse - lse).abs().max()) <= 1e-4
