"""What attention behind a shared prefix, differential attention and the join refuse before any launch: in Python on CPU tensors, and behind the C ABI with addresses
that are never read."""

import ctypes

import pytest
import torch

from nanovllm_voxcpm_b200 import _native as N
from nanovllm_voxcpm_b200 import attention as A

AT = 1 << 20  # a well-aligned address


def _cache(**kw):
    c = dict(k=AT, v=AT, num_blocks=4, block_size=16, k_block=2048, k_token=128, k_head=64, v_block=2048, v_token=128, v_head=64)
    c.update(kw)
    return N.PagedCache(**c)


def _differential(**kw):
    a = dict(out=AT, ot=1024, oh=64, q=AT, qt=1024, qh=64, T=2, heads=16, kv=2, dim=64, cache=_cache(), tables=AT, ld=4, width=4, ctx=AT,
             cu=None, n=2, lam=AT, lt=0, lh=1, weight=AT, eps=1e-5, scale=0.125, window=0, sinks=0, dtype=N.DT_BF16, ws=AT, bytes=1 << 30,
             stream=None)
    a.update(kw)
    a["cache"] = ctypes.byref(a["cache"]) if a["cache"] is not None else None
    return N.lib().lora_b200_differential_attention(*a.values())


@pytest.mark.parametrize("kw,code", [
    (dict(T=-1), N.E_INVAL), (dict(n=-1), N.E_INVAL), (dict(window=-1), N.E_INVAL), (dict(sinks=-1), N.E_INVAL), (dict(width=-1), N.E_INVAL),
    (dict(kv=0), N.E_INVAL), (dict(heads=15), N.E_INVAL), (dict(heads=0), N.E_INVAL), (dict(scale=0.0), N.E_INVAL),
    (dict(scale=float("nan")), N.E_INVAL), (dict(scale=3e38), N.E_INVAL), (dict(dtype=N.DT_F32), N.E_UNSUPPORTED), (dict(dim=96), N.E_UNSUPPORTED),
    (dict(dim=32), N.E_UNSUPPORTED), (dict(dim=256), N.E_UNSUPPORTED), (dict(out=None), N.E_INVAL), (dict(q=None), N.E_INVAL),
    (dict(tables=None), N.E_INVAL), (dict(ctx=None), N.E_INVAL), (dict(cache=None), N.E_INVAL), (dict(cache=_cache(k=None)), N.E_INVAL),
    (dict(cache=_cache(block_size=0)), N.E_INVAL), (dict(cache=_cache(v=AT + 8)), N.E_UNSUPPORTED), (dict(cache=_cache(k_token=132)), N.E_UNSUPPORTED),
    (dict(q=AT + 2), N.E_UNSUPPORTED), (dict(oh=68), N.E_UNSUPPORTED), (dict(lam=None), N.E_INVAL), (dict(n=3), N.E_INVAL),
    (dict(eps=0.0), N.E_INVAL), (dict(eps=float("inf")), N.E_INVAL), (dict(eps=float("nan")), N.E_INVAL), (dict(weight=AT + 8), N.E_UNSUPPORTED),
    (dict(width=1 << 16, ws=None), N.E_WORKSPACE), (dict(width=1 << 16, bytes=16), N.E_WORKSPACE), (dict(ws=AT + 4), N.E_UNSUPPORTED),
    (dict(cu=AT, width=1 << 16, ws=None), N.E_WORKSPACE), (dict(T=0), 0), (dict(n=0), 0), (dict(T=0, lam=None), 0),
])
def test_differential_statuses(kw, code):
    assert _differential(**kw) == code


def _shared(**kw):
    a = dict(out=AT, ot=1024, oh=64, lse=None, q=AT, qt=1024, qh=64, T=2, heads=16, kv=2, dim=64, cache=_cache(), tables=AT, ld=4, width=4, ctx=AT,
             cu=None, n=2, prefix=AT, cu_groups=AT, groups=1, scale=0.125, dtype=N.DT_BF16, ws=AT, bytes=1 << 30, stream=None)
    a.update(kw)
    a["cache"] = ctypes.byref(a["cache"]) if a["cache"] is not None else None
    return N.lib().lora_b200_shared_prefix_attention(*a.values())


@pytest.mark.parametrize("kw,code", [
    (dict(T=-1), N.E_INVAL), (dict(n=-1), N.E_INVAL), (dict(groups=-1), N.E_INVAL), (dict(width=-1), N.E_INVAL), (dict(kv=0), N.E_INVAL),
    (dict(heads=15), N.E_INVAL), (dict(scale=0.0), N.E_INVAL), (dict(scale=float("inf")), N.E_INVAL), (dict(dtype=N.DT_F32), N.E_UNSUPPORTED),
    (dict(dim=96), N.E_UNSUPPORTED), (dict(out=None), N.E_INVAL), (dict(q=None), N.E_INVAL), (dict(tables=None), N.E_INVAL),
    (dict(ctx=None), N.E_INVAL), (dict(cache=None), N.E_INVAL), (dict(cache=_cache(v=None)), N.E_INVAL), (dict(cache=_cache(num_blocks=0)), N.E_INVAL),
    (dict(cache=_cache(k=AT + 8)), N.E_UNSUPPORTED), (dict(q=AT + 2), N.E_UNSUPPORTED), (dict(oh=68), N.E_UNSUPPORTED), (dict(prefix=None), N.E_INVAL),
    (dict(cu_groups=None), N.E_INVAL), (dict(n=3), N.E_INVAL), (dict(width=1 << 16, ws=None), N.E_WORKSPACE), (dict(width=1 << 16, bytes=16), N.E_WORKSPACE),
    (dict(ws=AT + 4), N.E_UNSUPPORTED), (dict(cu=AT, width=1 << 16, ws=None), N.E_WORKSPACE), (dict(T=0), 0), (dict(n=0), 0),
    (dict(T=0, prefix=None), 0),
])
def test_shared_prefix_statuses(kw, code):
    assert _shared(**kw) == code


def _join(parts=2, **kw):
    a = dict(out=AT, ot=1024, oh=64, lse=None, outs=[AT] * parts, lses=[AT] * parts, n=parts, pt=1024, ph=64, lt=16, lh=1, T=2, heads=16, dim=64,
             dtype=N.DT_BF16, stream=None)
    a.update(kw)
    for name in ("outs", "lses"):
        if a[name] is not None:
            a[name] = (ctypes.c_void_p * max(1, len(a[name])))(*a[name])
    return N.lib().lora_b200_join_attention(*a.values())


@pytest.mark.parametrize("kw,code", [
    (dict(T=-1), N.E_INVAL), (dict(heads=0), N.E_INVAL), (dict(dim=0), N.E_INVAL), (dict(n=0), N.E_INVAL), (dict(parts=65), N.E_UNSUPPORTED),
    (dict(dtype=7), N.E_UNSUPPORTED), (dict(dim=68), N.E_UNSUPPORTED), (dict(dim=66, dtype=N.DT_F32), N.E_UNSUPPORTED), (dict(out=None), N.E_INVAL),
    (dict(outs=None), N.E_INVAL), (dict(lses=None), N.E_INVAL), (dict(outs=[AT, None]), N.E_INVAL), (dict(lses=[None, AT]), N.E_INVAL),
    (dict(outs=[AT, AT + 8]), N.E_UNSUPPORTED), (dict(out=AT + 8), N.E_UNSUPPORTED), (dict(ph=68), N.E_UNSUPPORTED), (dict(pt=1028), N.E_UNSUPPORTED),
    (dict(ot=1028), N.E_UNSUPPORTED), (dict(oh=68), N.E_UNSUPPORTED), (dict(T=2 ** 31 - 1, heads=65536, dim=65536), N.E_UNSUPPORTED), (dict(T=0), 0),
])
def test_join_statuses(kw, code):
    assert _join(**kw) == code


def test_python_refusals_without_a_gpu():
    q, cache = torch.zeros(2, 16, 64), torch.zeros(4, 16, 2, 64)
    ints = torch.zeros(2, 1, dtype=torch.int32)
    with pytest.raises(RuntimeError, match="CUDA tensors only"):
        A.differential_decode_attention(q, cache, cache, ints, ints[:, 0].contiguous(), torch.zeros(16))
    with pytest.raises(ValueError, match="cu_seqlens"):
        A.differential_prefill_attention(q, cache, cache, ints, ints[:, 0].contiguous(), None, torch.zeros(16))
    groups = torch.tensor([0, 2], dtype=torch.int32)
    with pytest.raises(RuntimeError, match="CUDA tensors only"):
        A.shared_prefix_decode_attention(q, cache, cache, ints, ints[:, 0].contiguous(), groups[:1], groups)
    with pytest.raises(ValueError, match="cu_seqlens"):
        A.shared_prefix_prefill_attention(q, cache, cache, ints, ints[:, 0].contiguous(), None, groups[:1], groups)
    with pytest.raises(RuntimeError, match="CUDA tensors only"):
        A.join_attention(torch.zeros(2, 2, 4, 64), torch.zeros(2, 2, 4))
    with pytest.raises(ValueError, match="one of each"):
        A.join_attention([], [])


def _on_gpu():
    q, cache = torch.zeros(2, 16, 64, device="cuda", dtype=torch.bfloat16), torch.zeros(4, 16, 2, 64, device="cuda", dtype=torch.bfloat16)
    tables, lens = torch.zeros(2, 1, dtype=torch.int32, device="cuda"), torch.ones(2, dtype=torch.int32, device="cuda")
    return q, cache, tables, lens, torch.zeros(16, device="cuda")


@pytest.mark.gpu
def test_python_refusals_on_a_gpu():
    q, cache, tables, lens, lam = _on_gpu()
    call = A.differential_decode_attention
    for bad in (lam[:8], lam.double(), lam.expand(3, 16), lam.view(1, 1, 16)):
        with pytest.raises(ValueError, match="lam"):
            call(q, cache, cache, tables, lens, bad)
    for bad in (lam, torch.ones(32, device="cuda", dtype=torch.bfloat16), torch.ones(128, device="cuda", dtype=torch.bfloat16)[::2]):
        with pytest.raises(ValueError, match="norm_weight"):
            call(q, cache, cache, tables, lens, lam, norm_weight=bad)
    weight = torch.ones(64, device="cuda", dtype=torch.bfloat16)
    for eps in (0.0, -1.0, float("nan")):
        with pytest.raises(ValueError, match="eps"):
            call(q, cache, cache, tables, lens, lam, norm_weight=weight, eps=eps)
    with pytest.raises(ValueError, match="sinks"):
        call(q, cache, cache, tables, lens, lam, sinks=1)
    with pytest.raises(ValueError, match="one of each"):
        call(q, cache, cache, tables[:1], lens[:1], lam)
    with pytest.raises(ValueError, match="scale"):
        call(q, cache, cache, tables, lens, lam, scale=0.0)
    with pytest.raises(RuntimeError, match="CUDA tensors only"):
        call(q, cache, cache, tables, lens, lam.cpu())
    with pytest.raises(ValueError, match="cu_seqlens"):
        A.differential_prefill_attention(q, cache, cache, tables, lens, lens, lam)
    with pytest.raises(RuntimeError, match="head_dim"):
        call(q[..., :32].contiguous(), cache[..., :32].contiguous(), cache[..., :32].contiguous(), tables, lens, lam)
    groups = torch.tensor([0, 2, 2], dtype=torch.int32, device="cuda")
    for prefix, cu, what in ((lens[:1], groups, "cu_groups"), (lens, groups[:2], "cu_groups"), (lens.long(), groups, "prefix_lens"),
                             (lens, groups.long(), "cu_groups"), (lens[None], groups, "vectors"), (groups[::2], groups, "vectors")):
        with pytest.raises(ValueError, match=what):
            A.shared_prefix_decode_attention(q, cache, cache, tables, lens, prefix, cu)
    with pytest.raises(RuntimeError, match="CUDA tensors only"):
        A.shared_prefix_decode_attention(q, cache, cache, tables, lens, lens.cpu(), groups)
    with pytest.raises(ValueError, match="one of each"):
        A.shared_prefix_decode_attention(q, cache, cache, tables[:1], lens[:1], lens, groups)
    outs, lses = torch.zeros(2, 3, 4, 64, device="cuda"), torch.zeros(2, 3, 4, device="cuda")
    for args, what in (((outs, lses[:1]), "one of each"), (([outs[0], outs[1, :2]], lses), "shape"), (([outs[0], outs[1].half()], lses), "dtype"),
                       ((outs, lses.double()), "float32"), ((outs[0], lses), "one of each|must be"), ((outs, lses[:, :, :2]), "float32")):
        with pytest.raises(ValueError, match=what):
            A.join_attention(*args)
    with pytest.raises(ValueError, match="out must"):
        A.join_attention(outs, lses, out=outs[0, :2])
    with pytest.raises(RuntimeError, match="head_dim"):
        A.join_attention(outs[..., :6].contiguous(), lses)
    with pytest.raises(RuntimeError, match="64 at most"):
        A.join_attention([outs[0]] * 65, [lses[0]] * 65)
