"""Decoder-layer glue around the projections as single launches: residual add + RMSNorm, RoPE + KV-cache
store, SiLU * up. Host mirror of the reference's modules for these steps
(``nanovllm_voxcpm/layers/layernorm.py``, ``layers/activation.py``, ``layers/attention.py:10-49``,
``models/voxcpm2/model.py:81-94``), and the form of the middle one with norms of the heads; the kernels are ``csrc/glue.cuh`` and
``csrc/head_norm.cuh`` behind ``lora_b200_glue_*``.
CUDA tensors only, bf16 / fp16; there is no fallback path.
"""

from __future__ import annotations

import ctypes

import torch
import torch.nn as nn

from . import _native as N


def _rows(t: torch.Tensor, name: str) -> torch.Tensor:
    if t.dim() != 2 or t.stride(1) != 1:
        raise ValueError(f"{name} must be 2-D with unit column stride")
    return t


def add_rms_norm(x: torch.Tensor, residual: torch.Tensor | None, weight: torch.Tensor, eps: float, *,
                 norm_of_rounded_sum: bool = True, out: torch.Tensor | None = None,
                 hidden_out: torch.Tensor | None = None) -> tuple[torch.Tensor, torch.Tensor | None]:
    """``hidden = residual + x`` and ``normed = rms_norm(hidden) * weight`` in one pass over the rows.

    Returns ``(normed, hidden)``; ``hidden`` is ``None`` without a residual. ``hidden_out`` may be ``residual``
    itself (in place). ``norm_of_rounded_sum=False`` gives ``RMSNorm.add_rms_forward``'s rounding.
    """
    if out is None and hidden_out is None:
        got = N.native().add_rms_norm(x, residual, weight, eps, norm_of_rounded_sum)
        if got is not None:
            N.check(got[0])
            return got[1], got[2]
    N.require_cuda(x, residual, weight, out, hidden_out)
    shape = x.shape
    x2 = _rows(x.reshape(-1, shape[-1]), "x")
    T, H = x2.shape
    if weight.numel() != H or weight.dtype != x.dtype:
        raise ValueError("weight must have the row width and the dtype of x")
    normed = out if out is not None else torch.empty(T, H, dtype=x.dtype, device=x.device)
    normed2 = _rows(normed.reshape(-1, H), "out")
    res2 = hid2 = None
    if residual is not None:
        if residual.shape != shape or residual.dtype != x.dtype:
            raise ValueError("residual must match x")
        res2 = _rows(residual.reshape(-1, H), "residual")
        hidden = hidden_out if hidden_out is not None else torch.empty(T, H, dtype=x.dtype, device=x.device)
        hid2 = _rows(hidden.reshape(-1, H), "hidden_out")
    with N.on_device(x.device):
        N.check(N.lib().lora_b200_glue_add_rmsnorm(
            normed2.data_ptr(), normed2.stride(0), N.ptr(hid2), hid2.stride(0) if hid2 is not None else 0,
            x2.data_ptr(), x2.stride(0), N.ptr(res2), res2.stride(0) if res2 is not None else 0, weight.data_ptr(),
            T, H, float(eps), 1 if norm_of_rounded_sum else 0, N.dtype_code(x.dtype), N.current_stream(x.device)))
    return normed2.view(shape), (hid2.view(shape) if hid2 is not None else None)


class RMSNorm(nn.Module):
    """``layers/layernorm.py:6-42``: ``forward(x)`` -> normed; ``forward(x, residual)`` -> (normed, x + residual)."""

    def __init__(self, hidden_size: int, eps: float = 1e-6) -> None:
        super().__init__()
        self.eps = eps
        self.hidden_size = hidden_size
        self.weight = nn.Parameter(torch.ones(hidden_size))

    def rms_forward(self, x: torch.Tensor) -> torch.Tensor:
        return add_rms_norm(x, None, self.weight, self.eps)[0]

    def add_rms_forward(self, x: torch.Tensor, residual: torch.Tensor) -> tuple[torch.Tensor, torch.Tensor]:
        return add_rms_norm(x, residual, self.weight, self.eps, norm_of_rounded_sum=False)

    def forward(self, x: torch.Tensor, residual: torch.Tensor | None = None):
        return self.rms_forward(x) if residual is None else self.add_rms_forward(x, residual)


def silu_and_mul(x: torch.Tensor, out: torch.Tensor | None = None) -> torch.Tensor:
    if out is None:
        got = N.native().silu_mul(x)
        if got is not None:
            N.check(got[0])
            return got[1]
    N.require_cuda(x, out)
    shape = x.shape
    if shape[-1] % 2:
        raise ValueError("the last dim holds gate | up and must be even")
    inter = shape[-1] // 2
    x2 = _rows(x.reshape(-1, shape[-1]), "x")
    res = out if out is not None else torch.empty(x2.size(0), inter, dtype=x.dtype, device=x.device)
    res2 = _rows(res.reshape(-1, inter), "out")
    with N.on_device(x.device):
        N.check(N.lib().lora_b200_glue_silu_mul(res2.data_ptr(), res2.stride(0), x2.data_ptr(), x2.stride(0), x2.size(0),
                                                inter, N.dtype_code(x.dtype), N.current_stream(x.device)))
    return res2.view(*shape[:-1], inter)


class SiluAndMul(nn.Module):
    """``layers/activation.py:6-14``."""

    def forward(self, x: torch.Tensor) -> torch.Tensor:
        return silu_and_mul(x)


def rope_kv_store(qkv: torch.Tensor, num_heads: int, num_kv_heads: int, head_dim: int, *,
                  positions: torch.Tensor | None = None, cos: torch.Tensor | None = None, sin: torch.Tensor | None = None,
                  k_cache: torch.Tensor | None = None, v_cache: torch.Tensor | None = None,
                  slot_mapping: torch.Tensor | None = None) -> tuple[torch.Tensor, torch.Tensor, torch.Tensor]:
    """Rotates q and k of the packed ``qkv [T, (heads + 2 kv_heads) * head_dim]`` rows IN PLACE and stores the
    rotated k and v rows into the paged cache; returns the ``q, k, v`` views ``[T, heads, head_dim]``.

    ``cos`` / ``sin``: ``[max_position, head_dim]`` (the reference's ``cos_cached``) or ``[max_position,
    head_dim / 2]``; ``positions`` int64. Without them nothing is rotated. ``slot_mapping`` int32, -1 = skip;
    the caches are ``[..., kv_heads, head_dim]`` contiguous.
    """
    got = N.native().rope_kv_store(qkv, num_heads, num_kv_heads, head_dim, positions, cos, sin, k_cache, v_cache, slot_mapping)
    if got is not None:
        N.check(got[0])
        return got[1], got[2], got[3]
    N.require_cuda(qkv, positions, cos, sin, k_cache, v_cache, slot_mapping)
    qkv2 = _rows(qkv, "qkv")
    T = qkv2.size(0)
    q_size, kv_size = num_heads * head_dim, num_kv_heads * head_dim
    if qkv2.size(1) != q_size + 2 * kv_size:
        raise ValueError("qkv rows must hold q | k | v")
    rope = positions is not None or cos is not None or sin is not None
    table_dim = table_dtype = max_pos = 0
    if rope:
        if positions is None or cos is None or sin is None:
            raise ValueError("rotation needs positions, cos and sin")
        if positions.dtype != torch.int64 or positions.numel() != T or not positions.is_contiguous():
            raise ValueError("positions must be a contiguous int64 tensor with one entry per row")
        if cos.shape != sin.shape or cos.dim() != 2 or cos.dtype != sin.dtype or not (cos.is_contiguous() and sin.is_contiguous()):
            raise ValueError("cos and sin must be contiguous [max_position, dim] tables of one dtype")
        max_pos, table_dim = cos.shape
        table_dtype = N.dtype_code(cos.dtype)
    if (k_cache is None) != (v_cache is None):
        raise ValueError("k_cache and v_cache come together")
    if k_cache is not None:
        if slot_mapping is None or slot_mapping.dtype != torch.int32 or slot_mapping.numel() != T or not slot_mapping.is_contiguous():
            raise ValueError("slot_mapping must be a contiguous int32 tensor with one entry per row")
        for c in (k_cache, v_cache):
            if not c.is_contiguous() or c.dtype != qkv.dtype or c.numel() % kv_size:
                raise ValueError("the caches must be contiguous [..., kv_heads, head_dim] tensors of the dtype of qkv")
    with N.on_device(qkv.device):
        N.check(N.lib().lora_b200_glue_rope_kv_store(
            qkv2.data_ptr(), qkv2.stride(0), T, num_heads, num_kv_heads, head_dim, N.ptr(positions) if rope else None,
            N.ptr(cos) if rope else None, N.ptr(sin) if rope else None, table_dim, table_dtype, max_pos, N.ptr(k_cache),
            N.ptr(v_cache), N.ptr(slot_mapping) if k_cache is not None else None, N.dtype_code(qkv.dtype),
            N.current_stream(qkv.device)))
    q, k, v = qkv2.split([q_size, kv_size, kv_size], dim=-1)
    return (q.view(T, num_heads, head_dim), k.view(T, num_kv_heads, head_dim), v.view(T, num_kv_heads, head_dim))


def paged_cache(k_cache: torch.Tensor, v_cache: torch.Tensor, dtype: torch.dtype, kv_heads: int | None, head_dim: int) -> N.PagedCache:
    """The caches ``[blocks, block_size, kv_heads, head_dim]`` (any strides with adjacent elements in a head) as the library takes
    them."""
    shape = k_cache.shape
    if k_cache.dim() != 4 or v_cache.shape != shape or shape[3] != head_dim or (kv_heads is not None and shape[2] != kv_heads) or \
            min(shape) < 1:
        raise ValueError(f"the caches must be [blocks, block_size, kv_heads, head_dim] tensors of one shape, got {tuple(shape)} and "
                         f"{tuple(v_cache.shape)}")
    if k_cache.dtype != dtype or v_cache.dtype != dtype:
        raise ValueError(f"the caches must be {dtype}, as the rows are")
    if k_cache.stride(3) != 1 or v_cache.stride(3) != 1:
        raise ValueError("the elements of a cache row must be adjacent")
    return N.PagedCache(k_cache.data_ptr(), v_cache.data_ptr(), shape[0], shape[1], *k_cache.stride()[:3], *v_cache.stride()[:3])


def qk_norm_rope_kv_store(qkv: torch.Tensor, num_heads: int, num_kv_heads: int, head_dim: int, q_weight: torch.Tensor,
                          k_weight: torch.Tensor, eps: float, *, positions: torch.Tensor | None = None,
                          cos: torch.Tensor | None = None, sin: torch.Tensor | None = None, k_cache: torch.Tensor | None = None,
                          v_cache: torch.Tensor | None = None, slot_mapping: torch.Tensor | None = None,
                          q_out: torch.Tensor | None = None) -> tuple[torch.Tensor, torch.Tensor | None, torch.Tensor]:
    """``rope_kv_store`` with an RMS norm of every query and key head (``q_weight`` / ``k_weight`` ``[head_dim]``) ahead of the
    rotation; fp32 throughout, rounded once. The caches are ``[blocks, block_size, kv_heads, head_dim]`` and may be strided (one
    tensor that holds k and v of a block, heads ahead of positions); ``slot_mapping`` int32 holds block * block_size + position in
    the block, each at most once; slots outside the cache (-1) are skipped.

    Returns the ``q, k, v`` views of ``qkv``, q and k replaced IN PLACE; or, with ``q_out [T, num_heads, head_dim]``, leaves
    ``qkv`` as it is and returns ``q_out, None, v``: k is in the cache only."""
    if k_cache is not None:
        got = N.native().qk_norm_rope_kv_store(qkv, num_heads, num_kv_heads, head_dim, q_weight, k_weight, eps, positions, cos, sin,
                                               k_cache, v_cache, slot_mapping, q_out)
        if got is not None:
            N.check(got[0])
            return got[1], got[2], got[3]
    N.require_cuda(qkv, q_weight, k_weight, positions, cos, sin, k_cache, v_cache, slot_mapping, q_out)
    qkv2 = _rows(qkv, "qkv")
    T = qkv2.size(0)
    q_size, kv_size = num_heads * head_dim, num_kv_heads * head_dim
    if min(num_heads, num_kv_heads, head_dim) < 0 or qkv2.size(1) != q_size + 2 * kv_size:
        raise ValueError("qkv rows must hold q | k | v")
    for w in (q_weight, k_weight):
        if w.dtype != qkv.dtype or w.numel() != head_dim or not w.is_contiguous():
            raise ValueError("the norm weights must be contiguous [head_dim] vectors of the dtype of qkv")
    rope = positions is not None or cos is not None or sin is not None
    table_dim = table_dtype = max_pos = 0
    if rope:
        if positions is None or cos is None or sin is None:
            raise ValueError("rotation needs positions, cos and sin")
        if positions.dtype != torch.int64 or positions.numel() != T or not positions.is_contiguous():
            raise ValueError("positions must be a contiguous int64 tensor with one entry per row")
        if cos.shape != sin.shape or cos.dim() != 2 or cos.dtype != sin.dtype or not (cos.is_contiguous() and sin.is_contiguous()):
            raise ValueError("cos and sin must be contiguous [max_position, dim] tables of one dtype")
        max_pos, table_dim = cos.shape
        table_dtype = N.dtype_code(cos.dtype)
    if (k_cache is None) != (v_cache is None):
        raise ValueError("k_cache and v_cache come together")
    cache = None
    if k_cache is not None:
        if slot_mapping is None or slot_mapping.dtype != torch.int32 or slot_mapping.numel() != T or not slot_mapping.is_contiguous():
            raise ValueError("slot_mapping must be a contiguous int32 tensor with one entry per row")
        cache = paged_cache(k_cache, v_cache, qkv.dtype, num_kv_heads, head_dim)
    if q_out is not None:
        if cache is None:
            raise ValueError("with q_out, k goes to the cache only: it needs one")
        if q_out.shape != (T, num_heads, head_dim) or q_out.dtype != qkv.dtype or q_out.stride(2) != 1 or \
                (num_heads > 1 and q_out.stride(1) != head_dim):
            raise ValueError("q_out must be [T, num_heads, head_dim] of the dtype of qkv, with a token's heads side by side")
    devices = {t.device for t in (qkv, q_weight, k_weight, positions, cos, sin, k_cache, v_cache, slot_mapping, q_out) if t is not None}
    if len(devices) > 1:
        raise ValueError(f"tensors on several devices: {sorted(map(str, devices))}")
    with N.on_device(qkv.device):
        N.check(N.lib().lora_b200_glue_qk_norm_rope_kv_store(
            qkv2.data_ptr(), qkv2.stride(0), T, num_heads, num_kv_heads, head_dim, q_weight.data_ptr(), k_weight.data_ptr(), float(eps),
            N.ptr(positions), N.ptr(cos), N.ptr(sin), table_dim, table_dtype, max_pos, N.ptr(q_out),
            0 if q_out is None else q_out.stride(0) if T > 1 else q_size, None if cache is None else ctypes.byref(cache),
            N.ptr(slot_mapping) if cache is not None else None, N.dtype_code(qkv.dtype), N.current_stream(qkv.device)))
    q, k, v = qkv2.split([q_size, kv_size, kv_size], dim=-1)
    v = v.view(T, num_kv_heads, head_dim)
    return (q.view(T, num_heads, head_dim), k.view(T, num_kv_heads, head_dim), v) if q_out is None else (q_out, None, v)


def store_kvcache(key: torch.Tensor, value: torch.Tensor, k_cache: torch.Tensor, v_cache: torch.Tensor,
                  slot_mapping: torch.Tensor) -> None:
    """``layers/attention.py:33-49`` for key / value that are the k | v column ranges of one packed qkv buffer is
    what ``rope_kv_store`` does; this form takes separate ``[T, kv_heads, head_dim]`` tensors and copies them."""
    T, heads, dim = key.shape
    packed = torch.empty(T, 2 * heads * dim, dtype=key.dtype, device=key.device)
    packed[:, : heads * dim] = key.reshape(T, -1)
    packed[:, heads * dim:] = value.reshape(T, -1)
    rope_kv_store(packed, 0, heads, dim, k_cache=k_cache, v_cache=v_cache, slot_mapping=slot_mapping)
