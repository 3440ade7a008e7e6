"""Attention over the paged key-value cache that ``glue.rope_kv_store`` and ``glue.qk_norm_rope_kv_store`` fill: the next token
of every request (``paged_decode_attention``) or packed runs of new tokens (``paged_prefill_attention``: whole prompts, chunks of
them, a few tokens behind a long context). Causal, over everything or over a sliding window of the last keys plus a few first
ones. Stands where the reference attends over its paged cache
(``nanovllm_voxcpm/layers/attention.py:70-79``); the kernels are ``csrc/paged_attention.cuh`` and ``csrc/paged_prefill.cuh`` behind
``lora_b200_paged_*``.
CUDA tensors only, bf16 / fp16, heads of 64 or 128; there is no fallback path and no backward pass.
"""

from __future__ import annotations

import ctypes
import math

import torch

from . import _native as N
from .glue import paged_cache


def _int32(t: torch.Tensor, name: str, shape: tuple) -> torch.Tensor:
    if t.dtype != torch.int32 or tuple(t.shape) != shape:
        raise ValueError(f"{name} must be an int32 tensor of shape {shape}, got {t.dtype} {tuple(t.shape)}")
    return t


def _paged_attention(q, k_cache, v_cache, block_tables, context_lens, cu_seqlens, scale, window, sinks, out, return_lse):
    if scale is None:
        scale = q.size(-1) ** -0.5
    got = N.native().paged_attention(q, k_cache, v_cache, block_tables, context_lens, cu_seqlens, scale, window, sinks, out,
                                     bool(return_lse))
    if got is not None:
        N.check(got[0])
        return (got[1], got[2]) if return_lse else got[1]
    # what the compiled path leaves: a tensor on another device than the current one, or something to refuse
    N.require_cuda(q, k_cache, v_cache, block_tables, context_lens, cu_seqlens, out)
    if q.dim() != 3 or q.stride(2) != 1:
        raise ValueError("q must be [tokens, heads, head_dim] with adjacent elements in a head")
    T, heads, dim = q.shape
    cache = paged_cache(k_cache, v_cache, q.dtype, None, dim)
    if context_lens.dim() != 1 or not context_lens.is_contiguous():
        raise ValueError("context_lens must be a contiguous vector")
    n = context_lens.numel()
    _int32(context_lens, "context_lens", (n,))
    if block_tables.dim() != 2 or (block_tables.size(1) > 1 and block_tables.stride(1) != 1):
        raise ValueError("block_tables must be [requests, blocks] with adjacent entries in a row")
    _int32(block_tables, "block_tables", (n, block_tables.size(1)))
    if cu_seqlens is not None:
        _int32(cu_seqlens, "cu_seqlens", (n + 1,))
        if not cu_seqlens.is_contiguous():
            raise ValueError("cu_seqlens must be contiguous")
    elif n != T:
        raise ValueError(f"{T} tokens, {n} requests: a decode batch has one of each")
    if not (math.isfinite(scale) and scale > 0):
        raise ValueError("scale must be positive and finite")
    if not (0 <= window < 2 ** 31 and 0 <= sinks < 2 ** 31):
        raise ValueError("window and sinks must not be negative")
    if sinks and not window:
        raise ValueError("sinks are the first tokens outside a window: they need one")
    if out is not None and (out.shape != q.shape or out.dtype != q.dtype or out.stride(2) != 1):
        raise ValueError("out must have the shape and dtype of q, and adjacent elements in a head")
    devices = {t.device for t in (q, k_cache, v_cache, block_tables, context_lens, cu_seqlens, out) if t is not None}
    if len(devices) > 1:
        raise ValueError(f"tensors on several devices: {sorted(map(str, devices))}")
    with N.on_device(q.device):
        if out is None:
            out = torch.empty(T, heads, dim, dtype=q.dtype, device=q.device)
        lse = torch.empty(T, heads, dtype=torch.float32, device=q.device) if return_lse else None
        kv_heads = k_cache.size(2)
        shape = (heads, kv_heads, dim, block_tables.size(1), k_cache.size(1), window)
        need = N.lib().lora_b200_paged_decode_workspace_bytes(T, *shape, sinks) if cu_seqlens is None else \
            N.lib().lora_b200_paged_prefill_workspace_bytes(T, n, *shape)
        workspace = torch.empty(need, dtype=torch.uint8, device=q.device) if need else None
        head = (out.data_ptr(), out.stride(0), out.stride(1), N.ptr(lse), q.data_ptr(), q.stride(0), q.stride(1), T, heads, kv_heads, dim,
                ctypes.byref(cache), block_tables.data_ptr(), block_tables.stride(0), block_tables.size(1), context_lens.data_ptr())
        tail = (float(scale), int(window), int(sinks), N.dtype_code(q.dtype), N.ptr(workspace), need, N.current_stream(q.device))
        if cu_seqlens is None:
            N.check(N.lib().lora_b200_paged_decode_attention(*head, *tail))
        else:
            N.check(N.lib().lora_b200_paged_prefill_attention(*head, cu_seqlens.data_ptr(), n, *tail))
    return (out, lse) if return_lse else out


def paged_decode_attention(q: torch.Tensor, k_cache: torch.Tensor, v_cache: torch.Tensor, block_tables: torch.Tensor,
                           context_lens: torch.Tensor, *, scale: float | None = None, window: int = 0, sinks: int = 0,
                           out: torch.Tensor | None = None, return_lse: bool = False):
    """One new token of every request, its key and value in the cache already.

    ``q [requests, heads, head_dim]``; ``k_cache`` / ``v_cache`` ``[blocks, block_size, kv_heads, head_dim]``; ``block_tables``
    int32 ``[requests, blocks of a request]``; ``context_lens`` int32, the new token included. The token at position ``p =
    context_len - 1`` sees every key, or with ``window`` the last ``window`` of them (its own among them) and the first ``sinks``.
    Blocks without a key that it sees are not touched, and their table entries are not used. An entry outside the cache (-1)
    stands for no block, as does what is behind the table's end: such keys are left out. A request of no visible key gives zeros.
    q, out and caches may be strided (adjacent elements in a head, 16-byte aligned heads).

    Returns ``out`` (fresh, or the given one), with ``return_lse`` also the fp32 ``[requests, heads]`` logarithm of the sum of the
    exponentials (``-inf`` without a key), with which two parts of a context are joined."""
    return _paged_attention(q, k_cache, v_cache, block_tables, context_lens, None, scale, window, sinks, out, return_lse)


def paged_prefill_attention(q: torch.Tensor, k_cache: torch.Tensor, v_cache: torch.Tensor, block_tables: torch.Tensor,
                            context_lens: torch.Tensor, cu_seqlens: torch.Tensor, *, scale: float | None = None, window: int = 0,
                            sinks: int = 0, out: torch.Tensor | None = None, return_lse: bool = False):
    """Packed new tokens: rows ``cu_seqlens[i] : cu_seqlens[i + 1]`` of ``q [tokens, heads, head_dim]`` are the last tokens of
    request ``i``, whose ``context_lens[i]`` counts them (ascending; a range that leaves the rows of q counts as none); keys and values
    of all of them are in the cache already. Every token sees what ``paged_decode_attention`` would show it at its position. Rows of
    ``out`` (and of the log sums) of no sequence are not written: a given ``out`` keeps them. Other arguments as
    ``paged_decode_attention``. Block sizes that are multiples of 8 go to the tensor-core kernel, others (and tables of 2^31 keys) to the
    decode kernel, a token at a time. A value that is not finite, of a key that some tokens of a block of a few see, may reach the
    block's other tokens; what no token of the block sees (stale rows, returned blocks) never does."""
    if cu_seqlens is None:
        raise ValueError("cu_seqlens says which rows of q are whose: paged_prefill_attention needs it")
    return _paged_attention(q, k_cache, v_cache, block_tables, context_lens, cu_seqlens, scale, window, sinks, out, return_lse)
