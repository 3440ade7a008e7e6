"""Attention over the paged key-value cache that ``glue.rope_kv_store`` and ``glue.qk_norm_rope_kv_store`` fill: the next token
of every request (``paged_decode_attention``) or packed runs of new tokens (``paged_prefill_attention``: whole prompts, chunks of
them, a few tokens behind a long context). Causal, over everything or over a sliding window of the last keys plus a few first
ones. Stands where the reference attends over its paged cache
(``nanovllm_voxcpm/layers/attention.py:70-79``). Besides: both for requests that begin alike, whose common keys are read once
(``shared_prefix_decode_attention``, ``shared_prefix_prefill_attention``); the difference of two softmax maps (``differential_decode_attention``,
``differential_prefill_attention``), and what joins results over parts of a context (``join_attention``). The kernels are
``csrc/paged_attention.cuh``, ``csrc/paged_prefill.cuh`` and ``csrc/attention_join.cuh`` behind ``lora_b200_paged_*``,
``lora_b200_shared_prefix_attention``, ``lora_b200_differential_attention`` and ``lora_b200_join_attention``.
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


def _checked(q, k_cache, v_cache, block_tables, context_lens, cu_seqlens, scale, window, sinks, out, *others) -> N.PagedCache:
    """The checks that the compiled path leaves to be named: it takes tensors on the current device and gives back the rest."""
    N.require_cuda(q, k_cache, v_cache, block_tables, context_lens, cu_seqlens, out, *others)
    if q.dim() != 3 or q.stride(2) != 1:
        raise ValueError("q must be [tokens, heads, head_dim] with adjacent elements in a head")
    T = q.size(0)
    cache = paged_cache(k_cache, v_cache, q.dtype, None, q.size(2))
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
    devices = {t.device for t in (q, k_cache, v_cache, block_tables, context_lens, cu_seqlens, out, *others) if t is not None}
    if len(devices) > 1:
        raise ValueError(f"tensors on several devices: {sorted(map(str, devices))}")
    return cache


def _paged_attention(q, k_cache, v_cache, block_tables, context_lens, cu_seqlens, scale, window, sinks, out, return_lse):
    if scale is None:
        scale = q.size(-1) ** -0.5
    got = N.native().paged_attention(q, k_cache, v_cache, block_tables, context_lens, cu_seqlens, scale, window, sinks, out,
                                     bool(return_lse))
    if got is not None:
        N.check(got[0])
        return (got[1], got[2]) if return_lse else got[1]
    # what the compiled path leaves: a tensor on another device than the current one, or something to refuse
    cache = _checked(q, k_cache, v_cache, block_tables, context_lens, cu_seqlens, scale, window, sinks, out)
    T, heads, dim = q.shape
    n = context_lens.numel()
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


def _shared_prefix(q, k_cache, v_cache, block_tables, context_lens, cu_seqlens, prefix_lens, cu_groups, scale, out, return_lse):
    if prefix_lens is None or cu_groups is None:
        raise ValueError("prefix_lens and cu_groups say who begins alike: an attention behind shared prefixes needs both")
    if scale is None:
        scale = q.size(-1) ** -0.5
    got = N.native().shared_prefix_attention(q, k_cache, v_cache, block_tables, context_lens, cu_seqlens, prefix_lens, cu_groups, scale,
                                             out, bool(return_lse))
    if got is not None:
        N.check(got[0])
        return (got[1], got[2]) if return_lse else got[1]
    cache = _checked(q, k_cache, v_cache, block_tables, context_lens, cu_seqlens, scale, 0, 0, out, prefix_lens, cu_groups)
    if prefix_lens.dim() != 1 or not prefix_lens.is_contiguous() or not cu_groups.is_contiguous():
        raise ValueError("prefix_lens and cu_groups must be contiguous vectors")
    groups = prefix_lens.numel()
    _int32(prefix_lens, "prefix_lens", (groups,))
    _int32(cu_groups, "cu_groups", (groups + 1,))
    T, heads, dim = q.shape
    with N.on_device(q.device):
        if out is None:
            out = torch.empty(T, heads, dim, dtype=q.dtype, device=q.device)
        lse = torch.empty(T, heads, dtype=torch.float32, device=q.device) if return_lse else None
        n, kv_heads, width, page = context_lens.numel(), k_cache.size(2), block_tables.size(1), k_cache.size(1)
        need = N.lib().lora_b200_shared_prefix_workspace_bytes(T, n, groups, heads, kv_heads, dim, width, page, cu_seqlens is not None)
        workspace = torch.empty(need, dtype=torch.uint8, device=q.device) if need else None
        N.check(N.lib().lora_b200_shared_prefix_attention(
            out.data_ptr(), out.stride(0), out.stride(1), N.ptr(lse), q.data_ptr(), q.stride(0), q.stride(1), T, heads, kv_heads, dim,
            ctypes.byref(cache), block_tables.data_ptr(), block_tables.stride(0), width, context_lens.data_ptr(), N.ptr(cu_seqlens), n,
            prefix_lens.data_ptr(), cu_groups.data_ptr(), groups, float(scale), N.dtype_code(q.dtype), N.ptr(workspace), need,
            N.current_stream(q.device)))
    return (out, lse) if return_lse else out


def shared_prefix_decode_attention(q: torch.Tensor, k_cache: torch.Tensor, v_cache: torch.Tensor, block_tables: torch.Tensor,
                                   context_lens: torch.Tensor, prefix_lens: torch.Tensor, cu_groups: torch.Tensor, *,
                                   scale: float | None = None, out: torch.Tensor | None = None, return_lse: bool = False):
    """``paged_decode_attention`` (without a window) of requests that begin alike: the keys that the requests of a group have in common
    are read once for all of them. Same result, but for the order of its sums.

    Requests ``cu_groups[g] : cu_groups[g + 1]`` have the same keys and values at their first ``prefix_lens[g]`` positions (any number:
    a prefix may end inside a block, of which every request has a copy of its own). Where those lie is read from the table of the group's
    first request, which holds them all, what follows from each one's own. ``prefix_lens`` int32 ``[groups]``, ``cu_groups`` int32 ``[groups + 1]``, ascending;
    requests of no group share nothing, a prefix of zero is none. Other arguments, strides, missing blocks, contexts of no key and the
    log sums as ``paged_decode_attention``. Calls whose tables are too narrow for a second launch to pay, whose block size is no multiple
    of 8 or that have no more requests than groups are attended request by request; in the others a group of one goes with the rest. The
    lengths are on the device, so that the tables' width decides: where most keys lie behind the prefixes, or groups have one to three
    requests, ``paged_decode_attention`` is the faster call. A value that is not finite, of a key of the prefix that some requests of a group see,
    may reach the group's others."""
    return _shared_prefix(q, k_cache, v_cache, block_tables, context_lens, None, prefix_lens, cu_groups, scale, out, return_lse)


def shared_prefix_prefill_attention(q: torch.Tensor, k_cache: torch.Tensor, v_cache: torch.Tensor, block_tables: torch.Tensor,
                                    context_lens: torch.Tensor, cu_seqlens: torch.Tensor, prefix_lens: torch.Tensor,
                                    cu_groups: torch.Tensor, *, scale: float | None = None, out: torch.Tensor | None = None,
                                    return_lse: bool = False):
    """``paged_prefill_attention`` (without a window) of requests that begin alike, grouped as in ``shared_prefix_decode_attention``;
    tokens inside a prefix see it up to themselves. Rows of no sequence are not written."""
    if cu_seqlens is None:
        raise ValueError("cu_seqlens says which rows of q are whose: shared_prefix_prefill_attention needs it")
    return _shared_prefix(q, k_cache, v_cache, block_tables, context_lens, cu_seqlens, prefix_lens, cu_groups, scale, out, return_lse)


def _differential(q, k_cache, v_cache, block_tables, context_lens, cu_seqlens, lam, norm_weight, eps, scale, window, sinks, out):
    if lam is None:
        raise ValueError("lam says what the second map counts: differential attention needs it")
    if scale is None:
        scale = (q.size(-1) // 2) ** -0.5
    got = N.native().differential_attention(q, k_cache, v_cache, block_tables, context_lens, cu_seqlens, lam, norm_weight, eps, scale,
                                            window, sinks, out)
    if got is not None:
        N.check(got[0])
        return got[1]
    cache = _checked(q, k_cache, v_cache, block_tables, context_lens, cu_seqlens, scale, window, sinks, out, lam, norm_weight)
    T, heads, dim = q.shape
    if lam.dtype != torch.float32 or tuple(lam.shape) not in ((heads,), (T, heads)):
        raise ValueError(f"lam must be a float32 tensor [heads] or [tokens, heads], got {lam.dtype} {tuple(lam.shape)}")
    if norm_weight is not None:
        if norm_weight.dtype != q.dtype or tuple(norm_weight.shape) != (dim,) or not norm_weight.is_contiguous():
            raise ValueError("norm_weight must be a contiguous [head_dim] vector of the dtype of q")
        if not (math.isfinite(eps) and eps > 0):
            raise ValueError("eps must be positive and finite")
    with N.on_device(q.device):
        if out is None:
            out = torch.empty(T, heads, dim, dtype=q.dtype, device=q.device)
        n, kv_heads, width, page = context_lens.numel(), k_cache.size(2), block_tables.size(1), k_cache.size(1)
        need = N.lib().lora_b200_differential_workspace_bytes(T, n, heads, kv_heads, dim, width, page, window, sinks, cu_seqlens is not None)
        workspace = torch.empty(need, dtype=torch.uint8, device=q.device) if need else None
        N.check(N.lib().lora_b200_differential_attention(
            out.data_ptr(), out.stride(0), out.stride(1), q.data_ptr(), q.stride(0), q.stride(1), T, heads, kv_heads, dim, ctypes.byref(cache),
            block_tables.data_ptr(), block_tables.stride(0), width, context_lens.data_ptr(), N.ptr(cu_seqlens), n, lam.data_ptr(),
            lam.stride(0) if lam.dim() == 2 else 0, lam.stride(-1), N.ptr(norm_weight), float(eps), float(scale), int(window), int(sinks),
            N.dtype_code(q.dtype), N.ptr(workspace), need, N.current_stream(q.device)))
    return out


def differential_decode_attention(q: torch.Tensor, k_cache: torch.Tensor, v_cache: torch.Tensor, block_tables: torch.Tensor,
                                  context_lens: torch.Tensor, lam: torch.Tensor, *, norm_weight: torch.Tensor | None = None,
                                  eps: float = 1e-5, scale: float | None = None, window: int = 0, sinks: int = 0,
                                  out: torch.Tensor | None = None):
    """Differential attention (Ye et al., "Differential Transformer", 2024) of one new token of every request. The halves of a head's
    columns of q and k make two softmax maps over the keys that ``paged_decode_attention`` would show the token; with ``S1`` and ``S2``
    their results over the whole columns of v, a head gives ``S1 - lam * S2``. With ``norm_weight [head_dim]`` that difference is
    RMS-normed over the head and scaled by it (a constant factor, ``1 - lambda_init``, belongs into it). All of it fp32, rounded once; a
    probability enters the product with v as the sum of two numbers of its type (off by 2^-15 of it at most in bf16, by 2^-23 in fp16).

    ``lam`` float32 ``[heads]`` or, of every token its own, ``[requests, heads]``; ``scale`` defaults to that of half a head. The halves
    are rotated as heads of their own: ``rope_kv_store`` fills such a cache as one of twice the heads of half the size. Other
    arguments, strides, missing blocks and contexts of no key as ``paged_decode_attention``."""
    return _differential(q, k_cache, v_cache, block_tables, context_lens, None, lam, norm_weight, eps, scale, window, sinks, out)


def differential_prefill_attention(q: torch.Tensor, k_cache: torch.Tensor, v_cache: torch.Tensor, block_tables: torch.Tensor,
                                   context_lens: torch.Tensor, cu_seqlens: torch.Tensor, lam: torch.Tensor, *,
                                   norm_weight: torch.Tensor | None = None, eps: float = 1e-5, scale: float | None = None,
                                   window: int = 0, sinks: int = 0, out: torch.Tensor | None = None):
    """``differential_decode_attention`` of packed new tokens, packed as ``paged_prefill_attention``'s (rows of no sequence are not
    written); ``lam`` float32 ``[heads]`` or ``[tokens, heads]``."""
    if cu_seqlens is None:
        raise ValueError("cu_seqlens says which rows of q are whose: differential_prefill_attention needs it")
    return _differential(q, k_cache, v_cache, block_tables, context_lens, cu_seqlens, lam, norm_weight, eps, scale, window, sinks, out)


def _steps(t: torch.Tensor) -> tuple:
    """The strides that matter: a dimension of one entry has none."""
    return tuple(s if n > 1 else 0 for n, s in zip(t.shape, t.stride()))


def join_attention(outs, lses, *, out: torch.Tensor | None = None, return_lse: bool = False):
    """The result over a whole context of results over its parts (each token's keys lie in one part each).

    ``outs`` ``[parts, tokens, heads, head_dim]`` or a sequence of ``[tokens, heads, head_dim]`` tensors of one shape and one set of
    strides (of dimensions with more than one entry), bf16, fp16 or fp32, up to 64 of them; ``lses`` the fp32 ``[tokens, heads]``
    logarithms of their sums that came with them (``return_lse``), as ``[parts, ...]`` or a sequence. A part without a key (``-inf``)
    counts for nothing, whatever its values; a row
    that has none in any part gives zeros. ``out`` may be one of the parts. Returns ``out``, with ``return_lse`` also the logarithm of
    the whole sum."""
    got = N.native().join_attention(outs, lses, out, bool(return_lse))
    if got is not None:
        N.check(got[0])
        return (got[1], got[2]) if return_lse else got[1]
    outs, lses = tuple(outs), tuple(lses)
    N.require_cuda(*outs, *lses, out)
    if not outs or len(outs) != len(lses):
        raise ValueError(f"{len(outs)} results and {len(lses)} logarithms: a part has one of each")
    first, lse0 = outs[0], lses[0]
    if first.dim() != 3 or first.stride(2) != 1:
        raise ValueError("a part must be [tokens, heads, head_dim] with adjacent elements in a head")
    if any(o.shape != first.shape or o.dtype != first.dtype or _steps(o) != _steps(first) for o in outs):
        raise ValueError("the parts must have one shape, dtype and set of strides")
    T, heads, dim = first.shape
    if any(x.dtype != torch.float32 or tuple(x.shape) != (T, heads) or _steps(x) != _steps(lse0) for x in lses):
        raise ValueError(f"the logarithms must be float32 tensors {(T, heads)} of one set of strides")
    if out is not None and (out.shape != first.shape or out.dtype != first.dtype or out.stride(2) != 1):
        raise ValueError("out must have the shape and dtype of a part, and adjacent elements in a head")
    devices = {t.device for t in (*outs, *lses, out) if t is not None}
    if len(devices) > 1:
        raise ValueError(f"tensors on several devices: {sorted(map(str, devices))}")
    with N.on_device(first.device):
        if out is None:
            out = torch.empty(T, heads, dim, dtype=first.dtype, device=first.device)
        lse = torch.empty(T, heads, dtype=torch.float32, device=first.device) if return_lse else None
        N.check(N.lib().lora_b200_join_attention(
            out.data_ptr(), *_steps(out)[:2], N.ptr(lse), N.ptr_array(outs), N.ptr_array(lses), len(outs), *_steps(first)[:2], *_steps(lse0),
            T, heads, dim, N.dtype_code(first.dtype), N.current_stream(first.device)))
    return (out, lse) if return_lse else out
