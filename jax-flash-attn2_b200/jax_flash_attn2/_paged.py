"""Serving with a paged key/value cache: the plan of a step, the write of its new keys and values, and their attention.

A server keeps a pool of pages of `page_size` tokens per layer (`k_cache`, `v_cache`: [pages, page_size, Hkv, D]), one
block table for all layers, and a list of free pages. A step brings new tokens for some requests, one each for those
that decode and more for those whose prompt is read; they lie one behind the other in packed tensors. Per step:

    plan = paged_step_plan(context_lens, new_lens, block_table, free_pages, page_size=..., num_tokens=..., heads_q=..., heads_kv=...)
    for every layer:
        paged_cache_write(k, v, k_cache, v_cache, plan.slot_map)
        out = paged_attention(q, k_cache, v_cache, plan, softcap=..., alibi_slopes=...)

Nothing is copied to the host, so a step can be captured into a CUDA graph and replayed with other lengths in the same
tensors (give `num_tokens` room then: rows behind the last request are left alone). The reference has no such path.
"""
from __future__ import annotations

import math
import typing as tp
from dataclasses import dataclass

import torch

from . import _capi, _native
from ._kernel_calls import _DTYPE_CODE, _launch
from ._scored_attention import _check_slopes, _check_softcap


@dataclass(eq=False)
class PagedStepPlan:
    """What `paged_step_plan` computed, on the device. `block_table` is the caller's, updated in place."""

    cu_seqlens: torch.Tensor    # int32 [B + 1]: first row of every request in the packed tensors
    seqlens_k: torch.Tensor     # int32 [B]: tokens in the cache, the new ones included
    block_table: torch.Tensor   # int32 [B, width]
    slot_map: torch.Tensor      # int64 [T]: page * page_size + place in the page; -1: no slot
    positions: torch.Tensor     # int32 [T]: position of the token in its request; 0 behind the last request
    pages_taken: torch.Tensor   # int32 [1]: entries of the free list that the step needs
    work: torch.Tensor          # int32: work list of the attention
    page_size: int
    num_tokens: int
    heads_q: int
    heads_kv: int


def _check_int32(x: torch.Tensor, shape, name: str, device) -> torch.Tensor:
    if x.dtype != torch.int32 or tuple(x.shape) != tuple(shape):
        raise ValueError(f"{name} must be int32 of shape {list(shape)}, got {x.dtype} {tuple(x.shape)}")
    if x.device != device:
        raise ValueError(f"{name} must live on the device of block_table")
    return x.contiguous()


def _check_pages(page_size: int) -> int:
    page_size = int(page_size)
    if page_size < 8 or page_size > 1 << 20 or page_size & (page_size - 1):
        raise ValueError(f"page_size must be a power of two from 8 to 2^20, got {page_size}")
    return page_size


def paged_step_plan(
    context_lens: torch.Tensor,
    new_lens: torch.Tensor,
    block_table: torch.Tensor,
    free_pages: torch.Tensor,
    *,
    page_size: int,
    num_tokens: int,
    heads_q: int,
    heads_kv: int,
    free_start: tp.Optional[torch.Tensor] = None,
) -> PagedStepPlan:
    """Block table, slots and work list of a serving step, in one launch.

    context_lens, new_lens: int32 [B], tokens that a request has in the cache and brings (0 allowed). block_table: int32
    [B, width], whose first ceil(context / page_size) entries of a row are the request's pages; pages that the new tokens
    open are taken from `free_pages` (int32 [F]) in order, beginning at `free_start` (int32 [1] on the device, default 0),
    and entered into the table. `num_tokens`: rows of the packed tensors, at least the sum of new_lens (tokens beyond it are
    cut off). heads_q / heads_kv: of the attention that will use the plan. Calling it again with the same arguments gives
    the same plan: the lengths and the free list are the caller's to advance (`free_start += plan.pages_taken` on the
    device). Where the list runs out (pages_taken says how much was needed), table entries and slots are -1: such tokens
    are not written, and attention reads zeros in their place."""
    parts = _native.load().paged_step_plan(context_lens, new_lens, block_table, free_pages, page_size, num_tokens, heads_q,
                                           heads_kv, free_start)
    if parts is not None:
        cu_seqlens, seqlens_k, slot_map, positions, pages_taken, work = parts
        return PagedStepPlan(cu_seqlens, seqlens_k, block_table, slot_map, positions, pages_taken, work, page_size, num_tokens,
                             heads_q, heads_kv)
    # the call is to be refused, or some operand has to be copied first
    if not block_table.is_cuda:
        raise RuntimeError("fa2_b200 runs on CUDA tensors only; there is no CPU path")
    page_size, num_tokens = _check_pages(page_size), int(num_tokens)
    device = block_table.device
    if block_table.dim() != 2 or block_table.dtype != torch.int32 or 0 in block_table.shape:
        raise ValueError(f"block_table must be int32 of shape [requests, pages per request], got {block_table.dtype} {tuple(block_table.shape)}")
    requests, width = block_table.shape
    if block_table.stride(1) != 1 or (requests > 1 and block_table.stride(0) < width):
        raise ValueError("block_table is updated in place: its rows must be contiguous and must not overlap")
    if num_tokens < 0:
        raise ValueError("num_tokens must not be negative")
    context_lens = _check_int32(context_lens, (requests,), "context_lens", device)
    new_lens = _check_int32(new_lens, (requests,), "new_lens", device)
    if free_pages.dim() != 1:
        raise ValueError(f"free_pages must be one-dimensional, got shape {tuple(free_pages.shape)}")
    free_pages = _check_int32(free_pages, tuple(free_pages.shape), "free_pages", device)
    if free_start is not None:
        free_start = _check_int32(free_start.reshape(-1), (1,), "free_start", device)
    lib = _capi.load()
    heads_q, heads_kv = int(heads_q), int(heads_kv)
    with torch.cuda.device(device):
        nbytes = lib.fa2_paged_work_bytes(requests, num_tokens, heads_q, heads_kv)
    if nbytes == 0:
        _capi.check(_capi.FA2_ERR_INVALID_ARG)
    # one buffer for all int32 results: work list (16-byte aligned), row starts, lengths, positions, pages taken
    at = nbytes // 4
    sizes = (at, requests + 1, requests, num_tokens, 1)
    work, cu_seqlens, seqlens_k, positions, pages_taken = torch.empty((sum(sizes),), dtype=torch.int32, device=device).split(sizes)
    slot_map = torch.empty((num_tokens,), dtype=torch.int64, device=device)
    a = _capi.PagedPlanParams()
    a.context_lens, a.new_lens, a.requests = context_lens.data_ptr(), new_lens.data_ptr(), requests
    a.block_table, a.table_width = block_table.data_ptr(), width
    a.table_stride = block_table.stride(0) if requests > 1 else width
    a.free_pages, a.n_free = free_pages.data_ptr(), free_pages.shape[0]
    a.free_start = None if free_start is None else free_start.data_ptr()
    a.page_size, a.num_tokens, a.heads_q, a.heads_kv = page_size, num_tokens, heads_q, heads_kv
    a.cu_seqlens, a.seqlens_k, a.slot_map = cu_seqlens.data_ptr(), seqlens_k.data_ptr(), slot_map.data_ptr()
    a.positions, a.pages_taken = positions.data_ptr(), pages_taken.data_ptr()
    a.work, a.work_bytes = work.data_ptr(), nbytes
    _launch(lib.fa2_paged_plan, a, device)
    _written(block_table)
    return PagedStepPlan(cu_seqlens, seqlens_k, block_table, slot_map, positions, pages_taken, work, page_size, num_tokens,
                         heads_q, heads_kv)


def _written(x: torch.Tensor) -> None:
    """Tells autograd of a write in place, so that a backward pass that saved `x` notices."""
    if not x.is_inference():
        torch.autograd.graph.increment_version(x)


def _check_no_grad(name: str, *tensors) -> None:
    if torch.is_grad_enabled() and any(x is not None and x.requires_grad for x in tensors):
        raise RuntimeError(f"{name} has no backward pass: call it under torch.no_grad()")


def _cache(x: torch.Tensor, name: str) -> _capi.PagedCache:
    if x.dim() != 4 or 0 in x.shape:
        raise ValueError(f"{name} must be [pages, page_size, heads, head_dim], got shape {tuple(x.shape)}")
    if x.stride(3) != 1:
        raise ValueError(f"{name}: the stride of head_dim must be 1")
    return _capi.PagedCache(x.data_ptr(), x.stride(0), x.stride(1), x.stride(2))


def _check_caches(k_cache, v_cache):
    if k_cache.shape != v_cache.shape or k_cache.dtype != v_cache.dtype or k_cache.device != v_cache.device:
        raise ValueError("k_cache and v_cache must have the same shape, dtype and device")
    if k_cache.dtype not in (torch.float16, torch.bfloat16):
        raise ValueError(f"the cache must be fp16 or bf16, got {k_cache.dtype}")
    _check_pages(k_cache.shape[1] if k_cache.dim() == 4 else 0)


def paged_cache_write(k: torch.Tensor, v: torch.Tensor, k_cache: torch.Tensor, v_cache: torch.Tensor,
                      slot_map: torch.Tensor) -> None:
    """Writes row t of k and v ([T, Hkv, D], strided rows and heads allowed) to slot `slot_map[t]` (int64 [T]) of the
    caches [pages, page_size, Hkv, D]. Slots outside the cache (-1) are skipped; no slot may occur twice. No gradients:
    inference only."""
    if _native.load().paged_cache_write(k, v, k_cache, v_cache, slot_map):
        return
    # the call is to be refused, or some operand has to be copied first
    if not k_cache.is_cuda:
        raise RuntimeError("fa2_b200 runs on CUDA tensors only; there is no CPU path")
    _check_no_grad("paged_cache_write", k, v, k_cache, v_cache)
    _check_caches(k_cache, v_cache)
    a = _capi.PagedWriteParams()
    a.k_cache, a.v_cache = _cache(k_cache, "k_cache"), _cache(v_cache, "v_cache")
    pages, page_size, heads, d = k_cache.shape
    tokens = k.shape[0]
    if tuple(k.shape) != (tokens, heads, d) or k.shape != v.shape:
        raise ValueError(f"k and v must be [tokens, {heads}, {d}], got {tuple(k.shape)} and {tuple(v.shape)}")
    if k.dtype != k_cache.dtype or v.dtype != k_cache.dtype:
        raise ValueError("k and v must have the dtype of the cache")
    if slot_map.dtype != torch.int64 or tuple(slot_map.shape) != (tokens,):
        raise ValueError(f"slot_map must be int64 of shape [{tokens}], got {slot_map.dtype} {tuple(slot_map.shape)}")
    if not (k.device == v.device == slot_map.device == k_cache.device):
        raise ValueError("k, v and slot_map must live on the device of the cache")
    if k.stride(2) != 1:
        k = k.contiguous()
    if v.stride(2) != 1:
        v = v.contiguous()
    slot_map = slot_map.contiguous()
    a.k, a.k_stride_t, a.k_stride_h = k.data_ptr(), k.stride(0), k.stride(1)
    a.v, a.v_stride_t, a.v_stride_h = v.data_ptr(), v.stride(0), v.stride(1)
    a.slot_map = slot_map.data_ptr()
    a.tokens, a.heads, a.head_dim, a.pages, a.page_size = tokens, heads, d, pages, page_size
    _launch(_capi.load().fa2_paged_cache_write, a, k_cache.device)
    _written(k_cache)
    _written(v_cache)


def paged_attention(
    q: torch.Tensor,
    k_cache: torch.Tensor,
    v_cache: torch.Tensor,
    plan: PagedStepPlan,
    softmax_scale: tp.Optional[float] = None,
    *,
    softcap: tp.Optional[float] = None,
    alibi_slopes: tp.Optional[torch.Tensor] = None,
    out: tp.Optional[torch.Tensor] = None,
    lse: tp.Optional[torch.Tensor] = None,
) -> torch.Tensor:
    """Attention of the new tokens q [T, Hq, D] over the paged cache, which holds their own keys and values already: the
    token at position p of its request sees the keys 0 .. p. The scores may be capped and biased as in
    `scored_flash_attention`. fp16 or bf16, D up to 128, Hq / Hkv up to 128, page_size a power of two from 8.

    Returns `out` [T, Hq, D] (allocated if not given); rows behind the last request are left as they were. `lse`: float32
    [T, Hq] to be filled with the natural log-sum-exp of the scores. Memory in a request's last page behind its last key
    is ignored whatever it holds. No gradients: inference only."""
    if isinstance(plan, PagedStepPlan):
        done = _native.load().paged_attention(q, k_cache, v_cache, plan.block_table, plan.work, plan.num_tokens, plan.heads_q,
                                              plan.heads_kv, plan.page_size, softmax_scale, softcap, alibi_slopes, out, lse)
        if done is not None:
            return done
    # the call is to be refused, or some operand has to be copied first
    if not q.is_cuda:
        raise RuntimeError("fa2_b200 runs on CUDA tensors only; there is no CPU path")
    _check_no_grad("paged_attention", q, k_cache, v_cache, out, lse)
    _check_caches(k_cache, v_cache)
    a = _capi.PagedAttentionParams()
    a.k_cache, a.v_cache = _cache(k_cache, "k_cache"), _cache(v_cache, "v_cache")
    pages, page_size, heads_kv, d = k_cache.shape
    if q.dim() != 3 or q.shape[2] != d or q.dtype != k_cache.dtype:
        raise ValueError(f"q must be [tokens, heads, {d}] in {k_cache.dtype}, got {tuple(q.shape)} in {q.dtype}")
    tokens, heads_q = q.shape[:2]
    if (tokens, heads_q, heads_kv, page_size) != (plan.num_tokens, plan.heads_q, plan.heads_kv, plan.page_size):
        raise ValueError(f"the plan is for {plan.num_tokens} tokens, {plan.heads_q} / {plan.heads_kv} heads and pages of "
                         f"{plan.page_size}, got {tokens} tokens, {heads_q} / {heads_kv} heads and pages of {page_size}")
    table = plan.block_table
    if not (q.device == k_cache.device == plan.work.device == table.device):
        raise ValueError("q, the caches and the plan must live on one device")
    if plan.work.dtype != torch.int32 or table.dtype != torch.int32 or table.dim() != 2 or 0 in table.shape or table.stride(1) != 1:
        raise ValueError("the plan must be what paged_step_plan returned")
    if q.stride(2) != 1:
        q = q.contiguous()
    if out is None:
        out = torch.empty((tokens, heads_q, d), dtype=q.dtype, device=q.device)
    elif tuple(out.shape) != tuple(q.shape) or out.dtype != q.dtype or out.device != q.device or out.stride(2) != 1:
        raise ValueError("out must have the shape, dtype and device of q and a head_dim stride of 1")
    if lse is not None:
        if lse.dtype != torch.float32 or tuple(lse.shape) != (tokens, heads_q) or lse.device != q.device or not lse.is_contiguous():
            raise ValueError(f"lse must be contiguous float32 of shape [{tokens}, {heads_q}] on the device of q")
        a.lse = lse.data_ptr()
    slopes = _check_slopes(alibi_slopes, heads_q, q.device)
    lib = _capi.load()
    a.q, a.q_stride_t, a.q_stride_h = q.data_ptr(), q.stride(0), q.stride(1)
    a.o, a.o_stride_t, a.o_stride_h = out.data_ptr(), out.stride(0), out.stride(1)
    a.tokens, a.heads_q, a.heads_kv, a.head_dim, a.dtype = tokens, heads_q, heads_kv, d, _DTYPE_CODE[q.dtype]
    a.pages, a.page_size = pages, page_size
    a.block_table, a.table_width, a.requests = table.data_ptr(), table.shape[1], table.shape[0]
    a.table_stride = table.stride(0) if table.shape[0] > 1 else table.shape[1]
    a.work = plan.work.data_ptr()
    a.softmax_scale = 1.0 / math.sqrt(d) if softmax_scale is None else float(softmax_scale)
    a.softcap = _check_softcap(softcap)
    if slopes is not None:
        a.alibi_slopes = slopes.data_ptr()
    with torch.cuda.device(q.device):
        nbytes = lib.fa2_paged_workspace_bytes(d)
    workspace = torch.empty((max(nbytes, 128),), dtype=torch.uint8, device=q.device)
    a.workspace, a.workspace_bytes = workspace.data_ptr(), nbytes
    _launch(lib.fa2_paged_attention, a, q.device)
    _written(out)
    if lse is not None:
        _written(lse)
    return out
