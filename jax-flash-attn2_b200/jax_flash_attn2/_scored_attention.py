"""Attention with changed scores: a tanh cap, a bias that falls with the distance, document and prefix masks.

    s_ij = softmax_scale * q_i . k_j
    s_ij <- softcap * tanh(s_ij / softcap)                    (softcap given)
    s_ij <- s_ij - alibi_slopes[h] * |i + Sk - Sq - j|        (alibi_slopes given)

and query i of batch element b sees key j iff all that is given holds:

    causal:        j <= i + Sk - Sq, or j < prefix_lens[b]
    document_ids:  i and j lie in the same document. A document is a run of equal ids in a row; tokens with a
                   negative id are padding: they see nothing and nothing sees them.

Queries that see nothing give zeros and take no gradient. q, k and v get gradients; the slopes are constants. All
values of q, k, v and of the cotangent must be finite, in padding and masked places too (a masked weight is an exact
zero, and zero times infinity is not a number). The reference has none of these score changes on its GPU path; the
two kernel calls stand beside `fwd_attention_kernel_call` and `bwd_attention_kernel_call` and share their kernels.
"""
from __future__ import annotations

import ctypes as C
import os
import typing as tp

import torch

from . import _capi, _native
from ._kernel_calls import _check_qkv, _launch, _problem, _strides, _unit_last


def _check_softcap(softcap) -> float:
    softcap = 0.0 if softcap is None else float(softcap)
    if softcap != 0.0 and not 2.0 ** -10 <= softcap <= 1024.0:
        raise ValueError(f"softcap must be None, 0 or in [2^-10, 1024], got {softcap}")
    return softcap


def _check_slopes(slopes: tp.Optional[torch.Tensor], heads: int, device: torch.device) -> tp.Optional[torch.Tensor]:
    if slopes is None:
        return None
    if slopes.dtype != torch.float32 or tuple(slopes.shape) != (heads,):
        raise ValueError(f"alibi_slopes must be float32 of shape [{heads}], got {slopes.dtype} {tuple(slopes.shape)}")
    if slopes.device != device:
        raise ValueError("alibi_slopes must live on the device of q")
    if slopes.requires_grad:
        raise ValueError("alibi_slopes are constants: they take no gradient")
    return slopes.contiguous()


def document_layout(document_ids: torch.Tensor) -> torch.Tensor:
    """The layout of packed documents that the kernel calls take, from int32 ids [B, S] on the GPU: for every token
    the bounds of its document and the same over every 128 tokens. It depends on the ids alone, so one layout serves
    the forward and backward of every layer."""
    if document_ids.dim() != 2 or document_ids.dtype != torch.int32:
        raise ValueError(f"document_ids must be int32 of shape [batch, seqlen], got {document_ids.dtype} {tuple(document_ids.shape)}")
    if not document_ids.is_cuda:
        raise RuntimeError("fa2_b200 runs on CUDA tensors only; there is no CPU path")
    if document_ids.stride(1) != 1 or document_ids.stride(0) < 0:
        document_ids = document_ids.contiguous()
    lib = _capi.load()
    batch, seqlen = document_ids.shape
    nbytes = lib.fa2_document_layout_bytes(batch, seqlen)
    if nbytes == 0:
        raise ValueError("document_ids must not be empty")
    # (the shape tells the layout of one batch and length from that of another)
    layout = torch.empty((batch, nbytes // 4 // batch), dtype=torch.int32, device=document_ids.device)
    index = document_ids.device.index
    with torch.cuda.device(index):
        stream = torch.cuda.current_stream(index).cuda_stream
        _capi.check(lib.fa2_document_layout(document_ids.data_ptr(), document_ids.stride(0), batch, seqlen,
                                            layout.data_ptr(), nbytes, C.c_void_p(stream)))
    return layout


def _check_devices(q, k, v):
    if not (q.device == k.device == v.device):
        raise ValueError(f"q, k and v must live on one device, got {q.device}, {k.device} and {v.device}")


def _score_mod(q, k, causal, softcap, alibi_slopes, layout, prefix_lens, rest=None):
    """(parameter block, tensors kept alive)."""
    mod = _capi.ScoreMod()
    batch, sq, heads = q.shape[:3]
    mod.softcap = _check_softcap(softcap)
    slopes = _check_slopes(alibi_slopes, heads, q.device)
    if slopes is not None:
        mod.alibi_slopes = slopes.data_ptr()
    if prefix_lens is not None:
        if not causal:
            raise ValueError("prefix_lens needs causal=True")
        if prefix_lens.dtype != torch.int32 or tuple(prefix_lens.shape) != (batch,):
            raise ValueError(f"prefix_lens must be int32 of shape [{batch}], got {prefix_lens.dtype} {tuple(prefix_lens.shape)}")
        if prefix_lens.device != q.device:
            raise ValueError("prefix_lens must live on the device of q")
        prefix_lens = prefix_lens.contiguous()
        mod.prefix_lens = prefix_lens.data_ptr()
    if layout is not None:
        if k.shape[1] != sq:
            raise ValueError("documents need as many keys as queries")
        words = _capi.load().fa2_document_layout_bytes(batch, sq) // 4 // batch
        if layout.dtype != torch.int32 or tuple(layout.shape) != (batch, words) or not layout.is_contiguous() or layout.device != q.device:
            raise ValueError("layout must be what document_layout returned for ids of shape "
                             f"[{batch}, {sq}] on the device of q")
        mod.document_layout = layout.data_ptr()
    if rest is not None:
        if rest.shape != q.shape or rest.dtype != q.dtype or rest.device != q.device or not rest.is_contiguous():
            raise ValueError("rest must be a contiguous tensor of the shape, dtype and device of q")
        mod.o_rest, mod.o_rest_strides = rest.data_ptr(), _strides(rest)
    return mod, (slopes, prefix_lens, layout)


def fwd_scored_attention_kernel_call(
    q: torch.Tensor,
    k: torch.Tensor,
    v: torch.Tensor,
    softmax_scale: tp.Optional[float] = None,
    causal: bool = False,
    *,
    softcap: tp.Optional[float] = None,
    alibi_slopes: tp.Optional[torch.Tensor] = None,
    layout: tp.Optional[torch.Tensor] = None,
    prefix_lens: tp.Optional[torch.Tensor] = None,
    rest: tp.Optional[torch.Tensor] = None,
) -> tp.Tuple[torch.Tensor, torch.Tensor]:
    """Forward launch; q [B,Sq,Hq,D], k and v [B,Sk,Hkv,D], `layout` from `document_layout`. `rest` (a contiguous tensor
    like q) receives what the rounding of the output dropped, for the backward call. Returns (out in q.dtype,
    lse float32 [B,Hq,ceil(Sq/128)*128] of the changed scores, natural log; columns >= Sq are not written)."""
    _check_qkv(q, k, v)
    _check_devices(q, k, v)
    lib = _capi.load()
    q, k, v = _unit_last(q), _unit_last(k), _unit_last(v)
    batch, sq, hq, d = q.shape
    mod, _keep = _score_mod(q, k, causal, softcap, alibi_slopes, layout, prefix_lens, rest)
    out = torch.empty((batch, sq, hq, d), dtype=q.dtype, device=q.device)
    lse = torch.empty((batch, hq, (sq + 127) // 128 * 128), dtype=torch.float32, device=q.device)
    a = _capi.FwdParams()
    a.p = _problem(q, k, softmax_scale, 0.0, causal, None, 0, 0, None)
    a.q, a.q_strides = q.data_ptr(), _strides(q)
    a.k, a.k_strides = k.data_ptr(), _strides(k)
    a.v, a.v_strides = v.data_ptr(), _strides(v)
    a.o, a.o_strides = out.data_ptr(), _strides(out)
    a.lse, a.lse_stride_b, a.lse_stride_h = lse.data_ptr(), lse.stride(0), lse.stride(1)
    nbytes = lib.fa2_fwd_workspace_bytes(C.byref(a.p))
    if nbytes:
        _keep_w = torch.empty((nbytes,), dtype=torch.uint8, device=q.device)
        a.workspace, a.workspace_bytes = _keep_w.data_ptr(), nbytes
    _launch(lib.fa2_scored_fwd, a, q.device, mod)
    return out, lse


def bwd_scored_attention_kernel_call(
    dO: torch.Tensor,
    q: torch.Tensor,
    k: torch.Tensor,
    v: torch.Tensor,
    o: torch.Tensor,
    M: torch.Tensor,
    softmax_scale: tp.Optional[float] = None,
    causal: bool = False,
    *,
    softcap: tp.Optional[float] = None,
    alibi_slopes: tp.Optional[torch.Tensor] = None,
    layout: tp.Optional[torch.Tensor] = None,
    prefix_lens: tp.Optional[torch.Tensor] = None,
    rest: tp.Optional[torch.Tensor] = None,
    deterministic: tp.Optional[bool] = None,
) -> tp.Tuple[torch.Tensor, torch.Tensor, torch.Tensor]:
    """Backward launch; `o`, `M` and `rest` (if it was given) are the forward's output, lse and rest. Returns (dq, dk, dv) in the input dtype. dk and dv
    are the same bits from call to call; dq is so with `deterministic=True` (default None: the environment variable
    FA2_B200_DETERMINISTIC decides, as in `bwd_attention_kernel_call`)."""
    _check_qkv(q, k, v)
    _check_devices(q, k, v)
    lib = _capi.load()
    if deterministic is None:
        deterministic = os.environ.get("FA2_B200_DETERMINISTIC", "0") not in ("", "0")
    q, k, v, o = map(_unit_last, (q, k, v, o))
    if dO.stride(-1) != 1 or dO.data_ptr() % 16 or any(s <= 0 or s % 8 for s in dO.stride()[:3]):
        dO = dO.clone(memory_format=torch.contiguous_format)      # a cotangent may be expanded or transposed
    assert tuple(dO.shape) == tuple(q.shape) and tuple(o.shape) == tuple(q.shape)
    assert dO.dtype == q.dtype and o.dtype == q.dtype
    mod, _keep = _score_mod(q, k, causal, softcap, alibi_slopes, layout, prefix_lens, rest)
    dq = torch.empty_like(q, memory_format=torch.contiguous_format)
    dk = torch.empty_like(k, memory_format=torch.contiguous_format)
    dv = torch.empty_like(v, memory_format=torch.contiguous_format)
    a = _capi.BwdParams()
    a.p = _problem(q, k, softmax_scale, 0.0, causal, None, 0, 0, None)
    with torch.cuda.device(q.device):
        nbytes = lib.fa2_scored_bwd_workspace_bytes(C.byref(a.p))
    if nbytes == 0:
        _capi.check(_capi.FA2_ERR_INVALID_ARG)
    workspace = torch.empty((nbytes,), dtype=torch.uint8, device=q.device)
    a.q, a.q_strides = q.data_ptr(), _strides(q)
    a.k, a.k_strides = k.data_ptr(), _strides(k)
    a.v, a.v_strides = v.data_ptr(), _strides(v)
    a.o, a.o_strides = o.data_ptr(), _strides(o)
    a.d_o, a.do_strides = dO.data_ptr(), _strides(dO)
    a.lse, a.lse_stride_b, a.lse_stride_h = M.data_ptr(), M.stride(0), M.stride(1)
    a.dq, a.dq_strides = dq.data_ptr(), _strides(dq)
    a.dk, a.dk_strides = dk.data_ptr(), _strides(dk)
    a.dv, a.dv_strides = dv.data_ptr(), _strides(dv)
    a.workspace, a.workspace_bytes = workspace.data_ptr(), nbytes
    a.deterministic = int(bool(deterministic))
    _launch(lib.fa2_scored_bwd, a, q.device, mod)
    return dq, dk, dv


class _ScoredAttentionCall(torch.autograd.Function):
    @staticmethod
    def forward(ctx, q, k, v, softmax_scale, causal, mods):
        # bf16: the rounding of the output is the largest error of the gradients where single keys dominate (dq of scores
        # with a standard deviation of 4 over 100 keys, in float64: 4.6e-3 with it, 3.1e-3 without); what it drops is kept
        rest = None
        if q.dtype == torch.bfloat16 and any(ctx.needs_input_grad):
            rest = torch.empty(q.shape, dtype=q.dtype, device=q.device)
        out, lse = fwd_scored_attention_kernel_call(q, k, v, softmax_scale, causal, rest=rest, **mods)
        ctx.save_for_backward(q, k, v, out, lse, mods["alibi_slopes"], mods["layout"], mods["prefix_lens"], rest)
        ctx.extras = (softmax_scale, causal, mods["softcap"])
        return out

    @staticmethod
    def backward(ctx, dO):
        if torch.is_grad_enabled():
            raise RuntimeError("scored_flash_attention has no second derivatives (create_graph=True)")
        q, k, v, out, lse, slopes, layout, prefix_lens, rest = ctx.saved_tensors
        softmax_scale, causal, softcap = ctx.extras
        dq, dk, dv = bwd_scored_attention_kernel_call(
            dO, q, k, v, out, lse, softmax_scale, causal, softcap=softcap, alibi_slopes=slopes, layout=layout,
            prefix_lens=prefix_lens, rest=rest)
        return dq, dk, dv, None, None, None


def scored_flash_attention(
    q: torch.Tensor,
    k: torch.Tensor,
    v: torch.Tensor,
    softmax_scale: tp.Optional[float] = None,
    causal: bool = False,
    *,
    softcap: tp.Optional[float] = None,
    alibi_slopes: tp.Optional[torch.Tensor] = None,
    document_ids: tp.Optional[torch.Tensor] = None,
    prefix_lens: tp.Optional[torch.Tensor] = None,
    layout: tp.Optional[torch.Tensor] = None,
) -> torch.Tensor:
    """Differentiable attention with changed scores (see the module's text for the formulas).

    q [B,Sq,Hq,D]; k, v [B,Sk,Hkv,D] with Hq a multiple of Hkv; fp16 or bf16; the head dims and strides of
    `triton_flash_attention`. softmax_scale (default 1/sqrt(D)) must be positive; softcap lies in [2^-10, 1024];
    alibi_slopes float32 [Hq]; document_ids int32 [B, S] with Sq == Sk == S (or their `layout`, so that several layers
    share it); prefix_lens int32 [B], with causal=True. All on the device of q. Returns [B,Sq,Hq,D] in q.dtype.

    The backward pass may be captured into a CUDA graph unless the graph of an earlier call on another stream still lives and
    ends in the same leaf tensors: autograd would synchronise with that stream, so the call is refused under capture."""
    out = _native.load().scored_flash_attention(q, k, v, softmax_scale, causal, softcap, alibi_slopes, document_ids,
                                                prefix_lens, layout)
    if out is not None:
        return out
    # the call is to be refused, or some operand has to be copied first
    _check_qkv(q, k, v)
    _check_devices(q, k, v)
    if document_ids is not None:
        if layout is not None:
            raise ValueError("give document_ids or their layout, not both")
        if tuple(document_ids.shape) != (q.shape[0], q.shape[1]) or k.shape[1] != q.shape[1]:
            raise ValueError(f"document_ids must be [{q.shape[0]}, {q.shape[1]}] with as many keys as queries, got "
                             f"{tuple(document_ids.shape)} for {k.shape[1]} keys")
        if document_ids.device != q.device:
            raise ValueError("document_ids must live on the device of q")
        layout = document_layout(document_ids)
    mods = dict(softcap=softcap, alibi_slopes=_check_slopes(alibi_slopes, q.shape[2], q.device), layout=layout,
                prefix_lens=prefix_lens)
    if torch.is_grad_enabled():
        _native.load().check_capture(q, k, v)
    return _ScoredAttentionCall.apply(q, k, v, softmax_scale, bool(causal), mods)
