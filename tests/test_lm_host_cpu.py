"""CPU tests of the operators for language models: exported symbols, refusals that come before any launch, and the
oracle the GPU tests use."""
import ctypes as C
import math
import os
import re

import pytest
import torch

import jax_flash_attn2 as J
from jax_flash_attn2 import _capi
from oracle import dense, scored

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))


def test_library_exports_what_the_header_declares():
    header = open(os.path.join(ROOT, "include", "fa2_b200_lm.h")).read()
    declared = set(re.findall(r"\b(fa2_[a-z_0-9]+)\s*\(", header))
    lib = _capi.load()
    assert set(_capi.LM_EXPORTED_SYMBOLS) == declared
    for name in declared:
        assert hasattr(lib, name), name
    assert lib.fa2_lm_version() == _capi.FA2_LM_ABI_VERSION
    assert f"#define FA2_LM_ABI_VERSION {_capi.FA2_LM_ABI_VERSION}" in header


def _fwd_params(Sq=128, Sk=128):
    """Parameters whose pointers are never followed: validation stops first."""
    a = _capi.FwdParams()
    a.p.batch, a.p.seqlen_q, a.p.seqlen_k = 2, Sq, Sk
    a.p.heads_q, a.p.heads_kv, a.p.head_dim = 4, 2, 128
    a.p.dtype, a.p.softmax_scale, a.p.heads_q_global = _capi.FA2_BF16, 0.1, 4
    for name in ("q", "k", "v", "o", "lse"):
        setattr(a, name, 0x10000)
    a.lse_stride_h, a.lse_stride_b = Sq, 4 * Sq
    return a


def _refused(a, mod, code, word):
    lib = _capi.load()
    assert lib.fa2_scored_fwd(C.byref(a), C.byref(mod), None) == code
    assert word in lib.fa2_last_error()
    b = _capi.BwdParams()
    b.p = a.p
    for name in ("q", "k", "v", "o", "d_o", "lse", "dq", "dk", "dv"):
        setattr(b, name, 0x10000)
    b.lse_stride_h, b.lse_stride_b = a.lse_stride_h, a.lse_stride_b
    b.workspace, b.workspace_bytes = 0x20000, lib.fa2_bwd_workspace_bytes(C.byref(b.p))
    b.bias, b.mask, b.seqlens = a.bias, a.mask, a.seqlens
    assert lib.fa2_scored_bwd(C.byref(b), C.byref(mod), None) == code
    assert word in lib.fa2_last_error()


@pytest.mark.parametrize("cap", [-1.0, 2.0 ** -11, 1025.0, math.inf, math.nan])
def test_caps_outside_their_range_are_refused(cap):
    mod = _capi.ScoreMod()
    mod.softcap = cap
    _refused(_fwd_params(), mod, _capi.FA2_ERR_INVALID_ARG, b"softcap")
    with pytest.raises(ValueError, match="softcap"):
        J._scored_attention._check_softcap(cap)


def test_combinations_that_are_not_offered_are_refused():
    mod = _capi.ScoreMod()
    a = _fwd_params()
    a.p.softmax_scale = 0.0
    _refused(a, mod, _capi.FA2_ERR_INVALID_ARG, b"softmax_scale")
    a = _fwd_params()
    a.p.dropout_p = 0.5
    _refused(a, mod, _capi.FA2_ERR_UNSUPPORTED, b"dropout")
    a = _fwd_params()
    a.bias.ptr = 0x30000
    _refused(a, mod, _capi.FA2_ERR_UNSUPPORTED, b"bias")
    a = _fwd_params()
    a.seqlens = 0x30000
    _refused(a, mod, _capi.FA2_ERR_UNSUPPORTED, b"seqlens")
    mod.prefix_lens = 0x30000
    _refused(_fwd_params(), mod, _capi.FA2_ERR_INVALID_ARG, b"causal")
    mod = _capi.ScoreMod()
    mod.document_layout = 0x30000
    _refused(_fwd_params(Sk=256), mod, _capi.FA2_ERR_INVALID_ARG, b"seqlen_q == seqlen_k")
    mod = _capi.ScoreMod()
    mod.alibi_slopes = 0x30002
    _refused(_fwd_params(), mod, _capi.FA2_ERR_INVALID_ARG, b"aligned")
    lib = _capi.load()
    assert lib.fa2_scored_fwd(C.byref(_fwd_params()), None, None) == _capi.FA2_ERR_INVALID_ARG


def test_document_layout_arguments():
    lib = _capi.load()
    assert lib.fa2_document_layout_bytes(3, 130) == 4 * 3 * (2 * 130 + 2 * 2)
    assert lib.fa2_document_layout_bytes(0, 130) == 0
    need = lib.fa2_document_layout_bytes(3, 130)
    call = lambda ids=0x1000, stride=130, b=3, s=130, out=0x2000, n=need: lib.fa2_document_layout(ids, stride, b, s, out, n, None)
    for kw in (dict(ids=None), dict(out=None), dict(b=0), dict(s=0), dict(stride=-1), dict(ids=0x1002), dict(out=0x2008), dict(n=need - 1)):
        assert call(**kw) == _capi.FA2_ERR_INVALID_ARG
    assert call(s=2 ** 31 - 1) == _capi.FA2_ERR_UNSUPPORTED


def test_python_layer_refuses_before_any_launch():
    q = torch.zeros(2, 8, 4, 64, dtype=torch.bfloat16)
    with pytest.raises(RuntimeError, match="CUDA"):
        J.scored_flash_attention(q, q, q)
    with pytest.raises(ValueError, match="int32"):
        J.document_layout(torch.zeros(2, 8))
    with pytest.raises(RuntimeError, match="CUDA"):
        J.document_layout(torch.zeros(2, 8, dtype=torch.int32))
    with pytest.raises(ValueError, match="alibi_slopes"):
        J._scored_attention._check_slopes(torch.zeros(3), 4, torch.device("cpu"))
    with pytest.raises(ValueError, match="no gradient"):
        J._scored_attention._check_slopes(torch.zeros(4, requires_grad=True), 4, torch.device("cpu"))
    mods = J._scored_attention._score_mod
    with pytest.raises(ValueError, match="causal"):
        mods(q, q, False, None, None, None, torch.zeros(2, dtype=torch.int32))
    with pytest.raises(ValueError, match="prefix_lens"):
        mods(q, q, True, None, None, None, torch.zeros(3, dtype=torch.int32))
    with pytest.raises(ValueError, match="as many keys"):
        mods(q, q[:, :4], True, None, None, torch.zeros(4, dtype=torch.int32), None)
    with pytest.raises(ValueError, match="document_layout"):
        mods(q, q, True, None, None, torch.zeros(4, dtype=torch.int32), None)


def test_scored_oracle_agrees_with_the_dense_one_and_with_automatic_differentiation():
    g = torch.Generator().manual_seed(1)
    q, k, v, do = (torch.randn(2, s, h, 16, generator=g, dtype=torch.float64) for s, h in ((9, 4), (13, 2), (13, 2), (9, 4)))
    seen = scored.visible_keys(2, 9, 13, True)
    r = scored.attention(q, k, v, seen, dO=do)
    want, lse = dense.attention(q, k, v, causal=True)
    torch.testing.assert_close(r["out"], want)
    torch.testing.assert_close(r["lse"], lse)
    for name, x in zip(("dq", "dk", "dv"), dense.attention_grads(do, q, k, v, causal=True)):
        torch.testing.assert_close(r[name], x)
    slopes, seen = torch.rand(4, generator=g, dtype=torch.float64), scored.visible_keys(2, 9, 13, True, None, [5, 0])
    leaves = [x.clone().requires_grad_(True) for x in (q, k, v)]
    out = scored.attention(*leaves, seen, softcap=2.0, alibi_slopes=slopes)["out"]
    auto = torch.autograd.grad(out, leaves, do)
    r = scored.attention(q, k, v, seen, softcap=2.0, alibi_slopes=slopes, dO=do)
    for name, x in zip(("dq", "dk", "dv"), auto):
        torch.testing.assert_close(r[name], x)
