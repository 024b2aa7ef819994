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
    assert lib.fa2_document_layout_bytes(3, 130) == 4 * 3 * (2 * 130 + 2 * 2 + 1)
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


def _plan_params():
    lib = _capi.load()
    a = _capi.PagedPlanParams()
    a.requests, a.table_width, a.table_stride, a.n_free, a.page_size, a.num_tokens, a.heads_q, a.heads_kv = 3, 5, 5, 4, 16, 100, 8, 2
    for name in ("context_lens", "new_lens", "block_table", "free_pages", "cu_seqlens", "seqlens_k", "slot_map", "positions", "pages_taken", "work"):
        setattr(a, name, 0x10000)
    a.work_bytes = lib.fa2_paged_work_bytes(3, 100, 8, 2)
    return a


@pytest.mark.parametrize("change,code,word", [
    (dict(requests=0), _capi.FA2_ERR_INVALID_ARG, b"positive"),
    (dict(requests=8193), _capi.FA2_ERR_UNSUPPORTED, b"8192"),
    (dict(num_tokens=-1), _capi.FA2_ERR_INVALID_ARG, b"negative"),
    (dict(page_size=24), _capi.FA2_ERR_UNSUPPORTED, b"power of two"),
    (dict(page_size=4), _capi.FA2_ERR_UNSUPPORTED, b"power of two"),
    (dict(page_size=2 ** 21), _capi.FA2_ERR_UNSUPPORTED, b"power of two"),
    (dict(heads_q=3), _capi.FA2_ERR_INVALID_ARG, b"divisible"),
    (dict(heads_q=129, heads_kv=1), _capi.FA2_ERR_UNSUPPORTED, b"128"),
    (dict(table_stride=4), _capi.FA2_ERR_INVALID_ARG, b"table_stride"),
    (dict(table_width=2 ** 27, table_stride=2 ** 27), _capi.FA2_ERR_UNSUPPORTED, b"2^30"),
    (dict(slot_map=None), _capi.FA2_ERR_INVALID_ARG, b"non-null"),
    (dict(free_pages=None), _capi.FA2_ERR_INVALID_ARG, b"non-null"),
    (dict(work=0x10008), _capi.FA2_ERR_INVALID_ARG, b"16-byte"),
    (dict(slot_map=0x10004), _capi.FA2_ERR_INVALID_ARG, b"8-byte"),
    (dict(context_lens=0x10002), _capi.FA2_ERR_INVALID_ARG, b"4-byte"),
    (dict(work_bytes=16), _capi.FA2_ERR_WORKSPACE, b"work"),
    (dict(num_tokens=2 ** 30, heads_q=128, heads_kv=1, table_width=2 ** 20, table_stride=2 ** 20, work_bytes=2 ** 40), _capi.FA2_ERR_UNSUPPORTED, b"too large"),
])
def test_plan_refusals(change, code, word):
    a = _plan_params()
    for name, x in change.items():
        setattr(a, name, x)
    lib = _capi.load()
    assert lib.fa2_paged_plan(C.byref(a), None) == code
    assert word in lib.fa2_last_error()


def test_paged_sizes():
    lib = _capi.load()
    sms = torch.cuda.get_device_properties(0).multi_processor_count if torch.cuda.is_available() else 148
    head = 16 + (4 * (sms + 1) + 7) // 8 * 8                                             # header and the CTAs' starts
    assert lib.fa2_paged_work_bytes(3, 100, 8, 2) == 4 * (head + 8 * (100 // 64 + 3))    # 64 tokens of 4 heads per item
    assert lib.fa2_paged_work_bytes(200, 100, 8, 8) == 4 * (head + 8 * 100)              # at most one item per token
    assert lib.fa2_paged_work_bytes(3, 100, 3, 2) == 0
    assert lib.fa2_paged_workspace_bytes(256) == 0 and lib.fa2_paged_workspace_bytes(20) == 0
    assert lib.fa2_paged_workspace_bytes(128) % (2 * 256 * 129 * 4) == 0


def _set_cache(c):
    c.ptr, c.stride_page, c.stride_slot, c.stride_head = 0x10000, 16 * 2 * 64, 2 * 64, 64


@pytest.mark.parametrize("change,code,word", [
    (dict(tokens=-1), _capi.FA2_ERR_INVALID_ARG, b"negative"),
    (dict(head_dim=20), _capi.FA2_ERR_UNSUPPORTED, b"multiple of 8"),
    (dict(page_size=12), _capi.FA2_ERR_UNSUPPORTED, b"power of two"),
    (dict(pages=0), _capi.FA2_ERR_INVALID_ARG, b"positive"),
    (dict(k=0x10008), _capi.FA2_ERR_UNSUPPORTED, b"16-byte"),
    (dict(v=None), _capi.FA2_ERR_INVALID_ARG, b"non-null"),
    (dict(k_stride_t=100), _capi.FA2_ERR_UNSUPPORTED, b"multiples of 8"),
    (dict(v_stride_h=-64), _capi.FA2_ERR_INVALID_ARG, b"negative"),
    (dict(slot_map=0x10004), _capi.FA2_ERR_INVALID_ARG, b"8-byte"),
])
def test_cache_write_refusals(change, code, word):
    a = _capi.PagedWriteParams()
    a.k = a.v = a.slot_map = 0x10000
    a.k_stride_t = a.v_stride_t = 128
    a.k_stride_h = a.v_stride_h = 64
    _set_cache(a.k_cache)
    _set_cache(a.v_cache)
    a.tokens, a.heads, a.head_dim, a.pages, a.page_size = 5, 2, 64, 7, 16
    for name, x in change.items():
        setattr(a, name, x)
    lib = _capi.load()
    assert lib.fa2_paged_cache_write(C.byref(a), None) == code
    assert word in lib.fa2_last_error()


@pytest.mark.parametrize("change,code,word", [
    (dict(head_dim=256), _capi.FA2_ERR_UNSUPPORTED, b"head_dim"),
    (dict(head_dim=72), _capi.FA2_ERR_UNSUPPORTED, b"head_dim"),
    (dict(dtype=_capi.FA2_FP32), _capi.FA2_ERR_UNSUPPORTED, b"fp16 and bf16"),
    (dict(heads_q=5), _capi.FA2_ERR_INVALID_ARG, b"divisible"),
    (dict(page_size=48), _capi.FA2_ERR_UNSUPPORTED, b"power of two"),
    (dict(softmax_scale=0.0), _capi.FA2_ERR_INVALID_ARG, b"softmax_scale"),
    (dict(softmax_scale=math.inf), _capi.FA2_ERR_INVALID_ARG, b"softmax_scale"),
    (dict(softcap=-1.0), _capi.FA2_ERR_INVALID_ARG, b"softcap"),
    (dict(q=None), _capi.FA2_ERR_INVALID_ARG, b"non-null"),
    (dict(o=0x10008), _capi.FA2_ERR_UNSUPPORTED, b"16-byte"),
    (dict(q_stride_t=4), _capi.FA2_ERR_UNSUPPORTED, b"multiples of 8"),
    (dict(o_stride_h=0), _capi.FA2_ERR_INVALID_ARG, b"positive"),
    (dict(table_stride=2), _capi.FA2_ERR_INVALID_ARG, b"table_stride"),
    (dict(work=0x10004), _capi.FA2_ERR_INVALID_ARG, b"16-byte"),
    (dict(requests=0), _capi.FA2_ERR_INVALID_ARG, b"positive"),
])
def test_paged_attention_refusals(change, code, word):
    a = _capi.PagedAttentionParams()
    for name in ("q", "o", "block_table", "work", "workspace"):
        setattr(a, name, 0x10000)
    a.q_stride_t = a.o_stride_t = 256
    a.q_stride_h = a.o_stride_h = 64
    _set_cache(a.k_cache)
    _set_cache(a.v_cache)
    a.tokens, a.heads_q, a.heads_kv, a.head_dim, a.dtype, a.pages, a.page_size = 5, 4, 2, 64, _capi.FA2_BF16, 7, 16
    a.table_width, a.table_stride, a.requests, a.softmax_scale = 3, 3, 2, 0.1
    for name, x in change.items():
        setattr(a, name, x)
    lib = _capi.load()
    assert lib.fa2_paged_attention(C.byref(a), None) == code
    assert word in lib.fa2_last_error()


def test_paged_python_layer_refuses_before_any_launch():
    ints = lambda *shape: torch.zeros(shape, dtype=torch.int32)
    with pytest.raises(RuntimeError, match="CUDA"):
        J.paged_step_plan(ints(2), ints(2), ints(2, 4), ints(3), page_size=16, num_tokens=2, heads_q=4, heads_kv=2)
    cache = torch.zeros(4, 16, 2, 64, dtype=torch.bfloat16)
    with pytest.raises(RuntimeError, match="CUDA"):
        J.paged_cache_write(cache[0], cache[0], cache, cache, torch.zeros(16, dtype=torch.int64))
    with pytest.raises(RuntimeError, match="CUDA"):
        J.paged_attention(cache[0], cache, cache, None)
    with pytest.raises(ValueError, match="power of two"):
        J._paged._check_pages(24)
    with pytest.raises(ValueError, match="same shape"):
        J._paged._check_caches(cache, cache[:2])
    with pytest.raises(ValueError, match="fp16 or bf16"):
        J._paged._check_caches(cache.float(), cache.float())


def test_a_layout_serves_the_shape_it_was_made_for_alone():
    # [1, 512] and [2, 256] take the same number of words: the shape tells them apart
    words = lambda b, s: J._capi.load().fa2_document_layout_bytes(b, s) // 4
    assert words(1, 512) == words(2, 256)
    short, long = torch.zeros(2, 256, 1, 64, dtype=torch.bfloat16), torch.zeros(1, 512, 1, 64, dtype=torch.bfloat16)
    layout = torch.zeros(1, words(1, 512), dtype=torch.int32)
    mods = J._scored_attention._score_mod
    mods(long, long, True, None, None, layout, None)
    for wrong in (layout.view(2, -1), layout.view(-1), layout[:, :-1]):
        with pytest.raises(ValueError, match="document_layout"):
            mods(long, long, True, None, None, wrong, None)
    with pytest.raises(ValueError, match="document_layout"):
        mods(short, short, True, None, None, layout, None)


def test_serving_calls_take_no_part_in_training():
    x = torch.zeros(2, requires_grad=True)
    with pytest.raises(RuntimeError, match="no backward"):
        J._paged._check_no_grad("paged_cache_write", torch.zeros(2), None, x)
    with torch.no_grad():
        J._paged._check_no_grad("paged_cache_write", x)
    y = torch.zeros(2)
    J._paged._written(y)
    assert y._version == 1
    with torch.inference_mode():
        J._paged._written(torch.zeros(2))


@pytest.mark.parametrize("shape,parts", [
    ((1, 512, 512, 32, 8, 128), 4), ((1, 1024, 1024, 32, 8, 64), 2), ((1, 512, 512, 12, 2, 64), 6), ((1, 512, 512, 20, 4, 256), 1),
    ((1, 512, 512, 24, 4, 256), 3), ((4, 4096, 4096, 32, 8, 128), 1), ((1, 128, 128, 8, 4, 64), 1), ((1, 256, 128, 8, 4, 64), 2),
    ((1, 64, 64, 8, 8, 64), 1),
])
def test_parts_of_the_query_heads(shape, parts):
    # 148 SMs are assumed where there is no device
    if torch.cuda.is_available() and torch.cuda.get_device_properties(0).multi_processor_count != 148:
        pytest.skip("written for 148 SMs")
    p = _capi.Problem()
    p.batch, p.seqlen_q, p.seqlen_k, p.heads_q, p.heads_kv, p.head_dim = shape
    p.heads_q_global, p.dtype, p.causal, p.softmax_scale = p.heads_q, _capi.FA2_BF16, 1, 0.1
    lib = _capi.load()
    more = lib.fa2_scored_bwd_workspace_bytes(C.byref(p)) - lib.fa2_bwd_workspace_bytes(C.byref(p))
    tiles = shape[0] * shape[4] * ((shape[2] + 127) // 128)
    assert more == (parts * 2 * tiles * 128 * shape[5] * 4 if parts > 1 else 0)
