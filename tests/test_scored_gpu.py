"""GPU tests of attention with changed scores (tanh cap, distance bias, document and prefix masks): forward, gradients,
refusals, streams, graphs, bit-reproducibility, against float64 with bounds that add up the 16-bit roundings."""
import pytest
import torch

import workloads as W
from oracle import scored as O

pytestmark = pytest.mark.gpu

BF16, FP16 = torch.bfloat16, torch.float16


def slopes_of(heads):
    return torch.tensor([2.0 ** (-8.0 * (i + 1) / heads) for i in range(heads)])


def ids_of(rows, seqlen):
    """rows: per batch row a list of (id, length); what is left of a row is padding (-1)."""
    ids = torch.full((len(rows), seqlen), -1, dtype=torch.int32)
    for b, row in enumerate(rows):
        at = 0
        for i, n in row:
            ids[b, at:at + n] = i
            at += n
        assert at <= seqlen
    return ids


def check(B, Sq, Sk, Hq, Hkv, D, dtype, causal, *, sharp=1.0, scale=None, cap=None, slopes=None, ids=None, prefix=None,
          transposed=False, train=True):
    import jax_flash_attn2 as J
    q, k, v, do = W.make_qkv(B, Sq, Sk, Hq, Hkv, D, dtype)
    q = (q.float() * sharp).to(dtype)
    seen = O.visible_keys(B, Sq, Sk, causal, ids, prefix)
    want = O.attention(q, k, v, seen, scale, cap, slopes, do if train else None)
    bound = O.bounds(want, dtype)

    def dev(x):
        if transposed:      # stored [B, H, S, D]
            return x.cuda().permute(0, 2, 1, 3).contiguous().permute(0, 2, 1, 3)
        return x.cuda()

    leaves = [dev(x).requires_grad_(train) for x in (q, k, v)]
    out = J.scored_flash_attention(*leaves, scale, causal, softcap=cap, alibi_slopes=None if slopes is None else slopes.cuda(),
                                   document_ids=None if ids is None else ids.cuda(),
                                   prefix_lens=None if prefix is None else torch.tensor(prefix, dtype=torch.int32, device="cuda"))
    got = dict(out=out.detach())
    if train:
        got["dq"], got["dk"], got["dv"] = torch.autograd.grad(out, leaves, dev(do))
    assert J.device_status() == 0
    for name, x in got.items():
        assert x.dtype == dtype
        assert O.worst(x, want[name], bound[name]) <= 1.0, name
    dead = ~seen.any(-1)                                    # [B, Sq]
    assert torch.all(out.detach().cpu()[dead] == 0)
    if train:
        assert torch.all(got["dq"].cpu()[dead] == 0)
        unseen = ~seen.any(1)
        assert torch.all(got["dk"].cpu()[unseen] == 0) and torch.all(got["dv"].cpu()[unseen] == 0)


@pytest.mark.parametrize("dtype", [BF16, FP16])
@pytest.mark.parametrize("D", [64, 128, 256, 40, 96])
@pytest.mark.parametrize("cap,slopes", [(None, False), (20.0, False), (None, True), (20.0, True)])
def test_every_kernel_with_documents(D, dtype, cap, slopes):
    ids = ids_of([[(0, 100), (1, 28), (2, 1), (3, 130)], [(5, 300)]], 300)
    check(2, 300, 300, 4, 2, D, dtype, True, sharp=3.0, cap=cap, slopes=slopes_of(4) if slopes else None, ids=ids)


@pytest.mark.parametrize("Sq,Sk", [(1, 1), (1, 300), (3, 2), (129, 129), (200, 456), (300, 130), (520, 520)])
@pytest.mark.parametrize("causal", [True, False])
@pytest.mark.parametrize("D", [64, 128])
def test_lengths(Sq, Sk, causal, D):
    check(2, Sq, Sk, 4, 1, D, BF16, causal, sharp=4.0, cap=30.0, slopes=slopes_of(4))


@pytest.mark.parametrize("Sq,Sk,D", [(300, 130, 256), (1, 1, 256), (65, 257, 256)])
def test_lengths_head_dim_256(Sq, Sk, D):
    check(1, Sq, Sk, 3, 3, D, FP16, True, sharp=4.0, cap=30.0, slopes=slopes_of(3))


@pytest.mark.parametrize("rows", [
    [[(0, 1)] * 130 + [(1, 1)] * 130],                      # equal ids run on: two documents of 130 tokens
    [[(0, 1), (1, 1)] * 130],                               # every token its own document
    [[(-1, 70), (4, 60), (-1, 130), (4, 100)]],             # padding in front, between and behind; an id used twice
    [[(-1, 360)]],                                          # nothing but padding
    [[(7, 360)]],
    [[(0, 128), (1, 128), (2, 104)]],                       # documents that end with the tiles
    [[(0, 127), (1, 2), (2, 126), (3, 105)]],               # and next to their ends
    [[(3, 10)], [(-5, 300), (0, 60)], [(9, 200), (8, 160)]],
])
@pytest.mark.parametrize("causal", [True, False])
@pytest.mark.parametrize("D", [64, 128, 256])
def test_documents(rows, causal, D):
    check(len(rows), 360, 360, 2, 1, D, BF16, causal, sharp=2.0, ids=ids_of(rows, 360))


@pytest.mark.parametrize("prefix", [[0, 1], [128, 200], [10 ** 6, -3], [129, 383]])
@pytest.mark.parametrize("D", [64, 128, 256])
@pytest.mark.parametrize("Sk", [383, 250])
def test_prefix(prefix, D, Sk):
    check(2, 383, Sk, 4, 2, D, FP16, True, sharp=2.0, prefix=prefix)


def test_prefix_inside_documents():
    ids = ids_of([[(0, 150), (1, 150)], [(2, 290), (-1, 10)]], 300)
    check(2, 300, 300, 4, 2, 128, BF16, True, sharp=2.0, prefix=[200, 140], ids=ids, cap=15.0)


@pytest.mark.parametrize("Hq,Hkv", [(1, 1), (6, 2), (7, 1), (8, 8)])
def test_head_groups(Hq, Hkv):
    check(2, 257, 257, Hq, Hkv, 64, FP16, True, sharp=2.0, cap=50.0, slopes=slopes_of(Hq))


@pytest.mark.parametrize("D", [64, 128, 256])
def test_storage_with_heads_before_rows(D):
    check(2, 200, 200, 4, 2, D, BF16, True, sharp=2.0, cap=10.0, slopes=slopes_of(4), transposed=True)


def test_zeros_under_a_tiny_cap_and_a_large_scale():
    # scores of exactly 0 where scale / cap is beyond what the polynomial's coefficients can hold
    import jax_flash_attn2 as J
    k, v = (x.cuda() for x in W.make_qkv(1, 64, 64, 1, 1, 64, BF16)[1:3])
    for scale in (1e6, 1e30):
        out = J.scored_flash_attention(torch.zeros_like(k), k, v, scale, False, softcap=2.0 ** -10)
        want = v.float().mean(1, keepdim=True).expand_as(v)
        assert torch.all((out.float() - want).abs() <= 2.0 ** -8 * (v.float().abs().mean(1, keepdim=True) + want.abs()) + 1e-4)


def test_blocks_of_rows_are_taken_longest_first():
    import jax_flash_attn2 as J
    B, S = 3, 2100
    ids = ids_of([[(0, 2100)], [(0, 300), (1, 1000), (2, 500)], [(i, 100) for i in range(20)]], S)
    order = J.document_layout(ids.cuda()).view(-1)[-B * 9:].tolist()
    assert sorted(order) == list(range(B * 9))
    seen = O.visible_keys(B, S, S, True, ids)

    def length(i):
        rows = seen[i // 9, i % 9 * 256:i % 9 * 256 + 256].any(0).nonzero().flatten()
        return 0 if not len(rows) else rows[-1].item() // 128 - rows[0].item() // 128 + 1

    lengths = [length(i) for i in order]
    assert lengths == sorted(lengths, reverse=True)


@pytest.mark.parametrize("cap", [2.0 ** -10, 0.5, 1024.0])
def test_caps_at_the_ends_of_their_range(cap):
    # at 1024 the exponent's error is 2 * 1024 * log2(e) * 2^-23 = 3.5e-4, inside the slack of the bounds
    check(1, 200, 200, 2, 2, 64, BF16, True, sharp=8.0, cap=cap)


def test_steep_and_negative_slopes():
    check(1, 400, 400, 3, 1, 128, BF16, True, slopes=torch.tensor([8.0, 0.0, -0.01]))


def test_explicit_scale_and_forward_alone():
    check(2, 150, 270, 4, 4, 96, BF16, True, scale=0.3, cap=25.0, train=False)


@pytest.mark.parametrize("B,Sk,D,Hq,Hkv", [(1, 5000, 128, 8, 2), (1, 3500, 256, 2, 2), (1, 4100, 64, 4, 4)])
def test_few_rows_over_many_keys_are_split(B, Sk, D, Hq, Hkv):
    check(B, 3, Sk, Hq, Hkv, D, BF16, True, sharp=3.0, cap=30.0, slopes=slopes_of(Hq), train=False)


def test_many_items_per_sm():
    # more (query block, head) items than SMs, documents of uneven lengths
    ids = ids_of([[(0, 37), (1, 500), (2, 163)], [(0, 650)], [(1, 5), (2, 5), (3, 680)]], 700)
    check(3, 700, 700, 32, 8, 64, BF16, True, sharp=2.0, ids=ids)


def test_gradients_agree_with_differences():
    """(f(x + h e) - f(x - h e)) / 2h of the float64 definition, f = sum(out * dO), against the kernel's gradients along
    e. The kernel may be off by the sum of its bounds times |e|; the difference quotient by its third derivative."""
    import jax_flash_attn2 as J
    B, S, Hq, Hkv, D, dtype, cap = 1, 96, 2, 1, 64, FP16, 5.0
    q, k, v, do = W.make_qkv(B, S, S, Hq, Hkv, D, dtype)
    ids = ids_of([[(0, 40), (1, 50)]], S)
    slopes, seen = slopes_of(Hq), O.visible_keys(B, S, S, True, ids)
    leaves = [x.cuda().requires_grad_(True) for x in (q, k, v)]
    out = J.scored_flash_attention(*leaves, None, True, softcap=cap, alibi_slopes=slopes.cuda(), document_ids=ids.cuda())
    grads = torch.autograd.grad(out, leaves, do.cuda())
    want = O.attention(q, k, v, seen, None, cap, slopes, do)
    bound = O.bounds(want, dtype)
    g = torch.Generator().manual_seed(9)
    for i, name in enumerate(("dq", "dk", "dv")):
        e = torch.randn((q, k, v)[i].shape, generator=g, dtype=torch.float64)
        h = 1e-4

        def f(t):
            x = [y.double() for y in (q, k, v)]
            x[i] = x[i] + t * e
            return (O.attention(*x, seen, None, cap, slopes)["out"] * do.double()).sum().item()

        slope = (f(h) - f(-h)) / (2 * h)
        mine = (grads[i].double().cpu() * e).sum().item()
        assert abs(mine - slope) <= (bound[name] * e.abs()).sum().item() + 1e-5 * abs(slope), name


@pytest.mark.parametrize("D", [64, 128, 256])
@pytest.mark.parametrize("docs", [True, False])
def test_deterministic_gradients_are_the_same_bits(D, docs):
    import jax_flash_attn2 as J
    B, S, Hq, Hkv = 2, 900, 4, 2
    q, k, v, do = (x.cuda() for x in W.make_qkv(B, S, S, Hq, Hkv, D, BF16))
    ids = ids_of([[(0, 300), (1, 17), (-1, 200), (2, 383)], [(0, 850)]], S).cuda()
    kw = dict(softcap=20.0, layout=J.document_layout(ids) if docs else None,
              prefix_lens=torch.tensor([200, 500], dtype=torch.int32, device="cuda"))
    out, lse = J.fwd_scored_attention_kernel_call(q, k, v, None, True, **kw)
    first = J.bwd_scored_attention_kernel_call(do, q, k, v, out, lse, None, True, deterministic=True, **kw)
    for _ in range(3):
        again = J.bwd_scored_attention_kernel_call(do, q, k, v, out, lse, None, True, deterministic=True, **kw)
        assert all(torch.equal(a, b) for a, b in zip(first, again))
    loose = J.bwd_scored_attention_kernel_call(do, q, k, v, out, lse, None, True, deterministic=False, **kw)
    assert torch.equal(loose[1], first[1]) and torch.equal(loose[2], first[2])
    assert J.device_status() == 0


def test_layout_is_shared_by_layers_and_rows_may_be_strided():
    import jax_flash_attn2 as J
    q, k, v, _ = (x.cuda() for x in W.make_qkv(2, 5000, 5000, 2, 1, 64, BF16))
    wide = torch.zeros(2, 6000, dtype=torch.int32)
    wide[:, :5000] = ids_of([[(0, 2), (1, 4200), (2, 700)], [(-1, 4096), (0, 904)]], 5000)
    ids = wide.cuda()[:, :5000]
    layout = J.document_layout(ids)
    a = J.scored_flash_attention(q, k, v, None, True, layout=layout)
    b = J.scored_flash_attention(q, k, v, None, True, document_ids=ids.contiguous())
    assert torch.equal(a, b)
    lo, hi = layout.view(-1)[:20000].view(2, 2, 5000).cpu()
    assert lo[0, 0] == 0 and hi[0, 1] == 2 and torch.all(lo[0, 2:4202] == 2) and torch.all(hi[0, 2:4202] == 4202)
    assert torch.all(hi[0, 4902:] == 0) and torch.all(lo[1, 4096:] == 4096) and torch.all(hi[1, 4096:] == 5000) and torch.all(hi[1, :4096] == 0)


def test_forward_and_backward_in_a_captured_graph():
    import jax_flash_attn2 as J
    q, k, v, do = (x.cuda() for x in W.make_qkv(1, 260, 260, 4, 2, 128, BF16))
    ids = ids_of([[(0, 200), (1, 60)]], 260).cuda()
    leaves = [x.requires_grad_(True) for x in (q, k, v)]

    def step():
        out = J.scored_flash_attention(*leaves, None, True, softcap=30.0, document_ids=ids)
        return (out,) + torch.autograd.grad(out, leaves, do)

    eager = step()
    torch.cuda.synchronize()
    # the eager graph still lives and ends in the same leaves: capturing a backward now would break the capture
    refused = torch.cuda.CUDAGraph()
    with pytest.raises(RuntimeError, match="drop its outputs"):
        with torch.cuda.graph(refused):
            step()
    del refused
    eager = tuple(x.detach() for x in eager)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step()
    torch.cuda.current_stream().wait_stream(side)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        captured = step()
    for _ in range(2):
        graph.replay()
    torch.cuda.synchronize()
    assert torch.equal(captured[0], eager[0]) and torch.equal(captured[2], eager[2]) and torch.equal(captured[3], eager[3])
    # other documents, same graph
    ids.copy_(ids_of([[(0, 20), (1, 240)]], 260))
    graph.replay()
    again = step()
    torch.cuda.synchronize()
    assert torch.equal(captured[0], again[0]) and not torch.equal(again[0], eager[0])


def test_a_side_stream():
    import jax_flash_attn2 as J
    q, k, v, _ = (x.cuda() for x in W.make_qkv(2, 512, 512, 4, 2, 64, FP16))
    want = J.scored_flash_attention(q, k, v, None, True, softcap=30.0)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        got = J.scored_flash_attention(q, k, v, None, True, softcap=30.0)
    side.synchronize()
    assert torch.equal(got, want)


def test_without_changes_it_is_the_plain_attention():
    """Same scores, same masks: only the order of float32 operations may differ, so the results agree to the 16-bit
    rounding of P and of the output (two half steps each way)."""
    import jax_flash_attn2 as J
    q, k, v, _ = (x.cuda() for x in W.make_qkv(2, 700, 700, 4, 2, 128, BF16))
    a = J.scored_flash_attention(q, k, v, None, True).float()
    b = J.triton_flash_attention(q, k, v, causal=True).float()
    weight = J.triton_flash_attention(q, k, v.abs(), causal=True).float()
    assert torch.all((a - b).abs() <= 2 * 2.0 ** -8 * (weight + b.abs()))


@pytest.mark.parametrize("D", [64, 256])
def test_cotangents_of_any_layout(D):
    """An expanded cotangent (strides of zero), a transposed one and a misaligned one give the dense one's gradients."""
    import jax_flash_attn2 as J
    q, k, v, do = (x.cuda() for x in W.make_qkv(2, 130, 130, 4, 2, D, BF16))
    leaves = [x.requires_grad_(True) for x in (q, k, v)]
    out = J.scored_flash_attention(*leaves, None, True, softcap=20.0)
    grads = lambda c: torch.autograd.grad(out, leaves, c, retain_graph=True)
    one = torch.full_like(do, 0.5)
    for got, want in ((grads(one[:1, :1, :1, :1].expand_as(one)), grads(one)),
                      (grads(do.permute(0, 2, 3, 1).contiguous().permute(0, 3, 1, 2)), grads(do)),
                      (grads(torch.cat([do.flatten()[:1], do.flatten()])[1:].view_as(do)), grads(do))):
        assert torch.equal(got[1], want[1]) and torch.equal(got[2], want[2])
    with pytest.raises(RuntimeError, match="second derivatives"):
        torch.autograd.grad(out, leaves, do, create_graph=True)


def test_some_operands_without_gradients_and_operands_to_be_copied():
    import jax_flash_attn2 as J
    q, k, v, do = (x.cuda() for x in W.make_qkv(1, 100, 100, 2, 2, 64, BF16))
    full = [x.clone().requires_grad_(True) for x in (q, k, v)]
    want = torch.autograd.grad(J.scored_flash_attention(*full, None, True, softcap=20.0), full, do)
    k2 = k.clone().requires_grad_(True)
    got = torch.autograd.grad(J.scored_flash_attention(q, k2, v, None, True, softcap=20.0), k2, do)
    assert torch.equal(got[0], want[1])
    # columns that do not lie next to each other are copied before the launch
    odd = [x.transpose(2, 3).contiguous().transpose(2, 3).requires_grad_(True) for x in (q, k, v)]
    assert odd[0].stride(3) != 1
    out = J.scored_flash_attention(*odd, None, True, softcap=20.0)
    again = torch.autograd.grad(out, odd, do)
    assert torch.equal(again[1], want[1]) and torch.equal(again[2], want[2])
    with torch.no_grad():
        assert torch.equal(J.scored_flash_attention(*full, None, True, softcap=20.0), out)
    with pytest.raises(J._capi.Fa2Error, match="head_dim"):
        J.scored_flash_attention(*(torch.zeros(1, 8, 2, 72, dtype=BF16, device="cuda") for _ in range(3)))
    with pytest.raises(ValueError, match="softcap"):
        J.scored_flash_attention(q, k, v, softcap=-1.0)
    with pytest.raises(AssertionError, match="fp16 and bf16"):
        J.scored_flash_attention(q.float(), k.float(), v.float())


@pytest.mark.parametrize("B,Sq,Sk,Hq,Hkv,D,dtype,docs", [
    (1, 300, 300, 8, 2, 64, BF16, False), (1, 300, 300, 8, 1, 128, FP16, True), (2, 200, 330, 6, 2, 256, BF16, False),
    (1, 515, 515, 12, 2, 96, BF16, True), (1, 129, 1, 8, 1, 40, FP16, False), (3, 257, 257, 4, 2, 160, FP16, True),
])
def test_query_heads_in_parts_and_in_one(B, Sq, Sk, Hq, Hkv, D, dtype, docs, monkeypatch):
    """The backward deals the query heads to several SMs where there are few key tiles (more scratch): against the formulas
    with and without, dq the same bits."""
    import ctypes as C
    import jax_flash_attn2 as J
    from jax_flash_attn2 import _capi, _kernel_calls
    lib = _capi.load()
    q, k, v, do = W.make_qkv(B, Sq, Sk, Hq, Hkv, D, dtype)
    ids = ids_of([[(0, Sq // 3), (1, Sq // 2)]] * B, Sq) if docs else None
    want = O.attention(q, k, v, O.visible_keys(B, Sq, Sk, True, ids), None, 20.0, slopes_of(Hq), do)
    bound = O.bounds(want, dtype)
    dq, dk, dv, ddo = (x.cuda() for x in (q, k, v, do))
    problem = _kernel_calls._problem(dq, dk, None, 0.0, True, None, 0, 0, None)
    assert lib.fa2_scored_bwd_workspace_bytes(C.byref(problem)) > lib.fa2_bwd_workspace_bytes(C.byref(problem))
    rest = torch.empty_like(dq)
    kw = dict(softcap=20.0, alibi_slopes=slopes_of(Hq).cuda(), layout=J.document_layout(ids.cuda()) if docs else None, rest=rest)
    out, lse = J.fwd_scored_attention_kernel_call(dq, dk, dv, None, True, **kw)
    run = lambda: J.bwd_scored_attention_kernel_call(ddo, dq, dk, dv, out, lse, None, True, deterministic=True, **kw)
    parts, again = run(), run()
    assert all(torch.equal(x, y) for x, y in zip(parts, again))
    monkeypatch.setattr(lib, "fa2_scored_bwd_workspace_bytes", lib.fa2_bwd_workspace_bytes)
    one = run()
    assert torch.equal(one[0], parts[0])
    for grads in (parts, one):
        for name, x in zip(("dq", "dk", "dv"), grads):
            assert O.worst(x, want[name], bound[name]) <= 1.0, name
    assert J.device_status() == 0


def test_tensors_of_more_than_2_31_elements():
    """Packed documents of 128 tokens: the last ones are the same problem as a short call."""
    import jax_flash_attn2 as J
    S, Hq, Hkv, D, tail = 2 ** 17 + 2 ** 11, 130, 1, 128, 1024
    g = torch.Generator(device="cuda").manual_seed(4)
    make = lambda h: torch.randn(1, S, h, D, generator=g, device="cuda", dtype=BF16)
    q, k, v, do = make(Hq), make(Hkv), make(Hkv), make(Hq)
    assert q.numel() > 2 ** 31
    ids = (torch.arange(S, device="cuda", dtype=torch.int32) // 128)[None]

    def run(q, k, v, do, ids):
        leaves = [x.detach().requires_grad_(True) for x in (q, k, v)]
        out = J.scored_flash_attention(*leaves, None, True, softcap=20.0, document_ids=ids)
        return [out.detach(), *torch.autograd.grad(out, leaves, do)]

    got = [x[:, -tail:].clone() for x in run(q, k, v, do, ids)]
    want = run(*(x[:, -tail:].contiguous() for x in (q, k, v, do, ids)))
    assert J.device_status() == 0
    # one key tile takes part in a row of dq, so that only the sums of dk and dv over the heads may be in another order:
    # half a step of the result and the sums of 130 heads x 128 queries in 32 bits
    assert torch.equal(got[0], want[0]) and torch.equal(got[1], want[1])
    for x, y in zip(got[2:], want[2:]):
        x, y = x.double(), y.double()
        assert torch.all((x - y).abs() <= 2 * 2 ** -8 * y.abs() + 2e-3 * y.abs().mean())


def test_batch_rows_far_apart():
    import jax_flash_attn2 as J
    shape, step = (2, 200, 2, 64), 2 ** 31 + 64
    near = W.make_qkv(2, 200, 200, 2, 2, 64, BF16)
    room = torch.empty(step + 200 * 2 * 64, dtype=BF16, device="cuda")
    base = [x.cuda().requires_grad_(True) for x in near[:3]]
    want = J.scored_flash_attention(*base, None, True, softcap=20.0)
    grads = torch.autograd.grad(want, base, near[3].cuda())
    far = torch.as_strided(room, shape, (step, 128, 64, 1))
    for which in range(3):
        with torch.no_grad():
            far.copy_(base[which])
        leaves = list(base)
        leaves[which] = far.detach().requires_grad_(True)
        out = J.scored_flash_attention(*leaves, None, True, softcap=20.0)
        assert torch.equal(out, want)
        assert torch.equal(torch.autograd.grad(out, leaves, near[3].cuda())[2], grads[2])
    with torch.no_grad():
        far.copy_(near[3])
    out = J.scored_flash_attention(*base, None, True, softcap=20.0)
    assert torch.equal(torch.autograd.grad(out, base, far)[1], grads[1])
    assert J.device_status() == 0


def test_graph_bookkeeping():
    """Second passes, changed operands, hooks and several consumers behave as for other torch operators."""
    import jax_flash_attn2 as J
    q, k, v, do = (x.cuda() for x in W.make_qkv(1, 70, 70, 2, 2, 64, BF16))
    leaves = [x.requires_grad_(True) for x in (q, k, v)]
    prefix = torch.tensor([5], dtype=torch.int32, device="cuda")
    f = lambda: J.scored_flash_attention(*leaves, None, True, softcap=20.0, prefix_lens=prefix)
    out = f()
    assert out.requires_grad and out.grad_fn.name() == "ScoredAttentionBackward" and not out.is_leaf
    first = torch.autograd.grad(out, leaves, do, retain_graph=True)
    second = torch.autograd.grad(out, leaves, do)
    assert all(torch.equal(x, y) for x, y in zip(first, second))
    with pytest.raises(RuntimeError, match="second time"):
        torch.autograd.grad(out, leaves, do)
    for what in ("prefix", "out"):
        out = f()
        with torch.no_grad():
            (prefix if what == "prefix" else out).add_(0)
        with pytest.raises(RuntimeError, match="modified by an inplace operation"):
            torch.autograd.grad(out, leaves, do)
    packed = []
    with torch.autograd.graph.saved_tensors_hooks(lambda x: packed.append(x.shape) or x.cpu(), lambda x: x.cuda()):
        out = f()
    assert len(packed) >= 4
    assert all(torch.equal(x, y) for x, y in zip(first, torch.autograd.grad(out, leaves, do)))
    # two layers on one input, and no gradient asked for one operand
    a = f() + f()
    assert torch.equal(torch.autograd.grad(a, leaves[1], do)[0], 2 * first[1])
    # gradients that are accumulated into
    f().backward(do)
    f().backward(do)
    assert torch.equal(leaves[2].grad, 2 * first[2])
    out = f()
    assert torch.autograd.grad(out.sum() * 0 + leaves[0].sum() * 0, leaves[0])[0].abs().max() == 0
