"""GPU tests of serving with a paged cache: the plan against a plain one in Python, the cache write, the attention
against float64 with bounds that add up the 16-bit roundings, and whole steps as a server runs them."""
import random

import pytest
import torch

from oracle import scored as O

pytestmark = pytest.mark.gpu

BF16, FP16 = torch.bfloat16, torch.float16


def plain_plan(context, new, table, free, page, tokens, start=0):
    """The plan, request by request and token by token."""
    table = [list(r) for r in table]
    width = len(table[0])
    cu, lens, slots, positions, taken = [0], [], [], [], 0
    for b, (c, n) in enumerate(zip(context, new)):
        c, n = max(0, c), max(0, n)
        n = min(n, tokens - cu[-1])
        cu.append(cu[-1] + n)
        lens.append(c + n)
        for pg in range(-(-c // page), min(width, -(-(c + n) // page))):
            table[b][pg] = free[start + taken] if start + taken < len(free) else -1
            taken += 1
        for i in range(n):
            pos = c + i
            positions.append(pos)
            pg = table[b][pos // page] if pos // page < width else -1
            slots.append(pg * page + pos % page if pg >= 0 else -1)
    return dict(cu_seqlens=cu, seqlens_k=lens, block_table=table, slot_map=slots + [-1] * (tokens - len(slots)),
                positions=positions + [0] * (tokens - len(positions)), pages_taken=[taken])


def make_step(context, new, page, seed=0, extra_width=2, spare_pages=3):
    """(block table with the pages of the contexts, free pages, pool size), pages in random order."""
    r = random.Random(seed)
    need = [-(-(c + n) // page) for c, n in zip(context, new)]
    have = [-(-c // page) for c in context]
    pool = list(range(sum(need) + spare_pages))
    r.shuffle(pool)
    width = max(need) + extra_width
    table = [[-1] * width for _ in new]
    at = 0
    for b, n in enumerate(have):
        table[b][:n] = pool[at:at + n]
        at += n
    return table, pool[at:], len(pool)


def dev_int(x):
    return torch.tensor(x, dtype=torch.int32, device="cuda")


PLANS = [
    ([0], [1], 16, 0), ([15], [1], 16, 0), ([16], [1], 16, 3), ([17], [40], 8, 0), ([0, 0, 0], [0, 0, 0], 16, 0),
    ([0, 0, 0], [0, 0, 0], 16, 5), ([5, 0, 33, 64, 1], [0, 7, 0, 1, 300], 32, 11),
    ([100] * 40, [1] * 40, 64, 0), ([3, 200, 0], [2500, 1, 5000], 128, 1),
    ([i % 50 for i in range(1500)], [i % 4 for i in range(1500)], 8, 9),
    ([i % 30 for i in range(8192)], [1 - i % 2 for i in range(8192)], 16, 0),
]


@pytest.mark.parametrize("case", range(len(PLANS)))
def test_plan(case):
    import jax_flash_attn2 as J
    context, new, page, spare = PLANS[case]
    table, free, _ = make_step(context, new, page, case)
    tokens = sum(new) + spare
    start = 2 if len(free) > sum(new) + 2 else 0
    want = plain_plan(context, new, table, free, page, tokens, start)
    dt = dev_int(table)
    args = (dev_int(context), dev_int(new), dt, dev_int(free))
    for _ in range(2):      # the same arguments give the same plan
        plan = J.paged_step_plan(*args, page_size=page, num_tokens=tokens, heads_q=8, heads_kv=2, free_start=dev_int([start]))
        for name, x in want.items():
            assert getattr(plan, name).tolist() == x, name
    assert plan.block_table is dt


@pytest.mark.parametrize("heads_q,heads_kv", [(4, 4), (32, 8), (7, 1), (128, 1), (96, 1)])
def test_work_list_covers_every_token_once(heads_q, heads_kv):
    import jax_flash_attn2 as J
    context, new, page = [0, 700, 130, 0, 3, 0], [1500, 1, 0, 129, 64, 1], 16
    table, free, _ = make_step(context, new, page)
    plan = J.paged_step_plan(dev_int(context), dev_int(new), dev_int(table), dev_int(free), page_size=page, num_tokens=sum(new) + 9,
                             heads_q=heads_q, heads_kv=heads_kv)
    per = 2 * (128 // (heads_q // heads_kv))
    want, before, start = [], 0, {2: 4, 3: 8}        # start: of the start and end of an item
    for b, (c, n) in enumerate(zip(context, new)):
        for t in range(0, n, per):
            m = min(per, n - t)
            tiles = -(-(c + t + m) // 128)
            cost = 3 if 2 * m > per else 2      # a key tile of an item that fills both query tiles, of another
            want.append([sum(new[:b]) + t, m, c + t, b, before, tiles, cost, 0])
            before += cost * tiles + start[cost]
    work = plan.work.tolist()
    sms = torch.cuda.get_device_properties(0).multi_processor_count
    at = 16 + (4 * (sms + 1) + 7) // 8 * 8
    assert work[:2] == [len(want), min(sms, before * heads_kv // 2)]
    assert work[at:at + 8 * len(want)] == [x for w in want for x in w]
    # the CTAs' starts go through every tile of every item and head once, in order
    starts = [tuple(work[16 + 4 * c:19 + 4 * c]) for c in range(work[1] + 1)]
    assert starts[0] == (0, 0, 0) and starts[-1] == (heads_kv, 0, 0) and starts == sorted(starts)
    assert all(tile < want[item][5] for _, item, tile in starts[:-1])
    share = before * heads_kv / work[1]
    cost = lambda s: s[0] * before + (want[s[1]][4] + s[2] * want[s[1]][6] + start[want[s[1]][6]] * (s[2] > 0) if s[0] < heads_kv else 0)
    # (borders move by two tiles of the dearer kind at most, and into the cost of a start)
    assert all(cost(b) - cost(a) <= share + 2 * (6 + 8) + 3 for a, b in zip(starts, starts[1:]))


def test_plan_without_enough_pages_width_or_rows():
    import jax_flash_attn2 as J
    # pages run out in the second request; the third's table row is too narrow; the packed rows end inside the fourth
    context, new, page = [3, 10, 60, 0], [30, 40, 30, 50], 16
    table = [[4] + [-1] * 4, [5] + [-1] * 4, [6, 7, 8, 9, -1], [-1] * 5]
    free = [20, 21, 22, 23]
    tokens = 130
    want = plain_plan(context, new, table, free, page, tokens)
    plan = J.paged_step_plan(dev_int(context), dev_int(new), dev_int(table), dev_int(free), page_size=page, num_tokens=tokens, heads_q=2, heads_kv=2)
    for name, x in want.items():
        assert getattr(plan, name).tolist() == x, name
    assert plan.pages_taken.item() > len(free) and (plan.slot_map == -1).any()
    # no free pages at all, lengths below zero
    plan = J.paged_step_plan(dev_int([-4, 0]), dev_int([3, -7]), dev_int([[-1], [-1]]), dev_int([]), page_size=16, num_tokens=4, heads_q=2, heads_kv=2)
    assert plan.cu_seqlens.tolist() == [0, 3, 3] and plan.seqlens_k.tolist() == [3, 0] and plan.slot_map.tolist() == [-1] * 4


@pytest.mark.parametrize("page,heads,D,dtype", [(16, 8, 128, BF16), (8, 1, 64, FP16), (128, 3, 40, BF16), (32, 5, 256, FP16)])
@pytest.mark.parametrize("heads_first", [False, True])
def test_cache_write(page, heads, D, dtype, heads_first):
    import jax_flash_attn2 as J
    g = torch.Generator().manual_seed(3)
    pages, tokens = 37, 75
    joint = torch.randn(tokens, 2 * heads + 3, D, generator=g).to(dtype).cuda()     # k and v as slices of one projection
    k, v = joint[:, 1:1 + heads], joint[:, 2 + heads:2 + 2 * heads]
    slots = torch.randperm(pages * page, generator=g)[:tokens]
    slots[::7] = -1
    slots[5], slots[6] = pages * page, 2 ** 40      # behind the cache: skipped as well
    shape = (pages, heads, page, D) if heads_first else (pages, page, heads, D)
    caches = [torch.randn(shape, generator=g).to(dtype).cuda() for _ in range(2)]
    if heads_first:
        caches = [c.permute(0, 2, 1, 3) for c in caches]
    want = [c.clone() for c in caches]
    for c, x in zip(want, (k, v)):
        for t, s in enumerate(slots.tolist()):
            if 0 <= s < pages * page:
                c[s // page, s % page] = x[t]
    J.paged_cache_write(k, v, *caches, slots.cuda())
    assert all(torch.equal(c, w) for c, w in zip(caches, want))
    J.paged_cache_write(k[:0], v[:0], *caches, slots[:0].cuda())
    assert all(torch.equal(c, w) for c, w in zip(caches, want))


def serve(context, new, Hq, Hkv, D, dtype, page, *, cap=None, slopes=None, sharp=2.0, spare=0, heads_first=False, seed=1, scale=None):
    """One step through plan, cache write and attention; every request against float64."""
    import jax_flash_attn2 as J
    g = torch.Generator().manual_seed(seed)
    table, free, pages = make_step(context, new, page, seed)
    tokens = sum(new) + spare
    shape = (pages, Hkv, page, D) if heads_first else (pages, page, Hkv, D)
    caches = [torch.full(shape, float("nan"), dtype=dtype).cuda() for _ in range(2)]   # unwritten memory holds anything
    if heads_first:
        caches = [c.permute(0, 2, 1, 3) for c in caches]
    keys = [torch.randn(2, c + n, Hkv, D, generator=g).to(dtype) for c, n in zip(context, new)]
    q = (torch.randn(tokens, Hq, D, generator=g) * sharp).to(dtype)
    fresh = [torch.cat([x[i, c:] for x, c in zip(keys, context)] + [torch.zeros(spare, Hkv, D, dtype=dtype)]) for i in range(2)]
    # the contexts as an earlier plan of whole prompts wrote them
    before = J.paged_step_plan(dev_int([0] * len(new)), dev_int(context), dev_int([[-1] * len(table[0])] * len(new)), dev_int([p for r in table for p in r if p >= 0]),
                               page_size=page, num_tokens=sum(context), heads_q=Hq, heads_kv=Hkv)
    J.paged_cache_write(*(torch.cat([x[i, :c] for x, c in zip(keys, context)]).cuda() for i in range(2)), *caches, before.slot_map)
    plan = J.paged_step_plan(dev_int(context), dev_int(new), before.block_table, dev_int(free), page_size=page, num_tokens=tokens, heads_q=Hq, heads_kv=Hkv)
    J.paged_cache_write(*(x.cuda() for x in fresh), *caches, plan.slot_map)
    out = torch.full((tokens, Hq, D), 7.0, dtype=dtype, device="cuda")
    lse = torch.full((tokens, Hq), 7.0, device="cuda")
    got = J.paged_attention(q.cuda(), *caches, plan, scale, softcap=cap, alibi_slopes=None if slopes is None else slopes.cuda(), out=out, lse=lse)
    assert got is out and J.device_status() == 0
    got, lse = out.cpu(), lse.cpu()
    at = 0
    for (c, n), x in zip(zip(context, new), keys):
        if n:
            r = O.attention(q[None, at:at + n], x[None, 0], x[None, 1], O.visible_keys(1, n, c + n, True), scale, cap, slopes)
            assert O.worst(got[None, at:at + n], r["out"], O.bounds(r, dtype)["out"]) <= 1.0, (c, n)
            assert (lse[at:at + n].T - r["lse"][0]).abs().max() <= 1e-3
        at += n
    assert torch.all(got[at:] == 7.0) and torch.all(lse[at:] == 7.0)


SLOPES = lambda n: torch.tensor([2.0 ** (-8.0 * (i + 1) / n) for i in range(n)])


@pytest.mark.parametrize("D,dtype", [(64, BF16), (128, BF16), (64, FP16), (128, FP16), (40, BF16), (96, FP16)])
@pytest.mark.parametrize("cap,slopes", [(None, False), (20.0, False), (None, True), (20.0, True)])
def test_mixed_step(D, dtype, cap, slopes):
    serve([0, 500, 127, 128, 1, 300], [70, 1, 1, 1, 3, 0], 8, 2, D, dtype, 16, cap=cap, slopes=SLOPES(8) if slopes else None, spare=5)


@pytest.mark.parametrize("page", [8, 16, 32, 64, 128, 256, 1024])
@pytest.mark.parametrize("D", [64, 128])
def test_page_sizes(page, D):
    serve([200, 0, 383, page - 1, page], [1, 300, 129, 1, 1], 4, 2, D, BF16, page, cap=30.0)


@pytest.mark.parametrize("Hq,Hkv", [(1, 1), (8, 8), (6, 2), (7, 1), (48, 1), (128, 1), (65, 1), (40, 8)])
def test_head_groups(Hq, Hkv):
    serve([130, 0, 5], [1, 40, 200], Hq, Hkv, 64, FP16, 32, slopes=SLOPES(Hq))


@pytest.mark.parametrize("context,new", [([0], [1]), ([0], [2]), ([127], [1]), ([128], [1]), ([0], [128]), ([1], [127]), ([4000], [1]),
                                         ([0], [1000]), ([2900], [333]), ([9000], [2])])
@pytest.mark.parametrize("D", [64, 128])
def test_one_request(context, new, D):
    serve(context, new, 8, 2, D, BF16, 16)


def test_more_requests_than_ctas_and_uneven_contexts():
    r = random.Random(4)
    context = [r.choice([0, 1, 15, 16, 100, 128, 1000]) for _ in range(180)]
    serve(context, [r.choice([0, 1, 1, 1, 2, 9]) for _ in context], 4, 4, 64, BF16, 16, cap=10.0, spare=3)


@pytest.mark.parametrize("heads_first", [False, True])
def test_cache_with_heads_before_places(heads_first):
    serve([100, 31], [1, 50], 4, 2, 128, BF16, 64, heads_first=heads_first)


def test_caps_and_scales_at_their_ends():
    for cap in (2.0 ** -10, 1024.0):
        serve([300], [5], 2, 1, 64, BF16, 16, cap=cap, sharp=8.0)
    serve([300], [5], 2, 1, 64, BF16, 16, scale=0.9)


def test_pages_outside_the_pool_read_as_zeros():
    import jax_flash_attn2 as J
    page, D, n = 16, 64, 40
    g = torch.Generator().manual_seed(5)
    k, v = (torch.randn(6, page, 1, D, generator=g).to(BF16) for _ in range(2))
    table = [[0, -1, 6]]      # no page, and one behind the pool
    plan = J.paged_step_plan(dev_int([n - 1]), dev_int([1]), dev_int(table), dev_int([]), page_size=page, num_tokens=1, heads_q=1, heads_kv=1)
    q = torch.randn(1, 1, D, generator=g).to(BF16)
    out = J.paged_attention(q.cuda(), k.cuda(), v.cuda(), plan)
    assert J.device_status() == 0
    full = [torch.cat([x[0], torch.zeros(24, 1, D, dtype=BF16)])[None] for x in (k, v)]
    r = O.attention(q[None], *full, O.visible_keys(1, 1, n, True))
    assert O.worst(out.cpu()[None], r["out"], O.bounds(r, BF16)["out"]) <= 1.0


def test_step_without_new_tokens():
    import jax_flash_attn2 as J
    cache = torch.zeros(2, 16, 1, 64, dtype=BF16, device="cuda")
    plan = J.paged_step_plan(dev_int([5]), dev_int([0]), dev_int([[0]]), dev_int([1]), page_size=16, num_tokens=3, heads_q=1, heads_kv=1)
    out = torch.full((3, 1, 64), 2.0, dtype=BF16, device="cuda")
    J.paged_attention(torch.ones(3, 1, 64, dtype=BF16, device="cuda"), cache, cache, plan, out=out)
    assert torch.all(out == 2.0) and J.device_status() == 0
    empty = J.paged_step_plan(dev_int([5]), dev_int([0]), dev_int([[0]]), dev_int([1]), page_size=16, num_tokens=0, heads_q=1, heads_kv=1)
    assert J.paged_attention(torch.ones(0, 1, 64, dtype=BF16, device="cuda"), cache, cache, empty).shape == (0, 1, 64)


def test_strided_queries_and_output():
    import jax_flash_attn2 as J
    g = torch.Generator().manual_seed(6)
    page, D, Hq, Hkv, n = 16, 128, 8, 2, 90
    pages = 8
    k, v = (torch.randn(pages, page, Hkv, D, generator=g).to(BF16).cuda() for _ in range(2))
    plan = J.paged_step_plan(dev_int([10]), dev_int([n]), dev_int([list(range(1)) + [-1] * 6]), dev_int(list(range(1, 8))), page_size=page,
                             num_tokens=n, heads_q=Hq, heads_kv=Hkv)
    joint = torch.randn(n, Hq + 4, D, generator=g).to(BF16).cuda()
    wide = torch.zeros(n, Hq + 2, D, dtype=BF16, device="cuda")
    q = joint[:, 3:3 + Hq]
    want = J.paged_attention(q.contiguous(), k, v, plan)
    J.paged_attention(q, k, v, plan, out=wide[:, 1:1 + Hq])
    assert torch.equal(wide[:, 1:1 + Hq], want) and torch.all(wide[:, 0] == 0) and torch.all(wide[:, -1] == 0)


@pytest.mark.parametrize("cap,slopes", [(None, False), (25.0, True)])
def test_a_prompt_in_chunks_then_single_tokens_equals_the_dense_operator(cap, slopes):
    """Three layers' worth of steps through one plan each: a prompt of 700 tokens read in chunks of 300, then 5 tokens one
    by one, against scored_flash_attention over the whole sequence. Both round P and the output to bf16: two half steps
    each way of the weighted |v|."""
    import jax_flash_attn2 as J
    Hq, Hkv, D, page, total = 8, 2, 64, 32, 705
    g = torch.Generator().manual_seed(8)
    sl = SLOPES(Hq).cuda() if slopes else None
    layers = [[torch.randn(1, total, h, D, generator=g).to(BF16).cuda() for h in (Hq, Hkv, Hkv)] for _ in range(3)]
    caches = [[torch.full((30, page, Hkv, D), float("nan"), dtype=BF16, device="cuda") for _ in range(2)] for _ in layers]
    table = dev_int([[-1] * 24])
    free, start = dev_int(list(range(29, -1, -1))), dev_int([0])
    outs, at = [[] for _ in layers], 0
    for n in [300, 300, 100, 1, 1, 1, 1, 1]:
        plan = J.paged_step_plan(dev_int([at]), dev_int([n]), table, free, page_size=page, num_tokens=n, heads_q=Hq, heads_kv=Hkv, free_start=start)
        start += plan.pages_taken
        for (q, k, v), cache, out in zip(layers, caches, outs):
            J.paged_cache_write(k[0, at:at + n], v[0, at:at + n], *cache, plan.slot_map)
            out.append(J.paged_attention(q[0, at:at + n], *cache, plan, softcap=cap, alibi_slopes=sl))
        at += n
    assert start.item() == 23 and J.device_status() == 0
    for (q, k, v), out in zip(layers, outs):
        want = J.scored_flash_attention(q, k, v, None, True, softcap=cap, alibi_slopes=sl)[0].float()
        weight = J.scored_flash_attention(q, k, v.abs(), None, True, softcap=cap, alibi_slopes=sl)[0].float()
        assert torch.all((torch.cat(out).float() - want).abs() <= 2 * 2.0 ** -8 * (weight + want.abs()))


def test_a_captured_step_is_replayed_with_other_lengths():
    import jax_flash_attn2 as J
    Hq, Hkv, D, page, T, B = 4, 2, 128, 16, 24, 6
    g = torch.Generator().manual_seed(10)
    pages = 200
    caches = [torch.randn(pages, page, Hkv, D, generator=g).to(BF16).cuda() for _ in range(2)]
    q, k, v = (torch.randn(T, h, D, generator=g).to(BF16).cuda() for h in (Hq, Hkv, Hkv))
    order = torch.randperm(pages, generator=g).to(torch.int32)
    table = order[:B * 25].view(B, 25).clone().cuda()
    context, new, free = dev_int([0] * B), dev_int([1] * B), order[B * 25:].clone().cuda()
    out = torch.zeros(T, Hq, D, dtype=BF16, device="cuda")

    def step():
        plan = J.paged_step_plan(context, new, table, free, page_size=page, num_tokens=T, heads_q=Hq, heads_kv=Hkv)
        J.paged_cache_write(k, v, *caches, plan.slot_map)
        J.paged_attention(q, *caches, plan, softcap=20.0, out=out)

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step()
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        step()
    for c, n in (([5, 380, 0, 17, 100, 31], [1, 1, 1, 1, 1, 1]), ([10, 0, 200, 64, 48, 399], [3, 9, 0, 4, 7, 1]), ([0] * 6, [0] * 6)):
        context.copy_(dev_int(c))
        new.copy_(dev_int(n))
        out.zero_()
        saved = [x.clone() for x in (table, *caches)]
        graph.replay()
        torch.cuda.synchronize()
        got = out.clone()
        for x, y in zip((table, *caches), saved):
            x.copy_(y)
        out.zero_()
        step()
        torch.cuda.synchronize()
        assert torch.equal(got, out) and torch.all(out[sum(n):] == 0)
    assert J.device_status() == 0


def test_steps_on_two_streams():
    import jax_flash_attn2 as J
    g = torch.Generator().manual_seed(12)
    page, Hq, Hkv, D = 16, 8, 2, 128
    work = []
    for seed in range(2):
        context, new = [700, 90, 0], [1, 200, 64]
        table, free, pages = make_step(context, new, page, seed)
        caches = [torch.randn(pages, page, Hkv, D, generator=g).to(BF16).cuda() for _ in range(2)]
        q = torch.randn(sum(new), Hq, D, generator=g).to(BF16).cuda()
        work.append((dev_int(context), dev_int(new), dev_int(table), dev_int(free), sum(new), q, caches))

    def run(c, n, t, f, tokens, q, caches):
        return J.paged_attention(q, *caches, J.paged_step_plan(c, n, t, f, page_size=page, num_tokens=tokens, heads_q=Hq, heads_kv=Hkv))

    want = [run(*w) for w in work]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in work]
    got = []
    for _ in range(4):
        for s, w in zip(streams, work):
            with torch.cuda.stream(s):
                got.append(run(*w))
    torch.cuda.synchronize()
    assert all(torch.equal(x, want[i % 2]) for i, x in enumerate(got))


def test_calls_that_are_not_offered():
    import jax_flash_attn2 as J
    cache = torch.zeros(4, 16, 2, 64, dtype=BF16, device="cuda")
    plan = J.paged_step_plan(dev_int([5]), dev_int([1]), dev_int([[0]]), dev_int([1]), page_size=16, num_tokens=1, heads_q=4, heads_kv=2)
    q = torch.zeros(1, 4, 64, dtype=BF16, device="cuda")
    with pytest.raises(ValueError, match="the plan is for"):
        J.paged_attention(torch.zeros(2, 4, 64, dtype=BF16, device="cuda"), cache, cache, plan)
    with pytest.raises(ValueError, match="the plan is for"):
        J.paged_attention(torch.zeros(1, 2, 64, dtype=BF16, device="cuda"), cache, cache, plan)
    with pytest.raises(RuntimeError, match="no backward"):
        J.paged_attention(q.clone().requires_grad_(True), cache, cache, plan)
    with pytest.raises(ValueError, match="q must be"):
        J.paged_attention(q.half(), cache, cache, plan)
    with pytest.raises(ValueError, match="out must"):
        J.paged_attention(q, cache, cache, plan, out=torch.zeros(1, 4, 32, dtype=BF16, device="cuda"))
    wide = torch.zeros(4, 16, 2, 256, dtype=BF16, device="cuda")
    with pytest.raises(J._capi.Fa2Error, match="head_dim"):
        J.paged_attention(torch.zeros(1, 4, 256, dtype=BF16, device="cuda"), wide, wide, plan)
    with pytest.raises(ValueError, match="slot_map"):
        J.paged_cache_write(cache[0, :1], cache[0, :1], cache, cache, torch.zeros(1, dtype=torch.int32, device="cuda"))


def test_writes_in_place_are_known_to_autograd():
    import jax_flash_attn2 as J
    cache, other = (torch.zeros(4, 16, 2, 64, dtype=BF16, device="cuda") for _ in range(2))
    table = dev_int([[0]])
    plan = J.paged_step_plan(dev_int([5]), dev_int([1]), table, dev_int([1]), page_size=16, num_tokens=1, heads_q=4, heads_kv=2)
    k = torch.ones(1, 2, 64, dtype=BF16, device="cuda")
    J.paged_cache_write(k, k, cache, other, plan.slot_map)
    out, lse = torch.zeros(1, 4, 64, dtype=BF16, device="cuda"), torch.zeros(1, 4, device="cuda")
    J.paged_attention(out.clone(), cache, other, plan, out=out, lse=lse)
    assert [x._version for x in (table, cache, other, out, lse)] == [1] * 5
    # copied operands go through the Python function
    J.paged_cache_write(k.transpose(1, 2).contiguous().transpose(1, 2), k, cache, other, plan.slot_map)
    assert cache._version == 2 and other._version == 2
    with pytest.raises(RuntimeError, match="no backward"):
        J.paged_cache_write(k.clone().requires_grad_(True), k, cache, other, plan.slot_map)
    with pytest.raises(RuntimeError, match="no backward"):
        J.paged_attention(out.detach(), cache, other, plan, out=torch.zeros_like(out).requires_grad_(True))
    with torch.inference_mode():
        fresh = torch.zeros(4, 16, 2, 64, dtype=BF16, device="cuda")
        J.paged_cache_write(k, k, fresh, fresh.clone(), plan.slot_map)
    assert torch.equal(fresh, cache)
    plan.block_table = table.cpu()
    with pytest.raises(ValueError, match="one device"):
        J.paged_attention(out.detach(), cache, other, plan)
    plan.block_table = table.long()
    with pytest.raises(ValueError, match="paged_step_plan"):
        J.paged_attention(out.detach(), cache, other, plan)


@pytest.mark.parametrize("requests", [4097, 5000])
def test_more_items_than_the_plan_keeps_in_shared_memory(requests):
    import jax_flash_attn2 as J
    g = torch.Generator().manual_seed(requests)
    page, width, Hq, Hkv, D = 8, 6, 4, 2, 64
    context = torch.randint(0, page * width - 1, (requests,), generator=g, dtype=torch.int32)
    pages = requests * width
    table = torch.randperm(pages, generator=g).to(torch.int32).view(requests, width)
    kc, vc = (torch.randn(pages, page, Hkv, D, generator=g).to(BF16) for _ in range(2))
    q = torch.randn(requests, Hq, D, generator=g).to(BF16)
    # (pages that the new tokens open are taken from the same pool: some page may serve two requests, which changes nothing here)
    plan = J.paged_step_plan(context.cuda(), torch.ones_like(context).cuda(), table.cuda(), table.flatten().cuda(), page_size=page,
                             num_tokens=requests, heads_q=Hq, heads_kv=Hkv)
    assert torch.equal(plan.seqlens_k.cpu(), context + 1)
    used = plan.block_table.cpu()
    out = J.paged_attention(q.cuda(), kc.cuda(), vc.cuda(), plan).cpu()
    assert J.device_status() == 0
    k, v = (x[used.long()].reshape(requests, page * width, Hkv, D).double() for x in (kc, vc))
    s = torch.einsum("rhgd,rjhd->rhgj", q.double().view(requests, Hkv, Hq // Hkv, D), k) / D ** 0.5
    seen = torch.arange(page * width) <= context[:, None]
    p = torch.softmax(s.masked_fill(~seen[:, None, None], -torch.inf), -1)
    want = torch.einsum("rhgj,rjhd->rhgd", p, v).reshape(requests, Hq, D)
    # half a step for the weights, half a step for the output, a hundredth of that for sums in 32 bits and the exponential
    size = torch.einsum("rhgj,rjhd->rhgd", p, v.abs()).reshape(requests, Hq, D)
    assert torch.all((out.double() - want).abs() <= 2.02 * 2 ** -8 * size + 1e-6)


def test_a_pool_of_more_than_2_31_elements():
    import jax_flash_attn2 as J
    g = torch.Generator().manual_seed(3)
    page, Hq, Hkv, D, used = 16, 4, 2, 64, 40
    pages = 2 ** 31 // (page * Hkv * D) + used
    context, new = [300, 17], [40, 1]
    small = [torch.randn(used, page, Hkv, D, generator=g).to(BF16).cuda() for _ in range(2)]
    large = [torch.empty(pages, page, Hkv, D, dtype=BF16, device="cuda") for _ in range(2)]
    for a, b in zip(large, small):
        a[-used:] = b
    assert large[0][-1].data_ptr() - large[0].data_ptr() > 2 * 2 ** 31
    q = torch.randn(sum(new), Hq, D, generator=g).to(BF16).cuda()
    k, v = (torch.randn(sum(new), Hkv, D, generator=g).to(BF16).cuda() for _ in range(2))
    order = torch.randperm(used, generator=g).to(torch.int32)
    outs = []
    for first, caches in ((0, small), (pages - used, large)):
        table = torch.full((2, 24), -1, dtype=torch.int32)
        table[0, :19] = order[:19] + first
        table[1, :2] = order[19:21] + first
        plan = J.paged_step_plan(dev_int(context), dev_int(new), table.cuda(), (order[21:] + first).cuda(), page_size=page,
                                 num_tokens=sum(new), heads_q=Hq, heads_kv=Hkv)
        J.paged_cache_write(k, v, *caches, plan.slot_map)
        outs.append(J.paged_attention(q, *caches, plan))
    assert torch.equal(outs[0], outs[1]) and torch.equal(small[0], large[0][-used:]) and torch.equal(small[1], large[1][-used:])
    assert torch.isfinite(outs[0].float()).all() and J.device_status() == 0


@pytest.mark.parametrize("D", [64, 96, 128])
@pytest.mark.parametrize("page", [8, 16, 64, 256])
def test_every_layout_of_the_cache_gives_the_same_bits(D, page):
    import jax_flash_attn2 as J
    g = torch.Generator().manual_seed(page + D)
    Hq, Hkv, context, new = 6, 3, [300, 0, 41, 700], [1, 130, 7, 1]
    table, free, pages = make_step(context, new, page)
    k, v = (torch.randn(pages, page, Hkv, D, generator=g).to(BF16).cuda() for _ in range(2))
    q = torch.randn(sum(new), Hq, D, generator=g).to(BF16).cuda()
    plan = J.paged_step_plan(dev_int(context), dev_int(new), dev_int(table), dev_int(free), page_size=page, num_tokens=sum(new),
                             heads_q=Hq, heads_kv=Hkv)
    both = torch.stack([k, v], 1)                                          # [pages, 2, page, Hkv, D]
    heads_first = [x.transpose(1, 2).contiguous().transpose(1, 2) for x in (k, v)]
    wide = [torch.nn.functional.pad(x, (0, 8)).contiguous()[..., :D] for x in (k, v)]      # rows of D + 8
    layouts = [(k, v), (both[:, 0], both[:, 1]), heads_first, (k, heads_first[1]), wide]
    assert heads_first[0].stride(1) == D and both[:, 0].stride(0) == 2 * page * Hkv * D
    outs = [J.paged_attention(q, *x, plan) for x in layouts]
    assert torch.isfinite(outs[0].float()).all() and all(torch.equal(x, outs[0]) for x in outs) and J.device_status() == 0
