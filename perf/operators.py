"""Measured cases of the attention operators for language models: attention with modified scores (forward and
backward), the plan of a serving step (block tables, slot maps), the write into a paged key/value cache, and the
attention of new tokens over that cache.

`run` computes an operator in its plain form (elementary torch operations in float32, rounded once at the end), or
with the framework's kernels where the module variable `own` is true. `exact` computes the same from the
definitions in float64, request by request and head by head.
"""
from __future__ import annotations

import math
import os
import random
import sys

import torch

own = False

_DEV = torch.device("cuda" if torch.cuda.is_available() else "cpu")
_DT = {"bf16": torch.bfloat16, "fp16": torch.float16}


def _package():
    root = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "jax-flash-attn2_b200")
    if root not in sys.path:
        sys.path.insert(0, root)
    import jax_flash_attn2
    return jax_flash_attn2


# ------------------------------------------------------------------------------------------------
# cases
# ------------------------------------------------------------------------------------------------
def _scored(name, **kw):
    """Attention with modified scores. `docs`: mean length of the documents packed into a row (0: none), the last
    `tail` tokens of every row being padding. `prefix`: largest length of the prefix every query sees. `train`:
    gradients as well. `sharp`: standard deviation of the scores."""
    case = dict(op="scored", name=name, batch=1, seq_q=0, seq_k=0, heads_q=8, heads_kv=8, dim=64, dtype="bf16", causal=True,
                cap=0.0, alibi=False, docs=0, tail=0, prefix=0, sharp=1.0, train=True, layout=1)
    case.update(kw)
    return case


def _paged(name, **kw):
    """Attention of new tokens over a paged cache: `requests` requests of which every `chunk_every`-th brings up to
    `chunk` new tokens and the others bring one; contexts between `ctx_min` and `ctx_max`. `spare`: rows of the packed
    tensors behind the last request."""
    case = dict(op="paged", name=name, requests=1, chunk=1, chunk_every=1, ctx_min=1, ctx_max=64, page=16, heads_q=8,
                heads_kv=8, dim=64, dtype="bf16", cap=0.0, alibi=False, sharp=1.0, spare=0, layout=1)
    case.update(kw)
    return case


def listed():
    return [
        # a short fine-tuning batch, where the launches count
        _scored("scored_cap_short", batch=2, seq_q=512, seq_k=512, heads_q=16, heads_kv=4, dim=64, dtype="fp16", cap=30.0, sharp=4.0),
        # pretraining on packed documents, padded at the end of every row
        _scored("scored_docs", batch=4, seq_q=4096, seq_k=4096, heads_q=32, heads_kv=8, dim=128, docs=700, tail=61, layout=5),
        # a prefix model with distance bias on a length that is no multiple of a tile
        _scored("scored_alibi_prefix_odd", batch=3, seq_q=1537, seq_k=1537, heads_q=16, heads_kv=16, dim=96, dtype="fp16", alibi=True, prefix=700, layout=3),
        # a long training row with capped scores
        _scored("scored_cap_long", batch=2, seq_q=8192, seq_k=8192, heads_q=32, heads_kv=8, dim=128, cap=50.0, sharp=4.0),
        # one user waiting for the next token
        _paged("paged_decode_one", requests=1, ctx_min=1000, ctx_max=1000, heads_q=32, heads_kv=8, dim=128),
        # a full decode batch with contexts of all lengths
        _paged("paged_decode_batch", requests=64, ctx_min=128, ctx_max=16384, heads_q=32, heads_kv=8, dim=128, page=16, layout=7),
        # a chunk of a long prompt
        _paged("paged_chunk_long", requests=1, chunk=4096, ctx_min=28672, ctx_max=28672, heads_q=64, heads_kv=8, dim=128, page=64),
        # prompts and decodes in one step, capped scores, rows behind the last request
        _paged("paged_mixed_cap", requests=24, chunk=700, chunk_every=6, ctx_min=1, ctx_max=6000, heads_q=16, heads_kv=4, dim=64,
               dtype="fp16", page=32, cap=30.0, sharp=4.0, spare=37, layout=11),
        # a decode step of a small server
        dict(op="plan", name="plan_decode", requests=32, chunk=1, chunk_every=1, ctx_min=1, ctx_max=8192, page=16, heads_q=32, heads_kv=8, spare=0, layout=2),
        # a step of a large server that mixes prompts and decodes
        dict(op="plan", name="plan_mixed", requests=700, chunk=2048, chunk_every=50, ctx_min=0, ctx_max=32768, page=64, heads_q=32, heads_kv=8, spare=100, layout=13),
        # the new keys and values of a decode step
        dict(op="write", name="write_decode", tokens=64, spare=0, heads_q=32, heads_kv=8, dim=128, dtype="bf16", page=16, pages=4096),
        # those of a step with long prompts
        dict(op="write", name="write_prompts", tokens=16384, spare=333, heads_q=32, heads_kv=8, dim=128, dtype="bf16", page=64, pages=1024),
    ]


def _log_int(rng, lo, hi):
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    op = rng.choice(["scored", "scored", "paged", "paged", "plan", "write"])
    dtype = rng.choice(["bf16", "fp16"])
    heads_kv = rng.choice([1, 2, 4, 8])
    heads_q = heads_kv * rng.choice([1, 2, 3, 4, 7, 8])
    dim = rng.choice([64, 96, 128])
    cap = rng.choice([0.0, 20.0, 50.0])
    layout = rng.randrange(1 << 20)
    if op == "scored":
        seq = _log_int(rng, 64, 6000)
        batch = rng.choice([1, 1, 2, 3]) if seq > 1500 else rng.choice([1, 2, 4, 6])
        docs = rng.choice([0, _log_int(rng, 16, max(17, seq))])
        causal = rng.random() < 0.8
        seq_k = seq if docs or rng.random() < 0.6 else max(1, seq + rng.randint(-seq // 3, seq // 2))
        case = dict(op=op, batch=batch, seq_q=seq, seq_k=seq_k, heads_q=heads_q, heads_kv=heads_kv, dim=rng.choice([dim, dim, 256]),
                    dtype=dtype, causal=causal, cap=cap, alibi=rng.random() < 0.4, docs=docs, tail=rng.randrange(0, 1 + seq // 8) if docs else 0,
                    prefix=rng.randrange(1, seq) if causal and rng.random() < 0.3 else 0, sharp=rng.choice([1.0, 4.0]),
                    train=rng.random() < 0.75, layout=layout)
        # no drawn case costs more than the largest listed one
        while 14.0 * batch * seq * seq_k * case["heads_q"] * case["dim"] > 3.8e12 and case["heads_kv"] > 1:
            case["heads_q"], case["heads_kv"] = case["heads_q"] // 2, case["heads_kv"] // 2
        if 14.0 * batch * seq * seq_k * case["heads_q"] * case["dim"] > 3.8e12:
            case["dim"] = 64
        return case
    if op == "paged":
        requests = _log_int(rng, 1, 100)
        ctx_max = _log_int(rng, 16, 400000 // requests if requests > 12 else 33000)
        chunk = rng.choice([1, rng.randint(2, 8), _log_int(rng, 16, 1500)])
        chunk = max(1, min(chunk, int(1e9 / (requests * (heads_q // heads_kv) * (ctx_max + chunk)))))
        return dict(op=op, requests=requests, chunk=chunk, chunk_every=rng.choice([1, 3, 9]) if chunk < 16 else max(1, requests // rng.choice([1, 2, 3])),
                    ctx_min=rng.choice([0, 1, ctx_max // 2]), ctx_max=ctx_max, page=rng.choice([16, 32, 64, 128]), heads_q=heads_q,
                    heads_kv=heads_kv, dim=dim, dtype=dtype, cap=cap, alibi=rng.random() < 0.3, sharp=rng.choice([1.0, 4.0]),
                    spare=rng.choice([0, 0, 13]), layout=layout)
    if op == "plan":
        requests = _log_int(rng, 1, 1000)
        chunk = _log_int(rng, 1, 2048)
        return dict(op=op, requests=requests, chunk=chunk, chunk_every=max(rng.randint(1, 60), requests * chunk // 20000), ctx_min=0, ctx_max=_log_int(rng, 16, 32768),
                    page=rng.choice([16, 32, 64, 128]), heads_q=heads_q, heads_kv=heads_kv, spare=rng.choice([0, rng.randrange(1, 200)]), layout=layout)
    tokens = _log_int(rng, 1, 16000)
    page = rng.choice([16, 32, 64, 128])
    return dict(op=op, tokens=tokens, spare=rng.choice([0, rng.randrange(1, 300)]), heads_q=heads_q, heads_kv=heads_kv, dim=dim, dtype=dtype,
                page=page, pages=(tokens * rng.choice([1, 2, 4])) // page + rng.randrange(2, 60))


# ------------------------------------------------------------------------------------------------
# lengths that follow from a case alone
# ------------------------------------------------------------------------------------------------
def _documents(case):
    """Lengths of the documents of every batch row (the rest of a row is padding), or None."""
    if not case["docs"]:
        return None
    r = random.Random(case["layout"])
    rows = []
    for _ in range(case["batch"]):
        left, row = case["seq_q"] - case["tail"], []
        while left > 0:
            n = min(left, max(1, int(r.expovariate(1.0 / case["docs"]))))
            row.append(n)
            left -= n
        rows.append(row)
    return rows


def _prefixes(case):
    r = random.Random(case["layout"] + 1)
    return [r.randint(0, case["prefix"]) for _ in range(case["batch"])] if case["prefix"] else None


def _requests(case):
    """(tokens in the cache, new tokens) of every request."""
    r = random.Random(case["layout"])
    lo, hi = max(1, case["ctx_min"]), max(1, case["ctx_max"])
    context, new = [], []
    for i in range(case["requests"]):
        chunked = i % case["chunk_every"] == 0
        new.append(r.randint((case["chunk"] + 1) // 2, case["chunk"]) if chunked and case["chunk"] > 1 and case["requests"] > 1 else case["chunk"] if chunked else 1)
        context.append(_log_int(r, lo, hi) if case["ctx_min"] or r.random() < 0.8 else 0)
    if case["requests"] > 4:
        new[r.randrange(case["requests"])] = 0      # a request that pauses
    return context, new


def _pairs(case):
    """Visible (query, key) pairs of a scored case, over the batch, per head."""
    sq, sk = case["seq_q"], case["seq_k"]
    docs, prefix = _documents(case), _prefixes(case)
    total = 0
    for b in range(case["batch"]):
        for start, n in _spans(docs[b]) if docs else [(0, None)]:
            p = prefix[b] if prefix else 0
            if n is None:
                if not case["causal"]:
                    total += sq * sk
                else:
                    total += sum(max(0, min(sk, max(i + sk - sq + 1, p))) for i in range(sq))
            elif not case["causal"]:
                total += n * n
            else:
                total += sum(min(n, max(i + 1, p - start)) for i in range(n))
    return total


def _spans(lengths):
    start = 0
    for n in lengths:
        yield start, n
        start += n


# ------------------------------------------------------------------------------------------------
# inputs
# ------------------------------------------------------------------------------------------------
def _ints(values, dtype=torch.int32):
    return torch.tensor(values, dtype=dtype, device=_DEV)


def _slopes(heads):
    return torch.tensor([2.0 ** (-8.0 * (i + 1) / heads) for i in range(heads)], dtype=torch.float32, device=_DEV)


def _noise(g, shape, dtype, scale=1.0):
    return (torch.randn(shape, generator=g, dtype=torch.float32, device=_DEV) * scale).to(dtype)


def prepare(case, seed):
    g = torch.Generator(device=_DEV).manual_seed(seed)
    state = {"case": case}
    if case["op"] == "scored":
        dt = _DT[case["dtype"]]
        b, sq, sk, hq, hkv, d = (case[n] for n in ("batch", "seq_q", "seq_k", "heads_q", "heads_kv", "dim"))
        state["q"] = _noise(g, (b, sq, hq, d), dt, case["sharp"])
        state["k"] = _noise(g, (b, sk, hkv, d), dt)
        state["v"] = _noise(g, (b, sk, hkv, d), dt)
        state["do"] = _noise(g, (b, sq, hq, d), dt)
        if case["train"]:
            for n in "qkv":
                state[n].requires_grad_(True)
        docs, prefix = _documents(case), _prefixes(case)
        state["document_ids"] = None
        if docs:
            ids = torch.full((b, sq), -1, dtype=torch.int32)
            for row, lengths in enumerate(docs):
                for i, (start, n) in enumerate(_spans(lengths)):
                    ids[row, start:start + n] = i
            state["document_ids"] = ids.to(_DEV)
        state["prefix_lens"] = _ints(prefix) if prefix else None
        state["alibi_slopes"] = _slopes(hq) if case["alibi"] else None
        return state
    if case["op"] == "write":
        dt = _DT[case["dtype"]]
        t, hq, hkv, d = case["tokens"] + case["spare"], case["heads_q"], case["heads_kv"], case["dim"]
        # keys and values as they come out of the joint projection: slices of its rows
        qkv = _noise(g, (t, hq + 2 * hkv, d), dt)
        state["k"], state["v"] = qkv[:, hq:hq + hkv], qkv[:, hq + hkv:]
        state["k_cache"] = _noise(g, (case["pages"], case["page"], hkv, d), dt)
        state["v_cache"] = _noise(g, (case["pages"], case["page"], hkv, d), dt)
        pages = torch.randperm(case["pages"], generator=g, device=_DEV)[:-(-case["tokens"] // case["page"])]
        slots = (pages[:, None] * case["page"] + torch.arange(case["page"], device=_DEV)).reshape(-1)[:case["tokens"]]
        state["slot_map"] = torch.cat([slots, torch.full((case["spare"],), -1, dtype=torch.int64, device=_DEV)])
        return state

    # a serving step: requests with pages in the cache, free pages, new tokens
    context, new = _requests(case)
    page, tokens = case["page"], sum(new) + case["spare"]
    have = [-(-c // page) for c in context]
    need = [-(-(c + n) // page) for c, n in zip(context, new)]
    width = max(need) + 2
    pages = sum(need) + 7
    order = torch.randperm(pages, generator=g, device=_DEV).to(torch.int32).cpu()
    table = torch.full((len(new), width), -1, dtype=torch.int32)
    at = 0
    for i, n in enumerate(have):
        table[i, :n] = order[at:at + n]
        at += n
    state.update(context_lens=_ints(context), new_lens=_ints(new), block_table=table.to(_DEV), free_pages=order[at:].to(_DEV), num_tokens=tokens)
    if case["op"] == "plan":
        return state
    dt = _DT[case["dtype"]]
    hq, hkv, d = case["heads_q"], case["heads_kv"], case["dim"]
    state["q"] = _noise(g, (tokens, hq, d), dt, case["sharp"])
    state["k_cache"] = _noise(g, (pages, page, hkv, d), dt)
    state["v_cache"] = _noise(g, (pages, page, hkv, d), dt)
    state["out"] = _noise(g, (tokens, hq, d), dt)
    state["alibi_slopes"] = _slopes(hq) if case["alibi"] else None
    # the plan is made once per step and serves the attention of every layer
    if own:
        state["plan"] = _package().paged_step_plan(state["context_lens"], state["new_lens"], state["block_table"], state["free_pages"], page_size=page,
                                                   num_tokens=tokens, heads_q=hq, heads_kv=hkv)
    else:
        state["plan"] = _plain_plan(state)
    return state


# ------------------------------------------------------------------------------------------------
# one pass
# ------------------------------------------------------------------------------------------------
def run(state):
    case = state["case"]
    op = case["op"]
    cap = case.get("cap") or None
    if op == "scored":
        if own:
            J = _package()
            out = J.scored_flash_attention(state["q"], state["k"], state["v"], causal=case["causal"], softcap=cap, alibi_slopes=state["alibi_slopes"],
                                           document_ids=state["document_ids"], prefix_lens=state["prefix_lens"])
            if not case["train"]:
                return {"out": out}
            dq, dk, dv = torch.autograd.grad(out, (state["q"], state["k"], state["v"]), state["do"])
            return {"out": out.detach(), "dq": dq, "dk": dk, "dv": dv}
        return _plain_scored(state)
    if op == "paged":
        if own:
            return {"out": _package().paged_attention(state["q"], state["k_cache"], state["v_cache"], state["plan"], softcap=cap,
                                                      alibi_slopes=state["alibi_slopes"], out=state["out"])}
        return _plain_paged(state)
    if op == "plan":
        if own:
            plan = _package().paged_step_plan(state["context_lens"], state["new_lens"], state["block_table"], state["free_pages"], page_size=case["page"],
                                              num_tokens=state["num_tokens"], heads_q=case["heads_q"], heads_kv=case["heads_kv"])
            return {"cu_seqlens": plan.cu_seqlens, "seqlens_k": plan.seqlens_k, "block_table": plan.block_table, "slot_map": plan.slot_map,
                    "positions": plan.positions, "pages_taken": plan.pages_taken}
        return _plain_plan(state)
    if own:
        _package().paged_cache_write(state["k"], state["v"], state["k_cache"], state["v_cache"], state["slot_map"])
    else:
        _plain_write(state)
    return {"k_cache": state["k_cache"], "v_cache": state["v_cache"]}


# ------------------------------------------------------------------------------------------------
# plain forms
# ------------------------------------------------------------------------------------------------
def _plain_visible(state):
    """[B, 1, Sq, Sk]: which keys a query sees."""
    case = state["case"]
    sq, sk = case["seq_q"], case["seq_k"]
    i = torch.arange(sq, device=_DEV)[:, None]
    j = torch.arange(sk, device=_DEV)[None, :]
    visible = torch.ones((case["batch"], sq, sk), dtype=torch.bool, device=_DEV)
    if case["causal"]:
        before = (j <= i + (sk - sq))[None]
        if state["prefix_lens"] is not None:
            before = before | (j[None] < state["prefix_lens"][:, None, None])
        visible = visible & before
    if state["document_ids"] is not None:
        ids = state["document_ids"]
        # a document is a run of equal ids; negative ids are padding
        run_of = torch.cat([torch.zeros_like(ids[:, :1]), (ids[:, 1:] != ids[:, :-1]).to(ids.dtype)], 1).cumsum(1)
        visible = visible & (run_of[:, :, None] == run_of[:, None, :]) & (ids >= 0)[:, :, None]
    return visible[:, None]


def _plain_scored(state):
    case = state["case"]
    dt = _DT[case["dtype"]]
    b, sq, sk, hq, hkv, d = (case[n] for n in ("batch", "seq_q", "seq_k", "heads_q", "heads_kv", "dim"))
    group, scale, cap = hq // hkv, 1.0 / math.sqrt(d), case["cap"]
    visible = _plain_visible(state)
    bias = None
    if case["alibi"]:
        i = torch.arange(sq, device=_DEV, dtype=torch.float32)[:, None]
        j = torch.arange(sk, device=_DEV, dtype=torch.float32)[None, :]
        bias = -(i + (sk - sq) - j).abs()
    out = torch.empty((b, sq, hq, d), dtype=dt, device=_DEV)
    grads = [torch.empty_like(state[n]) for n in "qkv"] if case["train"] else None
    for h in range(hkv):      # one key/value head at a time, to bound the memory of the scores
        mine = slice(h * group, (h + 1) * group)
        q = state["q"].detach()[:, :, mine].float().transpose(1, 2)
        k = state["k"].detach()[:, :, h].float()[:, None]
        v = state["v"].detach()[:, :, h].float()[:, None]
        s = (q @ k.transpose(-1, -2)) * scale
        slope = None
        if cap:
            t = torch.tanh(s / cap)
            s = cap * t
            slope = 1 - t * t
            del t
        if bias is not None:
            s = s + state["alibi_slopes"][mine][None, :, None, None] * bias
        s = torch.where(visible, s, -math.inf)
        top = s.amax(-1, keepdim=True)
        p = torch.exp(s - torch.where(top == -math.inf, 0.0, top))
        del s
        total = p.sum(-1, keepdim=True)
        p = p / torch.where(total == 0, 1.0, total)
        o = p @ v
        out[:, :, mine] = o.transpose(1, 2).to(dt)
        if grads is None:
            continue
        do = state["do"][:, :, mine].float().transpose(1, 2)
        grads[2][:, :, h] = (p.transpose(-1, -2) @ do).sum(1).to(dt)
        ds = p * (do @ v.transpose(-1, -2) - (do * o).sum(-1, keepdim=True))
        del p
        if slope is not None:
            ds = ds * slope
        ds = ds * scale
        grads[0][:, :, mine] = (ds @ k).transpose(1, 2).to(dt)
        grads[1][:, :, h] = (ds.transpose(-1, -2) @ q).sum(1).to(dt)
    if grads is None:
        return {"out": out}
    return {"out": out, "dq": grads[0], "dk": grads[1], "dv": grads[2]}


def _plain_plan(state):
    case = state["case"]
    page, tokens = case["page"], state["num_tokens"]
    context, new, table, free = (state[n] for n in ("context_lens", "new_lens", "block_table", "free_pages"))
    zero = torch.zeros((1,), dtype=torch.int32, device=_DEV)
    cu = torch.cat([zero, new.cumsum(0).to(torch.int32)])
    lens = context + new
    have = (context + page - 1) // page
    need = (lens + page - 1) // page
    first = torch.cat([zero, (need - have).cumsum(0).to(torch.int32)])
    column = torch.arange(table.shape[1], device=_DEV, dtype=torch.int32)[None]
    fresh = (column >= have[:, None]) & (column < need[:, None])
    source = (first[:-1, None] + column - have[:, None]).clamp(0, max(0, free.shape[0] - 1)).long()
    if free.shape[0]:
        table.copy_(torch.where(fresh, free[source], table))
    row = torch.arange(tokens, device=_DEV, dtype=torch.int32)
    request = (row[:, None] >= cu[None, 1:]).sum(1).clamp(max=new.shape[0] - 1)
    inside = row < cu[-1]
    position = torch.where(inside, context[request] + row - cu[request], 0).to(torch.int32)
    slot = table[request, (position // page).long()].long() * page + position % page
    slot = torch.where(inside, slot, -1)
    return {"cu_seqlens": cu, "seqlens_k": lens, "block_table": table, "slot_map": slot, "positions": position, "pages_taken": first[-1:]}


def _plain_write(state):
    hkv, d = state["k_cache"].shape[2:]
    kept = state["slot_map"] >= 0
    at = state["slot_map"][kept]
    state["k_cache"].view(-1, hkv, d)[at] = state["k"][kept]
    state["v_cache"].view(-1, hkv, d)[at] = state["v"][kept]


def _plain_paged(state):
    case, plan = state["case"], state["plan"]
    page, hq, hkv, d = (case[n] for n in ("page", "heads_q", "heads_kv", "dim"))
    group, scale, cap, dt = hq // hkv, 1.0 / math.sqrt(d), case["cap"], _DT[case["dtype"]]
    context, new = _requests(case)
    most_new, most = max(new), max(c + n for c, n in zip(context, new))
    cu, lens = plan["cu_seqlens"].long(), plan["seqlens_k"].long()
    i = torch.arange(most_new, device=_DEV)
    j = torch.arange(most, device=_DEV)
    count = cu[1:] - cu[:-1]
    rows = (cu[:-1, None] + i).clamp(max=state["num_tokens"] - 1)             # [B, N]
    real = i[None] < count[:, None]
    position = (lens - count)[:, None] + i[None]
    visible = (j[None, None] <= position[:, :, None]) & real[:, :, None]      # [B, N, L]
    kept = j[None] < lens[:, None]
    slots = plan["block_table"].long().clamp(min=0)[:, (j // page)] * page + j % page
    slots = torch.where(kept, slots, 0)
    out = state["out"]
    for h in range(hkv):      # one key/value head at a time, to bound the memory of the scores
        mine = slice(h * group, (h + 1) * group)
        k = state["k_cache"].view(-1, hkv, d)[:, h][slots].float()
        v = state["v_cache"].view(-1, hkv, d)[:, h][slots].float() * kept[:, :, None]
        q = state["q"][:, mine][rows].float()                                 # [B, N, G, D]
        s = (q.flatten(1, 2) @ k.transpose(-1, -2)).unflatten(1, (most_new, group)) * scale
        if cap:
            s = cap * torch.tanh(s / cap)
        if state["alibi_slopes"] is not None:
            far = (position[:, :, None] - j[None, None]).abs().float()
            s = s - state["alibi_slopes"][mine][None, None, :, None] * far[:, :, None]
        s = torch.where(visible[:, :, None], s, -math.inf)
        top = s.amax(-1, keepdim=True)
        p = torch.exp(s - torch.where(top == -math.inf, 0.0, top))
        total = p.sum(-1, keepdim=True)
        o = (p.flatten(1, 2) @ v).unflatten(1, (most_new, group)) / torch.where(total == 0, 1.0, total)
        out[rows[real][:, None], torch.arange(h * group, (h + 1) * group, device=_DEV)[None]] = o[real].to(dt)
    return {"out": out}


# ------------------------------------------------------------------------------------------------
# work
# ------------------------------------------------------------------------------------------------
def work(case):
    op = case["op"]
    if op == "scored":
        d, hq, hkv, b = case["dim"], case["heads_q"], case["heads_kv"], case["batch"]
        forward = 4.0 * _pairs(case) * hq * d
        q, kv = 2.0 * b * case["seq_q"] * hq * d, 2.0 * b * case["seq_k"] * hkv * d
        if not case["train"]:
            return {"bytes": 2 * q + 2 * kv, "flops": forward}
        return {"bytes": 4 * q + 4 * kv, "flops": 3.5 * forward}
    if op == "write":
        row = 2.0 * case["heads_kv"] * case["dim"]
        return {"bytes": 4.0 * case["tokens"] * row + 8.0 * (case["tokens"] + case["spare"]), "flops": 0.0}
    context, new = _requests(case)
    tokens = sum(new) + case["spare"]
    fresh = sum(-(-(c + n) // case["page"]) - -(-c // case["page"]) for c, n in zip(context, new))
    used = sum(-(-(c + n) // case["page"]) for c, n in zip(context, new) if n)
    if op == "plan":
        return {"bytes": 4.0 * 4 * len(new) + 8.0 * fresh + 12.0 * tokens, "flops": 0.0}
    d, hq, hkv = case["dim"], case["heads_q"], case["heads_kv"]
    pairs = sum(n * c + n * (n + 1) / 2.0 for c, n in zip(context, new))
    keys = sum(c + n for c, n in zip(context, new) if n)
    return {"bytes": 4.0 * keys * hkv * d + 4.0 * sum(new) * hq * d + 4.0 * used, "flops": 4.0 * pairs * hq * d}


# ------------------------------------------------------------------------------------------------
# the definitions in float64
# ------------------------------------------------------------------------------------------------
def _exact_attention(q, k, v, allowed, slope, distance, cap):
    """[n, D] of one head: q [n, D], k and v [m, D], allowed [n, m]."""
    score = q @ k.T / math.sqrt(q.shape[1])
    if cap:
        score = cap * torch.tanh(score / cap)
    if slope is not None:
        score = score - slope * distance
    score = score.masked_fill(~allowed, -math.inf)
    seen = allowed.any(1)
    weight = torch.zeros_like(score)
    weight[seen] = torch.softmax(score[seen], 1)
    return weight @ v


def exact(case, seed):
    state = prepare(case, seed)
    op = case["op"]
    if op == "scored":
        # gradients come from automatic differentiation, head by head
        sq, sk, hq, hkv = (case[n] for n in ("seq_q", "seq_k", "heads_q", "heads_kv"))
        docs, prefix = _documents(case), _prefixes(case)
        row, column = torch.arange(sq, device=_DEV)[:, None] + (sk - sq), torch.arange(sk, device=_DEV)[None]
        leaves = {n: state[n].detach().double() for n in "qkv"}
        out = torch.zeros_like(leaves["q"])
        grad = {n: torch.zeros_like(x) for n, x in leaves.items()}
        for b in range(case["batch"]):
            allowed = torch.ones((sq, sk), dtype=torch.bool, device=_DEV)
            if case["causal"]:
                allowed = column <= row
                if prefix:
                    allowed = allowed | (column < prefix[b])
            if docs:
                same = torch.zeros((sq, sk), dtype=torch.bool, device=_DEV)
                for start, n in _spans(docs[b]):
                    same[start:start + n, start:start + n] = True
                allowed = allowed & same
            for h in range(hq):
                hk = h // (hq // hkv)
                q, k, v = (x.clone().requires_grad_(case["train"]) for x in (leaves["q"][b, :, h], leaves["k"][b, :, hk], leaves["v"][b, :, hk]))
                slope = 2.0 ** (-8.0 * (h + 1) / hq) if case["alibi"] else None
                o = _exact_attention(q, k, v, allowed, slope, (row - column).abs().double() if case["alibi"] else None, case["cap"])
                out[b, :, h] = o.detach()
                if case["train"]:
                    gq, gk, gv = torch.autograd.grad(o, (q, k, v), state["do"][b, :, h].double())
                    grad["q"][b, :, h] += gq
                    grad["k"][b, :, hk] += gk
                    grad["v"][b, :, hk] += gv
        if not case["train"]:
            return {"out": out}
        return {"out": out, "dq": grad["q"], "dk": grad["k"], "dv": grad["v"]}
    if op == "write":
        caches = {}
        for n in ("k", "v"):
            cache = state[n + "_cache"].double()
            page = case["page"]
            for start in range(0, case["tokens"], page):      # a page's tokens lie one behind the other
                at = int(state["slot_map"][start])
                stop = min(start + page, case["tokens"])
                cache[at // page, :stop - start] = state[n][start:stop].double()
            caches[n + "_cache"] = cache
        return caches
    if op == "plan":
        return None
    context, new = _requests(case)
    page, hq, hkv, cap = case["page"], case["heads_q"], case["heads_kv"], case["cap"]
    table = state["block_table"].cpu().tolist()
    out = state["out"].double()
    at = 0
    for r, (c, n) in enumerate(zip(context, new)):
        if not n:
            continue
        pages = torch.tensor(table[r][:-(-(c + n) // page)], device=_DEV)
        keys = state["k_cache"][pages].flatten(0, 1)[:c + n].double()
        values = state["v_cache"][pages].flatten(0, 1)[:c + n].double()
        row, column = torch.arange(c, c + n, device=_DEV)[:, None], torch.arange(c + n, device=_DEV)[None]
        for h in range(hq):
            hk = h // (hq // hkv)
            slope = 2.0 ** (-8.0 * (h + 1) / hq) if case["alibi"] else None
            out[at:at + n, h] = _exact_attention(state["q"][at:at + n, h].double(), keys[:, hk], values[:, hk], column <= row, slope,
                                                 (row - column).double() if case["alibi"] else None, cap)
        at += n
    return {"out": out}
