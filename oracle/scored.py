"""TEST INFRASTRUCTURE ONLY — attention with changed scores in float64, and how far a kernel may be from it.

`attention` computes output, log-sum-exp and gradients densely from the formulas. `bounds` adds up the roundings a
kernel with 16-bit operands makes on the way, worst case, entry by entry (u: half a step of the 16-bit type):
  P is rounded to 16 bits before P V and P^T dO                       err(P)  = u P (+ 2^-25: fp16 subnormals)
  out is rounded once                                                 err(o)  = err(P) |V| + u |o|
  delta = rowsum(dO * out) uses the rounded out                       err(dl) = sum |dO| err(o)
  dS = P g (dP - delta): P (or P g) is rounded, then dS               err(dS) = 2 u |dS| + P g err(dl) (+ subnormals)
  a capped score's g = 1 - t^2 in float32 with t = 1 - 2 r, r a reciprocal off by at most 2^-23 and the difference by
  2^-24: err(t) <= 2^-22 + 2^-24, err(g) <= 2 err(t) + 2^-24 < 2^-20, and P err(g) |dP - delta| of it reaches dS
  dq, dk, dv are rounded once
`slack` covers what float32 loses inside the exponent (products of D terms, the cap's exponential and reciprocal,
a distance times a slope), as a relative change of P.

Only tests may import this module.
"""
from __future__ import annotations

import math

import torch


def visible_keys(batch, sq, sk, causal=False, document_ids=None, prefix_lens=None):
    """bool [B, Sq, Sk], built token by token."""
    seen = torch.zeros(batch, sq, sk, dtype=torch.bool)
    for b in range(batch):
        ids = None if document_ids is None else document_ids[b].tolist()
        prefix = 0 if prefix_lens is None else int(prefix_lens[b])
        for i in range(sq):
            lo, hi = 0, sk
            if ids is not None:
                if ids[i] < 0:
                    continue
                lo = hi = i
                while lo > 0 and ids[lo - 1] == ids[i]:
                    lo -= 1
                while hi < sk and ids[hi] == ids[i]:
                    hi += 1
            if causal:
                hi = min(hi, max(i + sk - sq + 1, prefix))
            if hi > lo:
                seen[b, i, lo:hi] = True
    return seen


def attention(q, k, v, seen, softmax_scale=None, softcap=None, alibi_slopes=None, dO=None):
    """q [B,Sq,Hq,D], k/v [B,Sk,Hkv,D], seen [B,Sq,Sk]. Returns a dict: out, lse [B,Hq,Sq], and with dO also dq, dk,
    dv and what `bounds` needs, all float64."""
    B, Sq, Hq, D = q.shape
    Sk, Hkv = k.shape[1], k.shape[2]
    G = Hq // Hkv
    scale = 1.0 / math.sqrt(D) if softmax_scale is None else softmax_scale
    qd = q.double().permute(0, 2, 1, 3)
    kd = k.double().permute(0, 2, 1, 3).repeat_interleave(G, dim=1)
    vd = v.double().permute(0, 2, 1, 3).repeat_interleave(G, dim=1)
    s = (qd @ kd.transpose(-1, -2)) * scale
    g = torch.ones_like(s)
    if softcap:
        # the derivative 1 - tanh(z)^2 = 4 e^(-2|z|) / (1 + e^(-2|z|))^2, without the cancellation of the first form
        e = torch.exp(-2 * (s / softcap).abs())
        s, g = softcap * torch.tanh(s / softcap), 4 * e / (1 + e) ** 2
    if alibi_slopes is not None:
        dist = (torch.arange(Sq, dtype=torch.float64)[:, None] + (Sk - Sq) - torch.arange(Sk, dtype=torch.float64)[None]).abs()
        s = s - alibi_slopes.double()[None, :, None, None] * dist
    s = s.masked_fill(~seen[:, None], -math.inf)
    lse = torch.logsumexp(s, dim=-1)
    dead = lse == -math.inf
    p = torch.exp(s - lse.masked_fill(dead, 0.0)[..., None])
    o = p @ vd
    r = dict(out=o.permute(0, 2, 1, 3), lse=lse, p=p, v=vd, o=o)
    if dO is not None:
        do = dO.double().permute(0, 2, 1, 3)
        delta = (do * o).sum(-1, keepdim=True)
        inner = do @ vd.transpose(-1, -2) - delta
        ds = p * g * inner
        groups = lambda x: x.view(B, Hkv, G, Sk, D).sum(2).permute(0, 2, 1, 3)
        r.update(dq=(scale * (ds @ kd)).permute(0, 2, 1, 3), dk=groups(scale * (ds.transpose(-1, -2) @ qd)),
                 dv=groups(p.transpose(-1, -2) @ do), ds=ds, pg=p * g, do=do, inner=inner, capped=bool(softcap), q=qd, k=kd, scale=scale, shape=(B, Hkv, G, Sk, D))
    return r


def bounds(r, dtype, slack=5e-4):
    """Largest errors of out, dq, dk, dv (those that `r` holds), in their shapes."""
    u = torch.finfo(dtype).eps / 2
    tiny = 2.0 ** -25 if dtype == torch.float16 else 0.0
    err_p = (u + slack) * r["p"] + tiny * (r["p"] > 0)
    err_o = err_p @ r["v"].abs() + u * r["o"].abs()
    b = dict(out=err_o.permute(0, 2, 1, 3))
    if "ds" in r:
        B, Hkv, G, Sk, D = r["shape"]
        groups = lambda x: x.view(B, Hkv, G, Sk, D).sum(2).permute(0, 2, 1, 3)
        do = r["do"].abs()
        err_delta = (do * err_o).sum(-1, keepdim=True)
        # the change of P by the float32 exponent enters dS as a factor too; dP and delta are float32 sums
        size = do @ r["v"].abs().transpose(-1, -2) + (do * r["o"].abs()).sum(-1, keepdim=True)
        err_ds = (2 * u + slack) * r["ds"].abs() + r["pg"] * (err_delta + 1e-5 * size)
        if r["capped"]:
            err_ds = err_ds + 2.0 ** -20 * r["p"] * r["inner"].abs()
        if tiny:
            err_ds = err_ds + tiny * size * (r["p"] > 0) + tiny * 2 * do.max() * (r["p"] > 0)
        b["dq"] = (r["scale"] * (err_ds @ r["k"].abs())).permute(0, 2, 1, 3) + u * r["dq"].abs()
        b["dk"] = groups(r["scale"] * (err_ds.transpose(-1, -2) @ r["q"].abs())) + u * r["dk"].abs()
        b["dv"] = groups(err_p.transpose(-1, -2) @ do) + u * r["dv"].abs()
    # values whose own size is below the 16-bit type's smallest step
    return {n: x * 1.01 + (2.0 ** -24 if dtype == torch.float16 else 0.0) for n, x in b.items()}


def worst(mine, want, bound):
    """Largest |mine - want| / bound (0/0 counts as 0; more than 1 is a failure)."""
    err = (mine.double().cpu() - want).abs()
    if not torch.isfinite(mine.float()).all():
        return math.inf
    return torch.where(err == 0, torch.zeros_like(err), err / bound.clamp(min=1e-300)).max().item()
