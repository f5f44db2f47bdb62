"""64-bit references of the bounded-cache operators and random problems for their tests."""

from __future__ import annotations

import math

import torch

HALF_STEP = {torch.float32: 2.0 ** -24, torch.bfloat16: 2.0 ** -8, torch.float16: 2.0 ** -11}


def make_problem(seed, ctx, L, Hq, Hkv, D, ps, kv_dtype, q_dtype=None, spare=2, width_extra=1, holes=()):
    """Pools with a random page order; ctx is a list of context lengths, holes (b, page) pairs
    unmapped after the pages were handed out."""
    gen = torch.Generator().manual_seed(seed)
    B = len(ctx)
    pages = [(c + ps - 1) // ps for c in ctx]
    P = sum(pages) + spare
    order = torch.randperm(P, generator=gen)
    bt = torch.full((B, max(pages + [0]) + width_extra), -1, dtype=torch.int32)
    at = 0
    for b, n in enumerate(pages):
        bt[b, :n] = order[at:at + n].int()
        at += n
    for b, j in holes:
        bt[b, j] = -1
    if kv_dtype == torch.int8:
        k = torch.randint(-127, 128, (P, Hkv, ps, D), generator=gen, dtype=torch.int8)
        v = torch.randint(-127, 128, (P, Hkv, ps, D), generator=gen, dtype=torch.int8)
        sd = q_dtype if q_dtype in (torch.float16, torch.bfloat16) else torch.float16
        ks = ((torch.rand(P, Hkv, ps, 1, generator=gen) + 0.5) * (2 / 127)).to(sd)
        vs = ((torch.rand(P, Hkv, ps, 1, generator=gen) + 0.5) * (2 / 127)).to(sd)
    else:
        k = torch.randn(P, Hkv, ps, D, generator=gen).to(kv_dtype)
        v = torch.randn(P, Hkv, ps, D, generator=gen).to(kv_dtype)
        ks = vs = None
    qd = q_dtype or (torch.float16 if kv_dtype == torch.int8 else kv_dtype)
    q = (1.5 * torch.randn(B, Hq, L, D, generator=gen)).to(qd)
    return {"q": q, "k": k, "v": v, "ks": ks, "vs": vs, "bt": bt, "cl": torch.tensor(ctx, dtype=torch.int32), "ps": ps}


def to_gpu(prob):
    return {n: x.cuda() if isinstance(x, torch.Tensor) else x for n, x in prob.items()}


def visible(n, limit, L, window, sinks, causal=True):
    """[L, limit] truth values: does row l of a context of n tokens see key j < limit."""
    pos = torch.arange(n - L, n)[:, None]
    j = torch.arange(limit)[None, :]
    ok = torch.ones(L, limit, dtype=torch.bool)
    if causal:
        ok &= j <= pos
    if window:
        ok &= (j < sinks) | (j > pos - window)
    return ok


def dense_rows(prob, b, limit):
    """K, V of request b's first `limit` tokens in 64 bits [Hkv, limit, D], and which are mapped."""
    ps, P = prob["ps"], prob["k"].shape[0]
    j = torch.arange(limit)
    page = prob["bt"][b].long()[j // ps] if limit else j
    mapped = (page >= 0) & (page < P)
    page = page.clamp(0, P - 1)
    out = []
    for x, s in (("k", "ks"), ("v", "vs")):
        rows = prob[x][page, :, j % ps].double().transpose(0, 1)
        if prob[s] is not None:
            rows = rows * prob[s][page, :, j % ps].double().transpose(0, 1)
        out.append(rows)
    return out[0], out[1], mapped


def _attend(q, k, v, ok, scale):
    """One (request, kv head): q [g, L, D], k/v [n, D], ok [L, n] -> out, weights, and what bounds
    the result of 32-bit arithmetic: sum of w |v|, and the largest sum of |q k| of a row."""
    z = torch.einsum("gld,nd->gln", q, k) * scale
    z = torch.where(ok, z, torch.full_like(z, -math.inf))
    top = z.amax(-1, keepdim=True) if z.shape[-1] else torch.zeros(*z.shape[:2], 1, dtype=z.dtype)
    top = torch.where(top == -math.inf, torch.zeros_like(top), top)
    e = torch.exp(z - top)
    total = e.sum(-1, keepdim=True)
    w = e / torch.where(total == 0, torch.ones_like(total), total)
    mag = torch.einsum("gld,nd->gln", q.abs(), k.abs()) * abs(scale)
    mag = torch.where(ok, mag, torch.zeros_like(mag)).amax(-1) if z.shape[-1] else torch.zeros(z.shape[:2], dtype=z.dtype)
    # the largest weight times sum |v| over the seen keys: what a fixed absolute error of e costs
    tail = (w.amax(-1) if z.shape[-1] else torch.zeros_like(mag))[..., None] * torch.einsum("ln,nd->ld", ok.double(), v.abs())
    return torch.einsum("gln,nd->gld", w, v), w, torch.einsum("gln,nd->gld", w, v.abs()), mag, tail


def paged_reference(prob, window=0, sinks=0, causal=True, mass=None, scale=None):
    """(out, its 32-bit error terms, mass, its error terms) of the windowed / scored operator."""
    B, Hq, L, D = prob["q"].shape
    Hkv, ps = prob["k"].shape[1], prob["ps"]
    g, scale = Hq // Hkv, scale if scale is not None else D ** -0.5
    cap = prob["bt"].shape[1] * ps
    out = torch.zeros(B, Hq, L, D, dtype=torch.float64)
    spread = torch.zeros_like(out)
    tails = torch.zeros_like(out)
    logit = torch.zeros(B, Hq, L, dtype=torch.float64)
    m = mass.double().clone() if mass is not None else None
    m_err = torch.zeros_like(m) if mass is not None else None
    for b in range(B):
        n = int(prob["cl"][b])
        limit = max(0, min(n, cap))
        k, v, mapped = dense_rows(prob, b, limit)
        ok = visible(n, limit, L, window, sinks, causal) & mapped
        any_row = ok.any(0)
        k = torch.where(any_row[None, :, None], k, torch.zeros_like(k))  # unseen keys may hold anything
        v = torch.where(any_row[None, :, None], v, torch.zeros_like(v))
        for h in range(Hkv):
            rows = slice(h * g, h * g + g)
            o, w, a, mag, tail = _attend(prob["q"][b, rows].double(), k[h], v[h], ok, scale)
            out[b, rows], spread[b, rows], logit[b, rows], tails[b, rows] = o, a, mag, tail
            if m is not None:
                end = min(limit, m.shape[2])
                j = torch.arange(end)
                m[b, h, :end] = torch.where(j < n - L, m[b, h, :end], torch.zeros(end, dtype=torch.float64))
                gain = w.sum((0, 1))[:end]
                m[b, h, :end] += gain
                delta = score_error(mag, D)
                m_err[b, h, :end] = 2 * delta.amax() * gain + 2.0 ** -22 * m[b, h, :end].abs() if mag.numel() else 0
    return out, (spread, logit, tails), m, m_err


def score_error(mag, D):
    """Relative error of a softmax weight from 32-bit scores: the dot product of D terms is off
    by at most (D + 8) 2^-24 sum |q k| (accumulation in any order, the scaling and the log2 e
    factor), 2^z by 2^-21 more, and the denominator by as much."""
    return 2 * ((D + 8) * 2.0 ** -24 * mag + 2.0 ** -21)


def out_bound(ref, terms, D, kv_dtype, out_dtype, q_dtype=None):
    """Bound on |got - ref|: weights enter the product with V in 16 bits (one rounding of half a
    step each; two for int8 pages, whose values are scaled in 16 bits), the 32-bit score error,
    and the result's own rounding."""
    spread, logit, tails = terms
    u = {torch.float32: 0.0, torch.bfloat16: HALF_STEP[torch.bfloat16], torch.float16: HALF_STEP[torch.float16],
         torch.int8: 2 * HALF_STEP[torch.float16]}[kv_dtype]
    delta = score_error(logit, D)[..., None]
    # e = 2^(z - max) in half is off by at most 2^-25 where it is below half's normal range
    floor = 2.0 ** -25 * tails if kv_dtype in (torch.float16, torch.int8) else 0.0
    return spread * (2 * u + 2 * delta) + HALF_STEP[out_dtype] * ref.abs() + floor + 1e-30


def assert_within(got, ref, bound, what=""):
    g = got.detach().double().cpu()
    assert torch.isfinite(g).all(), f"{what}: values that are not finite"
    off = (g - ref).abs()
    bad = off > bound
    assert not bad.any(), f"{what}: {int(bad.sum())} values off, worst {float((off / bound.clamp(min=1e-30)).max()):.3g} of the bound"


def evict_reference(prob, mass, budget, sinks, recent, refcount=None):
    """keep_index, kept, dropped, mass, and the new pools, one request and head at a time."""
    B, Hkv, S = mass.shape
    ps, P = prob["ps"], prob["k"].shape[0]
    keep = torch.full((B, Hkv, budget), -1, dtype=torch.int32)
    kept, dropped = prob["cl"].clone(), torch.zeros(B, dtype=torch.int32)
    new = {x: prob[x].clone() for x in ("k", "v", "ks", "vs") if prob[x] is not None}
    m = mass.clone()
    bad = False
    cap = prob["bt"].shape[1] * ps
    for b in range(B):
        n = int(prob["cl"][b])
        pages = prob["bt"][b].tolist()
        refuse = n < 0 or n > min(S, cap)
        if not refuse and n > budget:
            for i in range(sinks // ps, (n - 1) // ps + 1):
                if not 0 <= pages[i] < P or (refcount is not None and int(refcount[pages[i]]) != 1):
                    refuse = True
        if refuse:
            bad = True
            continue
        if n <= budget:
            keep[b, :, :n] = torch.arange(n, dtype=torch.int32)
            continue
        kept[b], dropped[b] = budget, n - budget
        for h in range(Hkv):
            w = [(1, 0.0) if math.isnan(x) else (0, -x) for x in mass[b, h, :n].tolist()]  # NaN below every number
            middle = sorted(range(sinks, n - recent), key=lambda i: (w[i], i))[:budget - sinks - recent]
            order = list(range(sinks)) + sorted(middle) + list(range(n - recent, n))
            keep[b, h] = torch.tensor(order, dtype=torch.int32)
            m[b, h, :budget] = mass[b, h, order]
            m[b, h, budget:n] = 0
            for to, src in enumerate(order):
                for x in new if to != src else ():
                    new[x][pages[to // ps], h, to % ps] = prob[x][pages[src // ps], h, src % ps]
    return keep, kept, dropped, m, new, bad
