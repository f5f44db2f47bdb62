"""Attention over 4-bit pages in 64 bits, with what each of its two kernels may be off by, whatever the sizes.

Let t be a row's scores, p its weights (softmax of t), v = s code + z a value of a group with scale s.  Roundings
are at most half a step: 2^-11 of a number in 16 bits (2^-25 below 2^-14), 2^-24 of one in 32.

Scores: d bounds the error of any t.  The matrix unit's and the fp32 sums over D elements take at most 2^-21 of
their terms' sizes, |scale| sum |q| (s code + |z|); the exponential and its argument 2^-21 (1 + |t|).  Weights and
their sum are then off by a factor of e^d each, the output by less than 2.1 d sum p |v| while d is below 0.05.

Row blocks: queries as they are (those of 32 bits to 11 bits), elements far below the row's largest to 2^-34 of
it.  The weight times s is rounded to 11 bits and multiplies code - 8, at most 8; below 2^-14 of its unit it is off by
2^-25 of that.  The unit is a power of two, at most twice the largest such product of the row and group (it may lag
2^10 behind it): 8 * 2^-24 of the largest product, for each of n keys.  Everything else is fp32: a sum of n / 16 terms and 64 more takes (n / 16 + 64) 2^-24 of its terms.

Prompts: K times 16 and V times 64 are held in 16 bits (where the scales are float16, as they are), the queries
times 2^8 and the scale's power of two; K and V are off by 2^-11 and 2^-29 or 2^-31, queries by 2^-32 of a score
per unit of K (and 2^-11 where they have 32 bits), weights by 2^-11, or 2^-25 of the row's largest.
"""

import torch

from u4_reference import GROUP, values64


def attention(q, kp, vp, ks, vs, bt, cl, ps, scale=None, causal=True):
    """(out, what row blocks may be off by, what prompts may be off by), each [B, Hq, L, D] in 64 bits."""
    B, Hq, L, D = q.shape
    Hkv, g = kp.shape[1], Hq // kp.shape[1]
    scale = D ** -0.5 if scale is None else scale
    out = torch.zeros(B, Hq, L, D, dtype=torch.float64, device=q.device)
    rows, prompts = torch.zeros_like(out), torch.zeros_like(out)
    for b in range(B):
        n = min(int(cl[b]), bt.shape[1] * ps)
        if n <= 0:
            continue
        key = torch.arange(n, device=q.device)
        page = bt[b].long()[key // ps]
        there = (page >= 0) & (page < kp.shape[0])
        page = page.clamp(0, kp.shape[0] - 1)
        pos = torch.arange(L, device=q.device)[:, None] + int(cl[b]) - L
        seen = there[None] & ((key[None] <= pos) if causal else torch.ones(L, n, dtype=torch.bool, device=q.device))
        any_row = seen.any(0)
        for h in range(Hkv):
            held = [x[page, h, key % ps].clone() for x in (kp, ks, vp, vs)]
            for x in held:
                x[~any_row] = 0
            k, v = values64(*held[:2]), values64(*held[2:])
            wide = lambda x: x.repeat_interleave(GROUP, -1)  # noqa: E731
            ksz, vsz = held[1].double().unflatten(-1, (-1, 2)), held[3].double().unflatten(-1, (-1, 2))
            sk, zk, sv, zv = wide(ksz[..., 0]), wide(ksz[..., 1]), wide(vsz[..., 0]), wide(vsz[..., 1])
            off_k = (k - zk).abs() + zk.abs()  # s code + |z|
            off_v = (v - zv).abs() + zv.abs() + 8 * sv
            for hq in range(h * g, (h + 1) * g):
                x = q[b, hq].double()
                t = ((x @ k.T) * scale).masked_fill(~seen, float("-inf"))
                top = t.amax(-1, keepdim=True)
                p = torch.exp(t - top.masked_fill(top.isinf(), 0))
                total = p.sum(-1, keepdim=True)
                p = p / total.masked_fill(total == 0, 1)
                out[b, hq] = p @ v
                common = 2.0 ** -21 * (abs(scale) * (x.abs() @ off_k.T) + 1 + t.masked_fill(~seen, 0).abs())
                plain = abs(scale) * (x.abs() @ k.abs().T)
                thin = 2.0 ** -11 * plain if q.dtype == torch.float32 else 0 * plain
                d = common + thin + 2.0 ** -34 * abs(scale) * x.abs().amax(-1, keepdim=True) * k.abs().sum(-1)
                d = d.masked_fill(~seen, 0).amax(-1, keepdim=True)
                sums = (n / 16 + 64) * 2.0 ** -24
                held_to = torch.einsum("ln,nd->lnd", p, sv).amax(1)
                rows[b, hq] = (2.1 * d + sums) * (p @ off_v) + 2.0 ** -11 * (p @ (v - zv - 8 * sv).abs()) + 2.0 ** -21 * n * held_to
                d = common + thin + 2.0 ** -11 * plain + 2.0 ** -29 * abs(scale) * x.abs().sum(-1, keepdim=True) + 2.0 ** -32 * k.abs().sum(-1)
                d = d.masked_fill(~seen, 0).amax(-1, keepdim=True)
                lost = 2.0 ** -25 * (seen.double() @ v.abs()) + 2.0 ** -31
                prompts[b, hq] = (2.1 * d + sums + 2.0 ** -10) * (p @ v.abs()) + lost
    return out, rows, prompts


def close(got, want, bound, what=""):
    half = torch.finfo(got.dtype).eps / 2
    tol = bound + (want.abs() + bound) * half * 1.001 + torch.finfo(got.dtype).smallest_normal * half
    off = (got.double() - want).abs()
    assert not got.isnan().any(), f"{what}: NaN"
    assert (off <= tol).all(), f"{what}: {(off / tol).max().item():.3g} times the bound"
