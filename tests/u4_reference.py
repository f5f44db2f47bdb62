"""The 4-bit cache restated for the tests: the row format in numpy fp32 (IEEE), attention in 64 bits
with the bound on its error.

A row's groups of 64 elements have a scale s and an offset z of a 16-bit type T:
z = min rounded toward -inf to T, s = fl((max - z) / 15) rounded toward +inf to T,
code = clip(rint(fl(fl(x - z) / s)), 0, 15) (0 where s = 0), value = fl(s * code + z).
"""

import numpy as np
import torch

GROUP = 64


def toward(x: np.ndarray, dtype: torch.dtype, up: bool) -> np.ndarray:
    """fp32 numbers rounded to the next one of a 16-bit type, as fp32."""
    near = torch.from_numpy(np.ascontiguousarray(x)).to(dtype)
    bits = near.view(torch.int16).numpy().astype(np.int32) & 0xFFFF
    key = np.where(bits & 0x8000, -(bits & 0x7FFF), bits)  # in the numbers' order
    v = near.float().numpy()
    key = np.where(up & (v < x), key + 1, np.where((not up) & (v > x), key - 1, key))
    bits = np.where(key < 0, -key | 0x8000, key).astype(np.uint16).view(np.int16)
    return torch.from_numpy(bits).view(dtype).float().numpy()


def quantise(x: torch.Tensor, dtype: torch.dtype):
    """Rows [..., D] -> (codes uint8 [..., D], s, z fp32 [..., D/64] holding values of dtype)."""
    g = x.detach().float().cpu().numpy()
    g = g.reshape(*g.shape[:-1], -1, GROUP)
    with np.errstate(all="ignore"):
        z = toward(g.min(-1), dtype, False)
        s = toward((g.max(-1) - z) / np.float32(15), dtype, True)
        bad = ~(np.isfinite(g).all(-1) & np.isfinite(s) & np.isfinite(z))
        z, s = np.where(bad, np.float32(np.nan), z), np.where(bad, np.float32(np.nan), s)
        q = np.rint((g - z[..., None]) / s[..., None])
    codes = np.where((s[..., None] > 0) & ~bad[..., None], np.clip(q, 0, 15), 0).astype(np.uint8)
    return codes.reshape(*x.shape), s.astype(np.float32), z.astype(np.float32)


def pack(codes: np.ndarray, s: np.ndarray, z: np.ndarray, dtype: torch.dtype):
    """-> (uint8 [..., D/2], dtype [..., 2 D/64]) as the pools hold them."""
    packed = torch.from_numpy(codes[..., 0::2] | codes[..., 1::2] << 4)
    scales = torch.from_numpy(np.stack([s, z], -1).reshape(*s.shape[:-1], -1)).to(dtype)
    return packed, scales


def values64(packed: torch.Tensor, scales: torch.Tensor) -> torch.Tensor:
    """The numbers that rows stand for, in 64 bits (codes [..., D/2], scales [..., 2 D/64])."""
    codes = torch.stack([packed & 15, packed >> 4], -1).flatten(-2).double().unflatten(-1, (-1, GROUP))
    sz = scales.double().unflatten(-1, (-1, 2))
    return (codes * sz[..., :1] + sz[..., 1:]).flatten(-2)


def parts64(packed, scales):
    """(s * code, s, |z|, s * |code - 8|) of every element, for the error bound."""
    codes = torch.stack([packed & 15, packed >> 4], -1).flatten(-2).double().unflatten(-1, (-1, GROUP))
    sz = scales.double().unflatten(-1, (-1, 2))
    one = torch.ones_like(codes)
    return (codes * sz[..., :1]).flatten(-2), (one * sz[..., :1]).flatten(-2), (one * sz[..., 1:].abs()).flatten(-2), \
        ((codes - 8).abs() * sz[..., :1]).flatten(-2)


def unpacked(rows, D, ps, scale):
    """Whether a call of so many query rows a kv head goes through unpacked pages."""
    return rows >= 256 and D == 128 and ps % 16 == 0 and scale > 0


def attend64(q, kp, vp, ks, vs, bt, cl, ps, scale=None, causal=True):
    """(out, bound): attention in 64 bits, request by request, and how far an fp32 result may be off.

    The bound counts, per output element: the weight times the value's scale held in 16 bits with 11,
    which multiplies the code less 8 (weight * (offset + 8 scale) is summed in fp32, and the sum of the
    rounded weights taken out 8 times): 2^-11 of weight * s * |code - 8|; the score held in fp32 (the matrix unit adds codes raised by 64, so
    2^-22 of sum |q| (64 + code) s and of |q| |z|, 2^-22 for the exponential) which moves weight and
    normaliser, and q held in 11 bits where it is fp32.  Rounding to the output type is the caller's.

    Calls of many rows (``unpacked``) hold K and V in f16, brought below 32 by a power of two: 2^-12 of a
    value, or 2^-25 of a unit below the normals, that is 2^-29 of the largest value; q likewise where it
    was not f16 (2^-25 of a unit against values below 32); weights are rounded to 11 bits against V itself."""
    B, Hq, L, D = q.shape
    Hkv = kp.shape[1]
    scale = D ** -0.5 if scale is None else scale
    many = unpacked(Hq // Hkv * L, D, ps, scale)
    out = torch.zeros(B, Hq, L, D, dtype=torch.float64, device=q.device)
    bound = torch.zeros_like(out)
    for b in range(B):
        n = min(int(cl[b]), bt.shape[1] * ps)
        if n <= 0:
            continue
        key = torch.arange(n, device=q.device)
        page = bt[b].long()[key // ps]
        there = (page >= 0) & (page < kp.shape[0])
        page = page.clamp(0, kp.shape[0] - 1)
        pos = torch.arange(L, device=q.device)[:, None] + int(cl[b]) - L
        seen = there[None] & (key[None] <= pos if causal else torch.ones(L, n, dtype=torch.bool, device=q.device))
        any_row = seen.any(0)
        for h in range(Hkv):
            rows = [t[page, h, key % ps].clone() for t in (kp, ks, vp, vs)]
            for r in rows:
                r[~any_row] = 0
            k, v = values64(*rows[:2]), values64(*rows[2:])
            sc_k, s_k, z_k, _ = parts64(*rows[:2])
            sc_v, s_v, z_v, off_v = parts64(*rows[2:])
            for hq in range(h * (Hq // Hkv), (h + 1) * (Hq // Hkv)):
                x = q[b, hq].double()
                t = (x @ k.T) * scale
                t = t.masked_fill(~seen, float("-inf"))
                top = t.amax(-1, keepdim=True)
                p = torch.exp(t - torch.where(top.isinf(), torch.zeros_like(top), top))
                total = p.sum(-1, keepdim=True)
                p = p / torch.where(total == 0, torch.ones_like(total), total)
                out[b, hq] = p @ v
                d = 2.0 ** -22 * abs(scale) * (x.abs() @ (64 * s_k + sc_k + z_k).T) + 2.0 ** -22 * (1 + t.abs())
                if q.dtype == torch.float32:
                    d = d + 2.0 ** -11 * abs(scale) * (x.abs() @ k.abs().T)
                if many:
                    d = d + abs(scale) * (2.0 ** -12 * (x.abs() @ k.abs().T) + 2.0 ** -29 * k.abs().max() * x.abs().sum(-1, keepdim=True))
                    if not (q.dtype == ks.dtype == torch.float16):
                        d = d + 2.0 ** -25 * 32 * D
                d = d.masked_fill(~seen, 0).amax(-1, keepdim=True)
                if many:
                    bound[b, hq] = (2.0 ** -11 + 2.0 ** -12) * (p @ v.abs()) + 2.0 ** -29 * v.abs().max()
                bound[b, hq] += 2.0 ** -11 * (p @ off_v) + (2 * d + 2.0 ** -20) * (p @ (64 * s_v + sc_v + z_v))
    return out, bound


def random_pools(gen, P, Hkv, ps, D, dtype, device="cuda"):
    """Pools as quantised unit normals leave them, about: even codes, scales and offsets that differ by row."""
    def one():
        codes = torch.randint(0, 256, (P, Hkv, ps, D // 2), generator=gen, dtype=torch.uint8)
        s = (torch.rand(P, Hkv, ps, D // GROUP, generator=gen) + 0.5) * 0.22
        z = -7.5 * s + 0.3 * torch.randn(s.shape, generator=gen)
        return codes.to(device), torch.stack([s, z], -1).flatten(-2).to(dtype).to(device)
    kp, ks = one()
    vp, vs = one()
    return kp, vp, ks, vs


def random_table(gen, lens, ps, holes=False, device="cuda", spare=3, width=None):
    pages = [(int(n) + ps - 1) // ps for n in lens]
    MP = max(max(pages), 1) if width is None else width
    P = sum(pages) + spare
    perm = torch.randperm(P, generator=gen).int()
    bt = torch.full((len(lens), MP), -1, dtype=torch.int32)
    at = 0
    for b, m in enumerate(pages):
        bt[b, :m] = perm[at:at + m]
        at += m
        if holes and m > 2:
            bt[b, 1] = -1
    return P, bt.to(device), torch.tensor([int(n) for n in lens], dtype=torch.int32, device=device)
