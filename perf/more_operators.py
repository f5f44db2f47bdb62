"""Cases of the 4-bit paged cache: appending keys and values to it with the position rotation applied on
the way, reading rows back, and attention over it.

A cached row (one token of one kv head) holds its elements in groups of 64 as 4-bit codes with a scale s
and an offset z a group: value = s * code + z.  ``run`` takes one pass through an operator: with ``own``
through the library's public calls, without it through the plain form (elementary torch operations in 32
bits, rounded once).
"""

import math
import os
import sys
import types

import torch

own = False

_DTYPES = {"bf16": torch.bfloat16, "f16": torch.float16}
_HEADS = [(16, 8), (32, 8), (64, 8), (32, 4), (28, 4), (8, 8)]
_GROUP = 64
_TABLE = 40960  # rows of the rotation's tables


def _library():
    if "nano_vllm_b200" not in sys.modules:
        sys.path.insert(0, os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "nano-vllm-metal_b200"))
    import nano_vllm_b200

    return nano_vllm_b200


# ---------------------------------------------------------------------------
# cases
# ---------------------------------------------------------------------------
def _append(name, B, L, Hq, Hkv, D, dtype, ps, norm, traditional=False):
    return {"name": name, "kind": "append", "B": B, "L": L, "Hq": Hq, "Hkv": Hkv, "D": D, "dtype": dtype, "ps": ps, "norm": norm,
            "traditional": traditional}


def _read(name, B, lo, hi, Hkv, D, dtype, ps):
    return {"name": name, "kind": "read", "B": B, "ctx_lo": lo, "ctx_hi": hi, "Hkv": Hkv, "D": D, "dtype": dtype, "ps": ps}


def _attend(name, B, L, Hq, Hkv, D, dtype, ps, lo, hi):
    return {"name": name, "kind": "attend", "B": B, "L": L, "Hq": Hq, "Hkv": Hkv, "D": D, "dtype": dtype, "ps": ps, "ctx_lo": lo,
            "ctx_hi": hi}


def listed():
    return [
        # one chat request's newest token: the latency of a single small call, before every layer's attention
        _append("append, 1 token", 1, 1, 16, 8, 128, "bf16", 16, True),
        # the decode step of a full serving batch
        _append("append, 256 tokens", 256, 1, 32, 8, 128, "bf16", 16, True),
        # whole prompts of a model without q/k norm, pages of the pool's default size
        _append("append, prompts without norm", 4, 2048, 32, 8, 128, "f16", 128, False),
        # a cached prefix taken out at working precision, to be attended by a dense kernel or stored elsewhere
        _read("read back, 1 request", 1, 1500, 2500, 8, 128, "bf16", 16),
        # the same for the requests of a batch
        _read("read back, 16 requests", 16, 2000, 8000, 8, 128, "bf16", 16),
        # one chat request a token at a time
        _attend("decode, 1 request", 1, 1, 16, 8, 128, "bf16", 16, 1500, 2500),
        # a full serving batch
        _attend("decode, 64 requests", 64, 1, 32, 8, 128, "bf16", 16, 2000, 16000),
        # the same with more query heads a kv head and pages of the pool's default size
        _attend("decode, 8 heads a kv head", 48, 1, 64, 8, 128, "f16", 128, 4000, 12000),
        # small heads, pages that no tile divides
        _attend("decode, heads of 64", 24, 1, 32, 8, 64, "f16", 24, 300, 9000),
        # a single request with a long document
        _attend("decode, long context", 1, 1, 32, 4, 128, "bf16", 64, 90000, 130000),
        # draft tokens verified
        _attend("verify, 5 tokens", 32, 5, 32, 4, 128, "f16", 16, 700, 9000),
        # one chunk of long prompts against their paged context
        _attend("chunk of 512", 4, 512, 32, 8, 128, "bf16", 16, 2000, 8000),
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    Hq, Hkv = rng.choice(_HEADS)
    dtype = rng.choice(["bf16", "f16"])
    D = rng.choice([64, 128, 128, 128])
    ps = rng.choice([16, 16, 32, 64, 128, rng.randint(1, 100)])
    kind = rng.choice(["append", "append", "read", "decode", "decode", "decode", "verify", "verify", "chunk"])
    if kind == "append":
        L = rng.choice([1, 1, _log(rng, 2, 2048)])
        B = _log(rng, 1, min(256, 8192 // L))
        return _without(_append("", B, L, Hq, Hkv, D, dtype, ps, rng.random() < 0.6, rng.random() < 0.3))
    if kind == "read":
        hi = _log(rng, 1, 8000)
        return _without(_read("", _log(rng, 1, 16), max(1, hi // rng.choice([1, 2, 5])), hi, Hkv, D, dtype, ps))
    if kind == "chunk":
        B, L = rng.choice([1, 2, 3, 4]), _log(rng, 9, 512)
        lo = L + rng.choice([0, rng.randint(0, 3000)])
        hi = lo if rng.random() < 0.3 else lo + rng.randint(0, 3000)
        return _without(_attend("", B, L, Hq, Hkv, D, dtype, ps, lo, hi))
    L = rng.randint(2, 8) if kind == "verify" else 1
    hi = _log(rng, 8, 16000)
    lo = max(L, hi // rng.choice([1, 2, 8]))
    B = _log(rng, 1, max(1, min(64, 500000 // hi)))
    return _without(_attend("", B, L, Hq, Hkv, D, dtype, ps, lo, max(lo, hi)))


def _without(case):
    return {k: v for k, v in case.items() if k != "name"}


# ---------------------------------------------------------------------------
# inputs
# ---------------------------------------------------------------------------
def _pages(case, lens, gen):
    """Block tables over pages in a random order, as a pool that many requests came and went through holds
    them; the tables have room for every request at its longest."""
    ps = case["ps"]
    pages = [(int(c) + ps - 1) // ps for c in lens]
    width = max((case.get("ctx_hi", 0) + ps - 1) // ps, max(pages))
    P = case["B"] * width + 8
    order = torch.randperm(P, generator=gen, dtype=torch.int32)
    table = torch.full((case["B"], width), -1, dtype=torch.int32)
    at = 0
    for b, n in enumerate(pages):
        table[b, :n] = order[at:at + n]
        at += n
    return P, table


def _pool(case, P, gpu):
    """Pages full of other rows: evenly spread codes, scales and offsets as unit-sized keys and values give."""
    Hkv, ps, D, dtype = case["Hkv"], case["ps"], case["D"], _DTYPES[case["dtype"]]
    state = {}
    for x in ("k", "v"):
        state[x] = torch.randint(0, 256, (P, Hkv, ps, D // 2), dtype=torch.uint8, device="cuda", generator=gpu)
        s = (torch.rand(P, Hkv, ps, D // _GROUP, device="cuda", generator=gpu) + 0.5) * 0.22
        z = -7.5 * s + 0.2 * torch.randn(s.shape, device="cuda", generator=gpu)
        state[x + "s"] = torch.stack([s, z], -1).flatten(-2).to(dtype)
    return state


def prepare(case, seed):
    gpu = torch.Generator(device="cuda").manual_seed(seed)
    gen = torch.Generator().manual_seed(seed)
    B, Hkv, D, ps, dtype = case["B"], case["Hkv"], case["D"], case["ps"], _DTYPES[case["dtype"]]
    rnd = lambda *s: torch.empty(s, dtype=dtype, device="cuda").normal_(generator=gpu)  # noqa: E731
    if case["kind"] == "append":
        L, Hq = case["L"], case["Hq"]
        start = torch.randint(0, 4000, (B,), generator=gen)  # tokens that are there already
        P, table = _pages(case, start + L, gen)
        state = _pool(case, P, gpu)
        pos = start[:, None] + torch.arange(L)
        slots = table.long().gather(1, pos // ps) * ps + pos % ps
        qkv = rnd(B, L, (Hq + 2 * Hkv) * D)  # the fused projection, read in place
        angle = torch.arange(_TABLE, dtype=torch.float64, device="cuda")[:, None] * 1e6 ** (
            -torch.arange(D // 2, dtype=torch.float64, device="cuda") / (D // 2))
        state.update(
            q=qkv[..., :Hq * D].view(B, L, Hq, D), nk=qkv[..., Hq * D:(Hq + Hkv) * D].view(B, L, Hkv, D),
            nv=qkv[..., (Hq + Hkv) * D:].view(B, L, Hkv, D), positions=pos.int().cuda(), slots=slots.reshape(-1).cuda(),
            wq=1 + 0.2 * rnd(D) if case["norm"] else None, wk=1 + 0.2 * rnd(D) if case["norm"] else None,
            rope=types.SimpleNamespace(dims=D, traditional=case["traditional"], cos_freqs=angle.cos().float(),
                                       sin_freqs=angle.sin().float()))
    else:
        if case["kind"] == "read":  # as many rows in all for every seed
            lens = torch.linspace(case["ctx_lo"], case["ctx_hi"], B + 2)[1:-1].int()[torch.randperm(B, generator=gen)]
        else:
            lens = torch.randint(case["ctx_lo"], case["ctx_hi"] + 1, (B,), generator=gen, dtype=torch.int32)
        P, table = _pages(case, lens, gen)
        state = _pool(case, P, gpu)
        if case["kind"] == "read":
            rows = [table[b].long()[torch.arange(int(n)) // ps] * ps + torch.arange(int(n)) % ps for b, n in enumerate(lens)]
            state["slots"] = torch.cat(rows).cuda()
        else:
            state.update(table=table.cuda(), lens=lens.cuda(), q=rnd(B, case["Hq"], case["L"], D) * 1.5)
    state["case"] = case
    return state


# ---------------------------------------------------------------------------
# one pass
# ---------------------------------------------------------------------------
def run(state):
    case = state["case"]
    if own:
        return _run_own(state, case)
    if case["kind"] == "append":
        return _plain_append(state, case)
    if case["kind"] == "read":
        return _plain_read(state, case)
    return _plain_attend(state, case)


def _run_own(state, case):
    lib = _library()
    if case["kind"] == "attend":
        return lib.paged_attention(state["q"], state["k"], state["v"], state["table"], state["lens"], case["ps"], state["ks"],
                                   state["vs"], mask="causal", out_dtype=state["q"].dtype)
    q = None
    if case["kind"] == "append":
        q = lib.qk_norm_rope_write(state["q"], state["nk"], state["nv"], state["wq"], state["wk"], state["rope"],
                                   state["positions"], state["k"], state["v"], state["slots"], eps=1e-6,
                                   key_scales=state["ks"], value_scales=state["vs"])
    # the values that the rows stand for
    k, v = lib.read_slots(state["slots"], state["k"], state["v"], state["ks"], state["vs"])
    return {"k": k, "v": v} if q is None else {"q": q, "k": k, "v": v}


def _values(codes, scales):
    """Packed codes [..., D/2] and scales [..., 2 D/64] to the values, in 32 bits."""
    c = torch.stack([codes & 15, codes >> 4], -1).flatten(-2).float().unflatten(-1, (-1, _GROUP))
    s, z = scales.float().unflatten(-1, (-1, 2)).split(1, -1)
    return (c * s + z).flatten(-2)


def _quantised(x):
    """Rows [..., D] of a 16-bit type to (packed codes, scales): the offset is the group's least value, the
    scale a fifteenth of its span rounded up, so that no value is off by more than half a step."""
    g = x.float().unflatten(-1, (-1, _GROUP))
    z = g.amin(-1, keepdim=True)
    span = g.amax(-1, keepdim=True) - z
    exact_s = span / torch.full_like(span, 15)  # by a tensor: a division by a number multiplies by its inverse
    s = exact_s.to(x.dtype)
    s = torch.where(s.float() < exact_s, (s.view(torch.int16) + 1).view(x.dtype), s)  # the next one up
    wide = s.float()
    c = torch.where(wide > 0, (g - z) / wide, torch.zeros_like(g)).round().clamp(0, 15).to(torch.uint8).flatten(-2)
    return c[..., 0::2] | (c[..., 1::2] << 4), torch.cat([s, z.to(x.dtype)], -1).flatten(-2)


def _normed(x, weight, eps):
    """RMSNorm of rows, rounded to their type; the squares are summed four apart, then by halves."""
    D = x.shape[-1]
    y = x.float()
    sq = (y * y).unflatten(-1, (2, 32, D // 64))
    if D == 128:
        part = sq[..., 0, :, 0] + sq[..., 0, :, 1] + sq[..., 1, :, 0] + sq[..., 1, :, 1]
    else:
        part = sq[..., 0, :, 0] + sq[..., 1, :, 0]
    part = part[..., :16] + part[..., 16:]
    part = part[..., :8] + part[..., 8:]
    part = part[..., :4] + part[..., 4:]
    part = part[..., :2] + part[..., 2:]
    total = part[..., :1] + part[..., 1:]
    return (y * (1.0 / torch.sqrt(total * (1.0 / D) + eps)) * weight.float()).to(x.dtype)


def _rotated(x, cos, sin, traditional):
    """Rows [B, L, H, D] turned by the angles of [B, L, 1, D/2], rounded to their type."""
    y = x.float()
    if traditional:
        a, b = y[..., 0::2], y[..., 1::2]
        return torch.stack([a * cos - b * sin, a * sin + b * cos], -1).flatten(-2).to(x.dtype)
    a, b = y.chunk(2, -1)
    return torch.cat([a * cos - b * sin, a * sin + b * cos], -1).to(x.dtype)


def _plain_append(state, case):
    rope, pos, ps = state["rope"], state["positions"].long(), case["ps"]
    cos, sin = rope.cos_freqs[pos][:, :, None], rope.sin_freqs[pos][:, :, None]
    q, k = state["q"], state["nk"]
    if case["norm"]:
        q, k = _normed(q, state["wq"], 1e-6), _normed(k, state["wk"], 1e-6)
    q, k = _rotated(q, cos, sin, rope.traditional), _rotated(k, cos, sin, rope.traditional)
    page, off = state["slots"] // ps, state["slots"] % ps
    for x, rows in (("k", k), ("v", state["nv"])):
        codes, scales = _quantised(rows.flatten(0, 1))
        state[x][page, :, off] = codes
        state[x + "s"][page, :, off] = scales
    return {"q": q.transpose(1, 2).contiguous(), **_plain_read(state, case)}


def _plain_read(state, case):
    page, off = state["slots"] // case["ps"], state["slots"] % case["ps"]
    dtype = _DTYPES[case["dtype"]]
    return {x: _values(state[x][page, :, off], state[x + "s"][page, :, off]).to(dtype) for x in ("k", "v")}


def _plain_attend(state, case):
    B, L, Hq, Hkv, D, ps = (case[x] for x in ("B", "L", "Hq", "Hkv", "D", "ps"))
    lens, table = state["lens"].long(), state["table"].long()
    key = torch.arange(table.shape[1] * ps, device="cuda")
    page, off = table[:, key // ps].clamp(min=0), (key % ps).expand(B, -1)
    k = _values(state["k"][page, :, off], state["ks"][page, :, off]).transpose(1, 2)  # [B, Hkv, keys, D]
    v = _values(state["v"][page, :, off], state["vs"][page, :, off]).transpose(1, 2)
    pos = lens[:, None] - L + torch.arange(L, device="cuda")
    seen = (key <= pos[:, :, None])[:, None, None]  # [B, 1, 1, L, keys]
    q = state["q"].float().reshape(B, Hkv, -1, D)
    s = torch.matmul(q, k.transpose(-1, -2)).view(B, Hkv, Hq // Hkv, L, -1) * D ** -0.5
    s = s.masked_fill(~seen, float("-inf"))
    p = torch.exp(s - s.amax(-1, keepdim=True))
    p = p / p.sum(-1, keepdim=True)
    return torch.matmul(p.view(B, Hkv, -1, p.shape[-1]), v).view(B, Hq, L, D).to(state["q"].dtype)


# ---------------------------------------------------------------------------
# what a pass cannot do without
# ---------------------------------------------------------------------------
def work(case):
    B, Hkv, D = case["B"], case["Hkv"], case["D"]
    row = 2 * (D // 2 + 4 * (D // _GROUP))  # a token's K and V of one kv head, in the cache
    if case["kind"] == "append":
        rows = B * case["L"]
        token = 2 * D * (2 * case["Hq"] + 2 * Hkv) + Hkv * row + 4 * D + 12  # q in and out, k, v; a row of the tables
        return {"bytes": rows * (token + Hkv * (row + 4 * D)), "flops": 0}  # and the rows read back
    n = (case["ctx_lo"] + case["ctx_hi"]) / 2
    if case["kind"] == "read":
        return {"bytes": B * n * (Hkv * (row + 4 * D) + 8), "flops": 0}
    L = case["L"]
    pairs = L * (n - (L - 1) / 2)
    return {"bytes": B * (n * Hkv * row + 4 * case["Hq"] * L * D), "flops": 4.0 * D * B * case["Hq"] * pairs}


# ---------------------------------------------------------------------------
# the definitions in 64 bits
# ---------------------------------------------------------------------------
def _exact_values(codes, scales):
    s, z = scales.double()[..., 0::2], scales.double()[..., 1::2]
    wide = torch.empty(*codes.shape[:-1], 2 * codes.shape[-1], dtype=torch.float64, device=codes.device)
    wide[..., 0::2], wide[..., 1::2] = codes % 16, codes // 16
    return wide * s.repeat_interleave(_GROUP, -1) + z.repeat_interleave(_GROUP, -1)


def _rounded_up(x, dtype):
    """The least value of a 16-bit type that is not below x, in 64 bits."""
    near = x.to(dtype)
    step = torch.where(near < 0, -1, 1).to(torch.int16)
    return torch.where(near.double() < x, (near.view(torch.int16) + step).view(dtype), near).double()


def exact(case, seed):
    state = prepare(case, seed)
    ps = case["ps"]
    if case["kind"] == "read":
        page, off = state["slots"] // ps, state["slots"] % ps
        return {x: _exact_values(state[x][page, :, off], state[x + "s"][page, :, off]) for x in ("k", "v")}
    if case["kind"] == "append":
        return _exact_append(state, case)
    B, L, Hq, Hkv, D = (case[x] for x in ("B", "L", "Hq", "Hkv", "D"))
    outs = []
    for b in range(B):
        n = int(state["lens"][b])
        pages = state["table"][b, :(n + ps - 1) // ps].long()
        dense = lambda x: _exact_values(  # noqa: E731
            *(state[y][pages].transpose(0, 1).reshape(Hkv, -1, state[y].shape[3])[:, :n] for y in (x, x + "s")))
        k, v = dense("k"), dense("v")
        hidden = torch.arange(n, device="cuda")[None, :] > torch.arange(n - L, n, device="cuda")[:, None]
        one = []
        for h in range(Hq):
            z = state["q"][b, h].double() @ k[h * Hkv // Hq].T / math.sqrt(D)
            one.append(torch.softmax(z.masked_fill(hidden, -math.inf), -1) @ v[h * Hkv // Hq])
        outs.append(torch.stack(one))
    return torch.stack(outs)


def _exact_append(state, case):
    D, dtype = case["D"], _DTYPES[case["dtype"]]
    turn = torch.complex(state["rope"].cos_freqs.double(), state["rope"].sin_freqs.double())[state["positions"].long()][:, :, None]

    def made(x, w):  # a normed row is of the inputs' type before it is rotated
        x = x.double()
        if w is not None:
            x = (x / (x.square().mean(-1, keepdim=True) + 1e-6).sqrt() * w.double()).to(dtype).double()
        pairs = (x[..., 0::2], x[..., 1::2]) if case["traditional"] else (x[..., :D // 2], x[..., D // 2:])
        y = torch.complex(*pairs) * turn
        out = torch.empty_like(x)
        if case["traditional"]:
            out[..., 0::2], out[..., 1::2] = y.real, y.imag
        else:
            out[..., :D // 2], out[..., D // 2:] = y.real, y.imag
        return out

    def held(x):  # what the cache then stands for: rows, scales and offsets are of the inputs' type
        x = x.flatten(0, 1).to(dtype).double()
        groups = x.view(*x.shape[:-1], -1, _GROUP)
        z = -_rounded_up(-groups.min(-1, keepdim=True).values, dtype)
        s = _rounded_up((groups.max(-1, keepdim=True).values - z) / 15, dtype)
        return ((((groups - z) / s).round().clamp(0, 15)) * s + z).view(x.shape)

    return {"q": made(state["q"], state["wq"]).transpose(1, 2), "k": held(made(state["nk"], state["wk"])), "v": held(state["nv"])}
