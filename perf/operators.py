"""Cases of the bounded-cache operators: attention with a sliding window and sinks, paged attention
that accumulates every cached key's attention weight, and eviction by that weight.

``run`` takes one pass through an operator: with ``own`` through the library's public calls, without it
through the plain form (elementary torch operations in 32 bits over gathered keys, rounded once).
"""

import math
import os
import sys

import torch

own = False

_DTYPES = {"bf16": torch.bfloat16, "f16": torch.float16}
_HEADS = [(16, 8), (32, 8), (64, 8), (32, 4), (28, 4), (8, 8)]


def _library():
    if "nano_vllm_b200" not in sys.modules:
        sys.path.insert(0, os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "nano-vllm-metal_b200"))
    import nano_vllm_b200

    return nano_vllm_b200


# ---------------------------------------------------------------------------
# cases
# ---------------------------------------------------------------------------
def _attend(name, B, L, Hq, Hkv, D, dtype, ps, lo, hi, window, sinks, mass, int8=False):
    return {"name": name, "kind": "paged", "B": B, "L": L, "Hq": Hq, "Hkv": Hkv, "D": D, "dtype": dtype, "ps": ps, "ctx_lo": lo,
            "ctx_hi": hi, "window": window, "sinks": sinks, "mass": mass, "int8": int8}


def _dense(name, B, L, S, Hq, Hkv, D, dtype, window, sinks):
    return {"name": name, "kind": "dense", "B": B, "L": L, "S": S, "Hq": Hq, "Hkv": Hkv, "D": D, "dtype": dtype, "window": window,
            "sinks": sinks}


def _evict(name, B, Hkv, D, dtype, ps, lo, hi, budget, sinks, recent, int8=False):
    return {"name": name, "kind": "evict", "B": B, "Hkv": Hkv, "D": D, "dtype": dtype, "ps": ps, "ctx_lo": lo, "ctx_hi": hi,
            "budget": budget, "sinks": sinks, "recent": recent, "int8": int8}


def listed():
    return [
        # one chat request a token at a time, a short window: the latency of a single small call
        _attend("window decode, 1 request", 1, 1, 16, 8, 128, "bf16", 16, 1500, 2500, 512, 4, False),
        # a full serving batch in long generations, where most of each cache lies outside the window
        _attend("window decode, 64 requests", 64, 1, 32, 8, 128, "bf16", 16, 4000, 16000, 4096, 4, False),
        # the same with 8-bit pages of the pool's default size
        _attend("window decode, int8 pages", 48, 1, 64, 8, 128, "f16", 128, 4000, 12000, 2048, 16, False, int8=True),
        # draft tokens verified under a window whose length no tile divides
        _attend("window verify, 5 tokens", 32, 5, 32, 4, 128, "f16", 16, 700, 9000, 1000, 3, False),
        # whole prompts under a window
        _dense("window prompt, dense", 2, 4096, 4096, 32, 8, 128, "bf16", 1024, 4),
        # one chunk of long prompts against their paged context
        _attend("window prompt, chunk of 512", 4, 512, 32, 8, 128, "bf16", 16, 2000, 8000, 2048, 4, False),
        # a decode step of one request that keeps score of its keys
        _attend("scored decode, 1 request", 1, 1, 32, 8, 128, "bf16", 16, 900, 1100, 0, 0, True),
        # a decode step of a full batch that keeps score of its keys
        _attend("scored decode, 64 requests", 64, 1, 32, 8, 128, "bf16", 16, 2000, 16000, 0, 0, True),
        # prompts whose keys get their first scores
        _attend("scored prompt", 2, 2048, 32, 8, 128, "bf16", 16, 2048, 2048, 0, 0, True),
        # one request trimmed to its budget every hundred tokens or so
        _evict("evict, 1 request", 1, 8, 128, "bf16", 16, 1100, 1200, 1024, 4, 64),
        # a batch trimmed after its prompts
        _evict("evict, 64 requests", 64, 8, 128, "bf16", 16, 2100, 8000, 2048, 4, 256),
        # the same with 8-bit pages of the pool's default size
        _evict("evict, int8 pages", 32, 8, 128, "f16", 128, 4000, 9000, 4000, 16, 128, int8=True),
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    Hq, Hkv = rng.choice(_HEADS)
    dtype = rng.choice(["bf16", "f16"])
    kind = rng.choice(["decode", "decode", "verify", "chunk", "dense", "scored decode", "scored decode", "scored verify",
                       "scored prompt", "evict", "evict"])
    int8 = kind not in ("dense",) and rng.random() < 0.3
    D = 128 if int8 else rng.choice([64, 128, 128, 128])
    ps = rng.choice([16, 16, 32, 64, 128])
    sinks = rng.choice([0, 1, 4, 16, rng.randint(2, 200)])
    window = _log(rng, 1, 6000)
    if kind == "dense":
        B, L = rng.choice([1, 2]), _log(rng, 1, 4096)
        return _without(_dense("", B, L, L + rng.choice([0, rng.randint(1, 500)]), Hq, Hkv, D, dtype, window, sinks))
    if kind == "evict":
        hi = _log(rng, 40, 8000)
        budget = rng.randint(max(1, hi // 4), hi)
        sinks = min(sinks, budget)
        recent = rng.randint(0, (budget - sinks) // 2)
        return _without(_evict("", _log(rng, 1, 48), Hkv, D, dtype, ps, max(1, hi // 3), hi, budget, sinks, recent, int8))
    scored = kind.startswith("scored")
    if kind in ("chunk", "scored prompt"):
        B, L = rng.choice([1, 2, 3]), _log(rng, 16, 1024 if kind == "chunk" else 2000)
        lo = L + rng.choice([0, rng.randint(0, 3000)])
        hi = lo if rng.random() < 0.3 else lo + rng.randint(0, 3000)
    else:
        L = rng.randint(2, 8) if kind.endswith("verify") else 1
        hi = _log(rng, 20, 16000)
        lo = max(L, hi // rng.choice([1, 2, 8]))
        B = _log(rng, 1, max(1, min(64, 700000 // hi)))
    if scored and rng.random() < 0.7:
        window, sinks = 0, 0
    return _without(_attend("", B, L, Hq, Hkv, D, dtype, ps, lo, max(lo, hi), window, sinks, scored, int8))


def _without(case):
    return {k: v for k, v in case.items() if k != "name"}


# ---------------------------------------------------------------------------
# inputs
# ---------------------------------------------------------------------------
def _lengths(case, seed):
    """Context lengths of the batch: drawn on the host from the seed alone."""
    gen = torch.Generator().manual_seed(seed)
    return torch.randint(case["ctx_lo"], case["ctx_hi"] + 1, (case["B"],), generator=gen, dtype=torch.int32), gen


def _pool(case, ctx, gen, gpu):
    """Pages in a random order, as a pool that many requests came and went through holds them; the pool
    and the block table have room for every request at its longest."""
    ps, Hkv, D = case["ps"], case["Hkv"], case["D"]
    pages = [(int(c) + ps - 1) // ps for c in ctx]
    width = (case["ctx_hi"] + ps - 1) // ps
    P = case["B"] * width + 8
    order = torch.randperm(P, generator=gen, dtype=torch.int32)
    table = torch.full((case["B"], width), -1, dtype=torch.int32)
    at = 0
    for b, n in enumerate(pages):
        table[b, :n] = order[at:at + n]
        at += n
    shape = (P, Hkv, ps, D)
    state = {"table": table.cuda(), "lens": ctx.cuda()}
    if case["int8"]:
        for x in ("k", "v"):
            state[x] = torch.randint(-127, 128, shape, dtype=torch.int8, device="cuda", generator=gpu)
            state[x + "s"] = ((torch.rand(P, Hkv, ps, 1, device="cuda", generator=gpu) + 0.5) * (2.5 / 127)).to(_DTYPES[case["dtype"]])
    else:
        for x in ("k", "v"):
            state[x] = torch.empty(shape, dtype=_DTYPES[case["dtype"]], device="cuda").normal_(generator=gpu)
            state[x + "s"] = None
    return state


def prepare(case, seed):
    gpu = torch.Generator(device="cuda").manual_seed(seed)
    B, Hkv, D = case["B"], case["Hkv"], case["D"]
    dtype = _DTYPES[case["dtype"]]
    if case["kind"] == "dense":
        rnd = lambda *s: torch.empty(s, dtype=dtype, device="cuda").normal_(generator=gpu)  # noqa: E731
        q = rnd(B, case["Hq"], case["L"], D) * 1.5
        return {"case": case, "q": q, "k": rnd(B, Hkv, case["S"], D), "v": rnd(B, Hkv, case["S"], D)}
    ctx, gen = _lengths(case, seed)
    state = _pool(case, ctx, gen, gpu)
    state["case"] = case
    S = state["table"].shape[1] * case["ps"]
    if case["kind"] == "evict" or case["mass"]:
        # accumulated attention weights: heavy-tailed, and some keys that nothing ever attended to
        mass = torch.exp(2 * torch.randn(B, Hkv, S, device="cuda", generator=gpu) - 4)
        state["mass"] = torch.where(torch.rand(B, Hkv, S, device="cuda", generator=gpu) < 0.1, torch.zeros_like(mass), mass)
    if case["kind"] == "evict":
        state["mass_out"] = torch.zeros_like(state["mass"])
    else:
        state["q"] = torch.empty((B, case["Hq"], case["L"], D), dtype=dtype, device="cuda").normal_(generator=gpu) * 1.5
    return state


# ---------------------------------------------------------------------------
# one pass
# ---------------------------------------------------------------------------
def run(state):
    case = state["case"]
    if own:
        return _run_own(state, case)
    if case["kind"] == "dense":
        return _plain_dense(state, case)
    if case["kind"] == "evict":
        return _plain_evict(state, case)
    return _plain_paged(state, case)


def _run_own(state, case):
    lib = _library()
    if case["kind"] == "dense":
        return lib.flash_attention(state["q"], state["k"], state["v"], mask="causal", window=case["window"], sinks=case["sinks"])
    if case["kind"] == "evict":
        got = lib.evict_tokens(state["k"], state["v"], state["table"], state["lens"], state["mass"], case["budget"], sinks=case["sinks"],
                               recent=case["recent"], key_scales=state["ks"], value_scales=state["vs"], mass_out=state["mass_out"])
        return _evict_outputs(state, got.keep_index, got.kept, got.dropped)
    out = lib.paged_attention(state["q"], state["k"], state["v"], state["table"], state["lens"], case["ps"], state["ks"], state["vs"],
                              mask="causal", out_dtype=state["q"].dtype, window=case["window"] or None, sinks=case["sinks"],
                              key_mass=state["mass"] if case["mass"] else None)
    return {"out": out, "mass": state["mass"]} if case["mass"] else out


def _evict_outputs(state, keep_index, kept, dropped):
    outs = {"keep_index": keep_index, "kept": kept, "dropped": dropped, "mass": state["mass_out"], "k": state["k"], "v": state["v"]}
    if state["ks"] is not None:
        outs["ks"], outs["vs"] = state["ks"], state["vs"]
    return outs


def _softmax_rows(s, seen):
    """Weights over the last axis of the scores that are seen; rows that see none are all zero."""
    s = s.masked_fill(~seen, float("-inf"))
    top = s.amax(-1, keepdim=True)
    p = torch.exp(s - torch.where(top == float("-inf"), torch.zeros_like(top), top))
    total = p.sum(-1, keepdim=True)
    return p / torch.where(total == 0, torch.ones_like(total), total)


def _plain_dense(state, case):
    B, L, S, Hq, Hkv, D = (case[x] for x in ("B", "L", "S", "Hq", "Hkv", "D"))
    pos = torch.arange(S - L, S, device="cuda")[:, None]
    key = torch.arange(S, device="cuda")[None, :]
    seen = (key <= pos) & ((key < case["sinks"]) | (key > pos - case["window"]))
    q = state["q"].float().view(B, Hkv, Hq // Hkv, L, D)
    s = torch.matmul(q, state["k"].float()[:, :, None].transpose(-1, -2)) * D ** -0.5
    out = torch.matmul(_softmax_rows(s, seen), state["v"].float()[:, :, None])
    return out.view(B, Hq, L, D).to(state["q"].dtype)


def _plain_paged(state, case):
    B, L, Hq, Hkv, D, ps, W, sinks = (case[x] for x in ("B", "L", "Hq", "Hkv", "D", "ps", "window", "sinks"))
    lens, table = state["lens"].long(), state["table"].long()
    cap = table.shape[1] * ps
    if W and sinks + W + L < cap:  # the sinks, then the window of the first query token up to the last key
        tail = lens[:, None] - (L + W - 1) + torch.arange(W + L - 1, device="cuda")
        head = torch.arange(sinks, device="cuda").expand(B, sinks)
        key = torch.cat([head, torch.where(tail < sinks, torch.full_like(tail, -1), tail)], 1)
    else:
        key = torch.arange(cap, device="cuda").expand(B, cap)
    there = (key >= 0) & (key < lens[:, None])
    at = key.clamp(0, cap - 1)
    page = table.gather(1, at // ps).clamp(min=0)
    fetch = lambda pool: pool[page, :, at % ps].float().transpose(1, 2)  # noqa: E731  [B, Hkv, keys, D]
    k, v = fetch(state["k"]), fetch(state["v"])
    if state["ks"] is not None:
        k, v = k * fetch(state["ks"]), v * fetch(state["vs"])
    pos = (lens[:, None] - L + torch.arange(L, device="cuda"))[:, :, None]
    seen = there[:, None] & (key[:, None] <= pos)
    if W:
        seen = seen & ((key[:, None] < sinks) | (key[:, None] > pos - W))
    q = state["q"].float().view(B, Hkv, Hq // Hkv, L, D)
    s = torch.matmul(q.reshape(B, Hkv, -1, D), k.transpose(-1, -2)).view(B, Hkv, Hq // Hkv, L, -1) * D ** -0.5
    p = _softmax_rows(s, seen[:, None, None])
    out = torch.matmul(p.view(B, Hkv, -1, p.shape[-1]), v).view(B, Hq, L, D).to(state["q"].dtype)
    if not case["mass"]:
        return out
    # the newest L keys start at zero, then every key gains what its rows gave it
    mass, every = state["mass"], torch.arange(state["mass"].shape[2], device="cuda")
    new = (every >= lens[:, None] - L) & (every < lens[:, None])
    mass.masked_fill_(new[:, None], 0.0)
    gained = torch.where(there[:, None], p.sum((2, 3)), torch.zeros((), device="cuda"))
    mass.scatter_add_(2, at[:, None].expand(B, Hkv, -1), gained)
    return {"out": out, "mass": mass}


def _plain_evict(state, case):
    B, Hkv, ps, budget, sinks, recent = (case[x] for x in ("B", "Hkv", "ps", "budget", "sinks", "recent"))
    lens, table, mass = state["lens"].long(), state["table"].long(), state["mass"]
    S = mass.shape[2]
    width = min(budget, S)
    every, n = torch.arange(S, device="cuda"), lens[:, None, None]
    inf = torch.full((), float("inf"), device="cuda")
    rank = torch.where((every < sinks) | (every >= n - recent), inf, mass)
    rank = torch.where(every >= n, -inf, rank)
    order = torch.sort(rank, dim=2, descending=True, stable=True).indices[:, :, :width].sort(2).values  # the kept, in order
    keep_index = torch.full((B, Hkv, budget), -1, dtype=torch.int32, device="cuda")
    keep_index[:, :, :width] = torch.where(order < n, order, -torch.ones_like(order)).int()
    kept = torch.minimum(lens, torch.full_like(lens, budget))
    # rows that move, one by one: (request, head, where to, where from)
    to = torch.arange(width, device="cuda")
    b, h, i = torch.nonzero((order < n) & (order != to), as_tuple=True)
    src = order[b, h, i]
    page_to, page_from = table[b, i // ps], table[b, src // ps]
    for pool in (state["k"], state["v"], state["ks"], state["vs"]):
        if pool is not None:
            pool[page_to, h, i % ps] = pool[page_from, h, src % ps]
    out = state["mass_out"]
    moved = torch.zeros_like(mass)
    moved[:, :, :width] = torch.where(order < n, mass.gather(2, order), torch.zeros((), device="cuda"))
    out.copy_(torch.where(every < n, moved, out))
    return _evict_outputs(state, keep_index, kept.int(), (lens - kept).int())


# ---------------------------------------------------------------------------
# what a pass cannot do without
# ---------------------------------------------------------------------------
def _seen_keys(n, L, window, sinks):
    """Keys that some of the last L rows of n see, and (row, key) pairs seen."""
    if not window:
        rows = min(L, n)
        return n, sum_pairs(n, rows)
    rows = min(L, n)
    first = max(0, n - rows - window + 1)
    keys = n if first <= sinks else n - first + sinks
    pairs = 0
    lo, hi = n - rows, n - 1  # positions of the rows; each sees min(pos + 1, window) and the sinks before that
    for cut, per in ((min(hi, window + sinks - 1), None), (hi, window + sinks)):
        if cut < lo:
            continue
        if per is None:
            pairs += (lo + 1 + cut + 1) * (cut - lo + 1) // 2
            lo = cut + 1
        else:
            pairs += per * (cut - lo + 1)
    return keys, pairs


def sum_pairs(n, rows):
    return (n - rows + 1 + n) * rows // 2


def work(case):
    B, Hkv, D = case["B"], case["Hkv"], case["D"]
    e = 1 if case.get("int8") else 2
    row = 2 * (D * e + (2 if e == 1 else 0))  # a key's K and V with their scales
    if case["kind"] == "evict":
        n = (case["ctx_lo"] + case["ctx_hi"]) / 2
        # a middle key stays with a chance below one, so all but the first few kept rows move
        moved = max(0, min(case["budget"], n) - case["sinks"]) if n > case["budget"] else 0
        return {"bytes": B * Hkv * (2 * moved * row + 8 * n + 4 * case["budget"]), "flops": 0}
    rows = B * case["Hq"] * case["L"] * D * 4  # q read, the result written, 2 bytes each
    n = case["S"] if case["kind"] == "dense" else (case["ctx_lo"] + case["ctx_hi"]) // 2
    keys, pairs = _seen_keys(n, case["L"], case["window"], case["sinks"])
    total = rows + B * Hkv * keys * row + (8 * B * Hkv * keys if case.get("mass") else 0)
    return {"bytes": total, "flops": 4.0 * D * B * case["Hq"] * pairs}


# ---------------------------------------------------------------------------
# the definitions in 64 bits, request by request
# ---------------------------------------------------------------------------
def exact(case, seed):
    state = prepare(case, seed)
    if case["kind"] == "evict":
        return None  # whole numbers and copies: nothing is computed
    B, L, Hq, Hkv, D, W, sinks = (case[x] for x in ("B", "L", "Hq", "Hkv", "D", "window", "sinks"))
    g, outs = Hq // Hkv, []
    mass = state["mass"].double() if case.get("mass") else None
    for b in range(B):
        if case["kind"] == "dense":
            n, k, v = case["S"], state["k"][b].double(), state["v"][b].double()
        else:
            n, ps = int(state["lens"][b]), case["ps"]
            pages = state["table"][b, :(n + ps - 1) // ps].long()
            dense = lambda x: state[x][pages].transpose(0, 1).reshape(Hkv, -1, state[x].shape[3])[:, :n].double()  # noqa: E731
            k, v = dense("k"), dense("v")
            if case["int8"]:
                k, v = k * dense("ks"), v * dense("vs")
        i = torch.arange(n - L, n, device="cuda").unsqueeze(1)
        j = torch.arange(n, device="cuda").unsqueeze(0)
        hidden = j > i
        if W:
            hidden |= (j >= sinks) & (i - j >= W)
        if mass is not None:
            mass[b, :, n - L:n] = 0
        one = []
        for h in range(Hq):
            z = state["q"][b, h].double() @ k[h // g].T / math.sqrt(D)
            w = torch.softmax(z.masked_fill(hidden, -math.inf), -1)
            one.append(w @ v[h // g])
            if mass is not None:
                mass[b, h // g, :n] += w.sum(0)
        outs.append(torch.stack(one))
    out = torch.stack(outs)
    return {"out": out, "mass": mass} if mass is not None else out
