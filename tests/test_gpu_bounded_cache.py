"""Windowed attention with sinks, attention with key scores, and eviction, against 64 bits."""

import math
import threading

import pytest
import torch

from bounded_reference import (HALF_STEP, assert_within, evict_reference, make_problem, out_bound, paged_reference, to_gpu,
                               visible)
from nano_vllm_b200 import DevicePageTable, TinyKvPagedCache, TinyKvPagedPool, evict_tokens, flash_attention, paged_attention
from nano_vllm_b200 import _native as nv
from nano_vllm_b200 import write_slots

pytestmark = pytest.mark.gpu

BF, HF, F32, I8 = torch.bfloat16, torch.float16, torch.float32, torch.int8


@pytest.fixture(params=["default", "generic"])
def path(request, monkeypatch):
    if request.param == "generic":
        monkeypatch.setenv("NVM_ATTN_FORCE_GENERIC", "1")
    return request.param


def poison_unseen(prob, L, window, sinks, causal=True):
    """NaN and infinities wherever no query token looks: stale slots, unowned pages, keys
    outside every window."""
    k, v, ps = prob["k"], prob["v"], prob["ps"]
    P = k.shape[0]
    seen = torch.zeros(P, ps, dtype=torch.bool)
    for b in range(prob["bt"].shape[0]):
        n = int(prob["cl"][b])
        limit = max(0, min(n, prob["bt"].shape[1] * ps))
        for j in torch.nonzero(visible(n, limit, L, window, sinks, causal).any(0)).flatten().tolist():
            pid = int(prob["bt"][b, j // ps])
            if 0 <= pid < P:
                seen[pid, j % ps] = True
    hide = (~seen)[:, None, :, None]
    odd = torch.arange(ps)[None, None, :, None] % 2 == 1
    for x in ("k", "v"):
        if k.dtype == I8:
            s = prob[x + "s"]
            prob[x + "s"] = torch.where(hide, torch.where(odd, math.nan, math.inf).to(s.dtype), s)
        else:
            prob[x] = torch.where(hide, torch.where(odd, math.nan, math.inf).to(k.dtype), prob[x])
    return prob


# ctx, L, Hq, Hkv, D, ps, kv, q, window, sinks
WINDOW_CASES = [
    ([1], 1, 8, 8, 128, 16, BF, BF, 1, 0),                        # one token, a window of itself
    ([0, 1, 2, 16, 17], 1, 16, 8, 128, 16, BF, BF, 2, 1),         # empty and tiny contexts
    ([700, 33, 1025, 5000], 1, 32, 8, 128, 16, BF, BF, 256, 4),   # tile-aligned window
    ([701, 290, 4999], 1, 28, 4, 128, 16, HF, HF, 257, 5),        # odd everything, 7 heads a group
    ([3000, 90], 1, 64, 8, 64, 32, HF, HF, 100, 33),              # D = 64, sinks across a tile
    ([2048, 600], 1, 16, 8, 128, 128, BF, BF, 512, 600),          # more sinks than one context holds
    ([900, 400, 60], 1, 64, 8, 128, 128, I8, HF, 300, 16),        # int8 pages
    ([900, 400, 61], 1, 32, 4, 128, 16, I8, BF, 31, 3),           # int8 pages, bf16 queries and scales
    ([6000], 1, 128, 8, 128, 16, BF, BF, 1000, 4),                # 16 query rows a kv head
    ([801, 5, 1300, 17], 5, 32, 4, 128, 16, BF, BF, 100, 3),      # verify, 40 rows a kv head
    ([801, 2, 130], 3, 16, 8, 128, 16, HF, HF, 7, 2),             # context shorter than the new tokens
    ([500, 129], 4, 16, 2, 64, 64, HF, HF, 64, 0),                # verify, D = 64
    ([700, 300], 2, 32, 8, 128, 128, I8, HF, 129, 1),             # verify, int8
    ([700, 64, 40], 9, 8, 1, 128, 16, I8, HF, 70, 20),            # 72 rows, int8
    ([400, 128], 128, 8, 2, 128, 16, BF, BF, 50, 4),              # a chunk shorter than its window's reach
    ([1500, 300], 200, 8, 2, 128, 16, BF, BF, 333, 70),           # chunk, sinks across a 64-key tile
    ([1400, 260], 130, 8, 4, 128, 16, HF, HF, 1, 1),              # a window of one key
    ([900, 100], 70, 4, 4, 64, 32, HF, HF, 128, 4),               # chunk, D = 64
    ([900, 200], 90, 8, 2, 128, 64, I8, HF, 128, 4),              # chunk, int8
    ([900, 200], 90, 8, 2, 128, 48, BF, BF, 100, 49),             # chunk, pages that a 64-key tile straddles
    ([700, 150], 150, 8, 2, 128, 128, HF, HF, 129, 4),            # chunk, pages of two tiles
    ([5000, 300, 4100], 5, 32, 4, 128, 32, BF, BF, 3500, 100),    # verify, several chunks a unit
    ([300, 50], 3, 6, 2, 80, 7, F32, F32, 40, 5),                 # odd head dim and page size, fp32
    ([3000, 0, 1], 7, 8, 1, 128, 16, BF, BF, 2000, 9),            # one row tile over eight chunks, empty and tiny contexts
    ([2500, 1800, 60, 3], 40, 16, 2, 128, 16, HF, HF, 700, 4),    # 320 rows a kv head: several row tiles
    ([3000, 900], 191, 8, 4, 128, 16, BF, BF, 2900, 4),           # a chunk whose keys a cluster shares
    ([900, 300], 300, 4, 1, 128, 128, I8, HF, 3, 0),              # int8 chunk, row blocks within heads of odd length
    ([500, 64], 64, 4, 2, 64, 16, HF, HF, 20, 1),                 # blocks of exactly one head each
    ([300, 20], 1, 4, 4, 96, 24, HF, F32, 33, 2),                 # odd head dim, fp32 queries over fp16
]


@pytest.mark.parametrize("case", WINDOW_CASES, ids=lambda c: "-".join(str(x).replace("torch.", "") for x in c[:3]) + f"-w{c[8]}")
@pytest.mark.parametrize("mass_on", [False, True], ids=["out", "scored"])
def test_paged_window(case, mass_on, path):
    ctx, L, Hq, Hkv, D, ps, kv, qd, window, sinks = case
    prob = make_problem(len(ctx) + L, ctx, L, Hq, Hkv, D, ps, kv, qd)
    poison_unseen(prob, L, window, sinks)
    gen = torch.Generator().manual_seed(5)
    S = max(ctx) + 3
    mass = torch.rand(len(ctx), Hkv, S, generator=gen) if mass_on else None
    ref, terms, mref, merr = paged_reference(prob, window, sinks, mass=mass)
    p = to_gpu(prob)
    gm = mass.cuda() if mass_on else None
    for od in (F32, qd):
        if gm is not None:
            gm.copy_(mass)
        got = paged_attention(p["q"], p["k"], p["v"], p["bt"], p["cl"], ps, p["ks"], p["vs"], mask="causal", out_dtype=od,
                              window=window, sinks=sinks, key_mass=gm)
        assert_within(got, ref, out_bound(ref, terms, D, kv, od), "out")
        if gm is not None:
            assert_within(gm, mref, merr + 1e-30, "mass")
            for b, n in enumerate(ctx):
                assert torch.equal(gm[b, :, n:].cpu(), mass[b, :, n:])  # entries past the context


SCORED_CASES = [
    ([1, 0, 5], 1, 8, 8, 128, 16, BF, BF),
    ([777, 64, 2100], 1, 32, 8, 128, 16, BF, BF),
    ([5000, 4500], 1, 64, 8, 128, 16, HF, HF),       # several chunks a unit
    ([9000, 200, 3], 1, 7, 1, 64, 32, BF, BF),       # dozens of chunks, 7 rows, merged by the scores' kernel
    ([3000, 2600], 2, 8, 2, 128, 128, I8, HF),       # the same for two tokens over int8 pages
    ([300] * 12 + [4000] * 8, 1, 64, 8, 128, 16, BF, BF),  # more units than SMs, merged by their own CTAs
    ([33, 1000], 1, 28, 4, 64, 32, HF, HF),
    ([600, 1025], 1, 64, 8, 128, 128, I8, HF),
    ([600, 40], 1, 128, 8, 128, 16, BF, BF),         # 16 rows a kv head
    ([600, 4], 4, 32, 8, 128, 16, BF, BF),           # a context no longer than the new tokens
    ([3, 600], 5, 32, 4, 128, 16, HF, HF),           # shorter
    ([300, 70], 6, 8, 8, 128, 64, I8, HF),
    ([256, 300], 256, 8, 2, 128, 16, BF, BF),        # whole prompts and chunks
    ([700, 301], 300, 4, 2, 64, 16, HF, HF),
    ([400, 150], 130, 8, 2, 128, 16, I8, HF),
    ([100, 31], 2, 4, 2, 40, 5, F32, F32),
]


@pytest.mark.parametrize("case", SCORED_CASES, ids=lambda c: "-".join(str(x).replace("torch.", "") for x in c))
@pytest.mark.parametrize("causal", [True, False])
def test_key_mass(case, causal, path):
    ctx, L, Hq, Hkv, D, ps, kv, qd = case
    prob = make_problem(3 * L + len(ctx), ctx, L, Hq, Hkv, D, ps, kv, qd, holes=[(1, 1)] if ctx[1] > 2 * ps else [])
    poison_unseen(prob, L, 0, 0, causal)
    gen = torch.Generator().manual_seed(7)
    # rows of a larger buffer, transposed heads: strides of its own
    S = max(ctx)
    store = torch.rand(Hkv, len(ctx), S + 9, generator=gen).cuda()
    gm = store.transpose(0, 1)[:, :, 2:2 + S]
    before = store.clone()
    ref, terms, mref, merr = paged_reference(prob, causal=causal, mass=gm.cpu())
    p = to_gpu(prob)
    got = paged_attention(p["q"], p["k"], p["v"], p["bt"], p["cl"], ps, p["ks"], p["vs"], mask="causal" if causal else None,
                          key_mass=gm)
    assert_within(got, ref, out_bound(ref, terms, D, kv, F32), "out")
    assert_within(gm, mref, merr + 1e-30, "mass")
    assert torch.equal(store[:, :, :2], before[:, :, :2]) and torch.equal(store[:, :, 2 + S:], before[:, :, 2 + S:])
    # every row of weights sums to one, so a sequence gains Hq * L in all
    if not causal:
        for b, n in enumerate(ctx):
            old = before.transpose(0, 1)[b, :, 2:2 + max(0, n - L)].double().sum()
            total = gm[b, :, :n].double().sum() - old
            rows = Hq * L if n > 0 else 0
            assert abs(float(total.cpu()) - rows) <= 1e-4 * max(rows, 1) + 2 ** -22 * float(old), (float(total), rows)


@pytest.mark.parametrize("L", [1, 3, 70])
@pytest.mark.parametrize("kv,qd", [(BF, F32), (BF, HF), (I8, F32)])
def test_key_mass_with_queries_of_another_type(L, kv, qd):
    prob = make_problem(40 + L, [300, 90], L, 16, 4, 128, 16, kv, qd)
    taken = dict(prob, q=prob["q"].to(HF if kv == I8 else kv))  # as the tensor cores take it
    mass = torch.rand(2, 4, 300)
    ref, terms, mref, merr = paged_reference(taken, 0, 0, mass=mass)
    p, gm = to_gpu(prob), mass.cuda()
    got = paged_attention(p["q"], p["k"], p["v"], p["bt"], p["cl"], 16, p["ks"], p["vs"], mask="causal", key_mass=gm)
    assert_within(got, ref, out_bound(ref, terms, 128, kv, F32), "out")
    assert_within(gm, mref, merr + 1e-30, "mass")


def test_more_sequences_than_a_grid_axis_holds(path):
    B = 9000  # x 8 kv heads: more than 65535 rows of key_mass
    gen = torch.Generator().manual_seed(6)
    ctx = torch.randint(0, 20, (B,), generator=gen).tolist()
    prob = make_problem(7, ctx[:50], 1, 16, 8, 64, 16, BF, width_extra=0)
    pick = torch.randint(0, 50, (B,), generator=gen)
    prob = dict(prob, q=prob["q"][pick], bt=prob["bt"][pick], cl=prob["cl"][pick])
    mass = torch.zeros(B, 8, 32)
    check = torch.tensor([0, 1, 4500, B - 2, B - 1])
    small = dict(prob, q=prob["q"][check], bt=prob["bt"][check], cl=prob["cl"][check])
    ref, terms, mref, merr = paged_reference(small, 0, 0, mass=mass[check])
    p, gm = to_gpu(prob), mass.cuda()
    got = paged_attention(p["q"], p["k"], p["v"], p["bt"], p["cl"], 16, mask="causal", key_mass=gm)
    assert_within(got[check.cuda()], ref, out_bound(ref, terms, 64, BF, F32), "out")
    assert_within(gm[check.cuda()], mref, merr + 1e-30, "mass")
    total = gm.double().sum((1, 2)).cpu()
    assert ((total - 16.0 * (prob["cl"] > 0)).abs() <= 1e-3).all()


def test_key_mass_shorter_than_the_context(path):
    prob = make_problem(1, [200, 90], 1, 16, 8, 128, 16, BF)
    mass = torch.rand(2, 8, 100)
    _, _, mref, merr = paged_reference(prob, mass=mass)
    p, gm = to_gpu(prob), mass.cuda()
    paged_attention(p["q"], p["k"], p["v"], p["bt"], p["cl"], 16, mask="causal", key_mass=gm)
    assert_within(gm, mref, merr + 1e-30, "mass")


@pytest.mark.parametrize("L,D,kv", [(1, 128, BF), (6, 128, HF), (256, 128, BF), (256, 64, HF), (256, 128, I8), (30, 64, BF)])
def test_a_query_row_of_nan_shows_in_every_score_it_makes(L, D, kv, path):
    ctx, mass = 400, torch.rand(1, 2, 400)
    for head, row in ((0, 0), (1, L // 3), (2, L // 2 + 1), (3, L - 1), (1, 11), (2, 13), (0, 130), (3, 255)):
        if row >= L:
            continue
        prob = make_problem(50, [ctx], L, 8, 2, D, 16, kv)
        ref, terms, mref, merr = paged_reference(prob, mass=mass)
        prob["q"][0, head, row] = math.nan
        p, gm = to_gpu(prob), mass.cuda()
        out = paged_attention(p["q"], p["k"], p["v"], p["bt"], p["cl"], 16, p["ks"], p["vs"], mask="causal", key_mass=gm)
        seen = ctx - L + row + 1  # by the NaN row
        assert gm[0, 0, :seen].isnan().all(), (head, row, int(gm[0, 0, :seen].isnan().sum()))
        assert_within(gm[0, 0, seen:], mref[0, 0, seen:], merr[0, 0, seen:] + 1e-30, "keys it does not see")
        others = torch.ones(8, L, dtype=torch.bool)
        others[head, row] = False
        assert_within(out[0].cpu()[others], ref[0][others], out_bound(ref, terms, D, kv, F32)[0][others], "other rows")
        assert_within(gm[0, 1], mref[0, 1], merr[0, 1] + 1e-30, "the other kv head")


@pytest.mark.parametrize("L,Hq,kv", [(1, 64, BF), (2, 32, I8)])
def test_scores_of_wide_tables_are_kept_in_parts(L, Hq, kv):
    """81 requests of 128K-token tables, 8 rows a kv head: 2.7 GB of scores, taken in two parts of 41 and 40."""
    B, Hkv, D = 81, 8, 128
    ctx = [0, 1, 17, 5000] + torch.randint(2, 400, (B - 6,), generator=torch.Generator().manual_seed(8)).tolist() + [2600, 3]
    prob = make_problem(5, ctx, L, Hq, Hkv, D, 16, kv)
    prob["bt"] = torch.nn.functional.pad(prob["bt"], (0, 8192 - prob["bt"].shape[1]), value=-1)
    S = 4000  # shorter than one context
    store = torch.rand(Hkv, B, S + 2).cuda()
    gm = store.transpose(0, 1)[:, :, :S]
    p = to_gpu(prob)
    prob["bt"] = prob["bt"][:, :320]  # what the reference walks
    ref, terms, mref, merr = paged_reference(prob, mass=gm.cpu())
    before = store.clone()
    got = paged_attention(p["q"], p["k"], p["v"], p["bt"], p["cl"], 16, p["ks"], p["vs"], mask="causal", key_mass=gm)
    bound = out_bound(ref, terms, D, kv, F32)
    if kv == I8:
        # The weight times the value's scale is rounded to half: below 2^-14 by up to 2^-25, and then
        # multiplies the 8-bit value, |v| / scale.  `terms[2]` is the sum of |v| over the denominator.
        bound = bound + 2.0 ** -25 * terms[2] / float(prob["vs"].min())
    assert_within(got, ref, bound, "out")
    assert_within(gm, mref, merr + 1e-30, "mass")
    assert torch.equal(store[:, :, S:], before[:, :, S:])
    for b, n in enumerate(ctx):
        assert torch.equal(gm[b, :, n:], before.transpose(0, 1)[b, :, n:S])


@pytest.mark.parametrize("window", [None, 5000])
def test_more_units_than_merge_tickets(window):
    """257 prompts of 8192 tokens and 8 heads: 263168 blocks of 64 rows, whose chunks merge in two launches."""
    B, Hq, L, D, ps, mp = 257, 8, 8192, 64, 16, 545
    gen = torch.Generator(device="cuda").manual_seed(1)
    k, v = (torch.randn(600, 1, ps, D, device="cuda", generator=gen).to(BF) for _ in range(2))
    q = torch.empty(B, Hq, L, D, device="cuda", dtype=BF).normal_(generator=gen)
    bt = torch.stack([torch.randperm(600)[:mp] for _ in range(B)]).int()
    cl = torch.randint(8192, mp * ps + 1, (B,)).int()
    out = paged_attention(q, k, v, bt.cuda(), cl.cuda(), ps, mask="causal", window=window, sinks=4, out_dtype=BF)
    pick = [(b, h, r) for b in (0, 1, 127, 128, 129, 130, 255, 256) for h, r in ((0, 0), (3, 4000), (7, L - 1))]
    b, h, r = (torch.tensor(x) for x in zip(*pick))
    # a row is a decode call of its own at its position
    prob = {"q": q[b.cuda(), h.cuda(), r.cuda()].cpu()[:, None, None], "k": k.cpu(), "v": v.cpu(), "ks": None, "vs": None,
            "bt": bt[b], "cl": cl[b] - L + r.int() + 1, "ps": ps}
    ref, terms, _, _ = paged_reference(prob, window or 0, 4)
    assert_within(out[b.cuda(), h.cuda(), r.cuda()][:, None, None], ref, out_bound(ref, terms, D, BF, BF), "out")
    assert out.isfinite().all()
    assert not nv._workspaces[nv._workspace_key(out.device)][:1 << 20].any()  # every ticket is zero again


@pytest.mark.parametrize("L", [1, 6, 80])
def test_c_call_with_key_mass_of_no_length(L, path):
    """A buffer of no entries keeps no score, and the output is written all the same."""
    ctx, Hq, Hkv, D = [9000, 200, 3], 7 if L == 1 else 8, 1, 64
    prob = make_problem(2 + L, ctx, L, Hq, Hkv, D, 32, BF)
    ref, terms, _, _ = paged_reference(prob)
    p, lib = to_gpu(prob), nv.lib()
    mp, mass = p["bt"].shape[1], torch.full((8,), 3.0, device="cuda")
    out = torch.full((3, Hq, L, D), math.nan, device="cuda")
    need = lib.nvm_paged_attention_window_workspace_size(3, Hq, Hkv, L, D, 32, mp, nv.NVM_BF16, 0, 0, 1)
    ws = torch.zeros(max(need, 1), dtype=torch.uint8, device="cuda")
    nv.check(lib.nvm_paged_attention_window(
        p["q"].data_ptr(), nv.NVM_BF16, p["k"].data_ptr(), p["v"].data_ptr(), nv.NVM_BF16, None, None, nv.NVM_F16,
        p["bt"].data_ptr(), p["cl"].data_ptr(), out.data_ptr(), nv.NVM_F32, 3, Hq, Hkv, L, D, p["k"].shape[0], 32, mp, D ** -0.5,
        1, 0, 0, mass.data_ptr(), 0, 0, 0, ws.data_ptr(), need, nv.stream_ptr(out.device)))
    assert_within(out, ref, out_bound(ref, terms, D, BF, F32), "out")
    assert (mass == 3).all() and not ws[:min(need, 1 << 20)].any()  # the tickets are zero again


def test_out_at_any_alignment(path):
    for L in (1, 5, 80):
        prob = make_problem(12 + L, [300, 90], L, 16, 8, 128, 16, BF)
        p = to_gpu(prob)
        ref = paged_attention(p["q"], p["k"], p["v"], p["bt"], p["cl"], 16, mask="causal", window=100, out_dtype=BF)
        exact, terms, _, _ = paged_reference(prob, 100, 0)
        for shift in (1, 4):
            store = torch.zeros(ref.numel() + 8, dtype=BF, device="cuda")
            out = store[shift:shift + ref.numel()].view(ref.shape)
            got = paged_attention(p["q"], p["k"], p["v"], p["bt"], p["cl"], 16, mask="causal", window=100, out=out)
            assert got is out
            assert_within(out, exact, out_bound(exact, terms, 128, BF, BF), "out")
            assert not store[:shift].any() and not store[shift + ref.numel():].any()


def test_window_as_long_as_the_context_changes_nothing(path):
    prob = make_problem(2, [500, 77, 1300], 1, 32, 8, 128, 16, BF)
    p = to_gpu(prob)
    plain = paged_attention(p["q"], p["k"], p["v"], p["bt"], p["cl"], 16, mask="causal")
    wide = paged_attention(p["q"], p["k"], p["v"], p["bt"], p["cl"], 16, mask="causal", window=5000, sinks=3)
    ref, terms, _, _ = paged_reference(prob)
    b = out_bound(ref, terms, 128, BF, F32)
    assert_within(plain, ref, b)
    assert_within(wide, ref, b)


def test_window_without_causal(path):
    for L, window, sinks in ((1, 40, 2), (4, 9, 0), (80, 33, 5)):
        prob = make_problem(L, [300, 90], L, 8, 2, 128, 16, HF)
        ref, terms, _, _ = paged_reference(prob, window, sinks, causal=False)
        p = to_gpu(prob)
        got = paged_attention(p["q"], p["k"], p["v"], p["bt"], p["cl"], 16, window=window, sinks=sinks)
        assert_within(got, ref, out_bound(ref, terms, 128, HF, F32), f"L={L}")


@pytest.mark.parametrize("case", [([1020], 512, 8, 8, 64, BF, 64, 0, 64), ([1500, 1100], 1024, 8, 8, 128, I8, 256, 4, 128),
                                  ([1024], 1024, 2, 1, 128, BF, 64, 0, 64)], ids=["d64", "int8", "tcgen05"])
def test_long_windows_without_causal_find_their_workspace(case):
    ctx, L, Hq, Hkv, D, kv, window, sinks, mp = case
    prob = make_problem(L, ctx, L, Hq, Hkv, D, 16, kv)
    prob["bt"] = torch.nn.functional.pad(prob["bt"], (0, mp - prob["bt"].shape[1]), value=-1)
    ref, terms, _, _ = paged_reference(prob, window, sinks, causal=False)
    p = to_gpu(prob)
    run = lambda: paged_attention(p["q"], p["k"], p["v"], p["bt"], p["cl"], 16, p["ks"], p["vs"], window=window, sinks=sinks)  # noqa: E731
    fresh = torch.cuda.Stream()  # no earlier call grew this stream's workspace
    fresh.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(fresh):
        got = run()
    fresh.synchronize()
    assert_within(got, ref, out_bound(ref, terms, D, kv, F32), "out")
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got = run()
    graph.replay()
    torch.cuda.synchronize()
    assert_within(got, ref, out_bound(ref, terms, D, kv, F32), "captured")


def test_holes_inside_the_window(path):
    prob = make_problem(9, [400, 200], 1, 16, 8, 128, 16, BF, holes=[(0, 20), (1, 0), (1, 11)])
    ref, terms, mref, merr = paged_reference(prob, 100, 20, mass=torch.zeros(2, 8, 400))
    p, gm = to_gpu(prob), torch.zeros(2, 8, 400).cuda()
    got = paged_attention(p["q"], p["k"], p["v"], p["bt"], p["cl"], 16, mask="causal", window=100, sinks=20, key_mass=gm)
    assert_within(got, ref, out_bound(ref, terms, 128, BF, F32), "out")
    assert_within(gm, mref, merr + 1e-30, "mass")


def test_block_table_shorter_than_the_context(path):
    prob = make_problem(4, [640, 333], 1, 16, 8, 128, 16, BF, width_extra=0)
    prob["bt"] = prob["bt"][:, :15].contiguous()  # 240 keys of 640 are reachable
    for window in (500, 100):  # the second window begins past the table's end
        ref, terms, _, _ = paged_reference(prob, window, 4)
        p = to_gpu(prob)
        got = paged_attention(p["q"], p["k"], p["v"], p["bt"], p["cl"], 16, mask="causal", window=window, sinks=4)
        assert_within(got, ref, out_bound(ref, terms, 128, BF, F32), f"window {window}")


DENSE_CASES = [  # B, L, S, Hq, Hkv, D, dtype, window, sinks, causal
    (1, 1, 1, 4, 4, 128, BF, 1, 0, True),
    (2, 300, 300, 8, 2, 128, BF, 64, 4, True),
    (1, 257, 700, 8, 4, 128, HF, 100, 65, True),
    (1, 128, 500, 4, 1, 128, BF, 1, 0, True),
    (2, 5, 90, 8, 2, 128, HF, 20, 3, True),
    (1, 1, 900, 16, 4, 64, BF, 129, 2, True),
    (1, 200, 200, 4, 2, 64, HF, 33, 1, True),
    (1, 70, 150, 4, 2, 128, BF, 40, 2, False),
    (1, 40, 60, 4, 2, 72, F32, 11, 2, True),
    (1, 90, 2000, 8, 2, 128, BF, 1500, 4, True),     # few rows, many keys: a cluster shares them
    (1, 20, 900, 8, 2, 128, HF, 800, 4, True),       # the rows of a group in one tile, the same
    (1, 20, 8, 4, 2, 128, BF, 3, 1, True),          # more rows than keys: the first rows see none
]


@pytest.mark.parametrize("case", DENSE_CASES, ids=lambda c: "-".join(str(x).replace("torch.", "") for x in c))
def test_dense_window(case, path):
    B, L, S, Hq, Hkv, D, dt, window, sinks, causal = case
    gen = torch.Generator().manual_seed(L + S)
    q = (1.5 * torch.randn(B, Hq, L, D, generator=gen)).to(dt)
    k, v = (torch.randn(B, Hkv, S, D, generator=gen).to(dt) for _ in range(2))
    # a dense sequence is one page of S tokens
    prob = {"q": q, "k": k, "v": v, "ks": None, "vs": None, "ps": S, "bt": torch.arange(B, dtype=torch.int32)[:, None],
            "cl": torch.full((B,), S, dtype=torch.int32)}
    ref, terms, _, _ = paged_reference(prob, window, sinks, causal)
    for od in (dt, F32):
        got = flash_attention(q.cuda(), k.cuda(), v.cuda(), mask="causal" if causal else None, window=window, sinks=sinks,
                              out_dtype=od)
        assert got.dtype == od
        assert_within(got, ref, out_bound(ref, terms, D, dt, od), "out")


def test_dense_window_unseen_keys_may_hold_anything(path):
    gen = torch.Generator().manual_seed(3)
    q = torch.randn(1, 4, 100, 128, generator=gen).to(BF)
    k, v = (torch.randn(1, 2, 400, 128, generator=gen).to(BF) for _ in range(2))
    ok = visible(400, 400, 100, 50, 5).any(0)
    clean = flash_attention(q.cuda(), k.cuda(), v.cuda(), mask="causal", window=50, sinks=5)
    k[:, :, ~ok], v[:, :, ~ok] = math.inf, math.nan
    assert torch.equal(flash_attention(q.cuda(), k.cuda(), v.cuda(), mask="causal", window=50, sinks=5), clean)


@pytest.mark.parametrize("L", [1, 6, 80])
def test_pages_past_two_to_the_31_elements(L, path):
    prob = make_problem(50 + L, [700, 90], L, 16, 8, 128, 16, BF)
    P, big = prob["k"].shape[0], 150000  # 2.5e9 elements a pool
    mass = torch.rand(2, 8, 700)
    ref, terms, mref, merr = paged_reference(prob, 300, 4, mass=mass)
    p, gm = to_gpu(prob), mass.cuda()
    pools = []
    for x in ("k", "v"):
        pool = torch.empty(big, 8, 16, 128, dtype=BF, device="cuda")
        pool[big - P:] = p[x]
        pools.append(pool)
    bt = torch.where(p["bt"] >= 0, p["bt"] + (big - P), p["bt"])
    got = paged_attention(p["q"], *pools, bt, p["cl"], 16, mask="causal", window=300, sinks=4, key_mass=gm)
    assert_within(got, ref, out_bound(ref, terms, 128, BF, F32), "out")
    assert_within(gm, mref, merr + 1e-30, "mass")
    keep, _, _, eref, new, _ = evict_reference(prob, mass, 200, 4, 20)
    gm = mass.cuda()
    r = evict_tokens(*pools, bt, p["cl"], gm, 200, sinks=4, recent=20)
    assert torch.equal(r.keep_index.cpu(), keep) and torch.equal(gm.cpu(), eref)
    assert torch.equal(pools[0][big - P:].cpu(), new["k"]) and torch.equal(pools[1][big - P:].cpu(), new["v"])


def test_refusals():
    prob = to_gpu(make_problem(1, [40], 1, 8, 4, 128, 16, BF))
    call = lambda **kw: paged_attention(prob["q"], prob["k"], prob["v"], prob["bt"], prob["cl"], 16, mask="causal", **kw)  # noqa: E731
    for m in (torch.zeros(1, 4, 64), torch.zeros(1, 3, 64).cuda(), torch.zeros(1, 4, 64, dtype=HF).cuda(),
              torch.zeros(4, 64).cuda(), torch.zeros(1, 4, 128).cuda()[:, :, ::2], torch.zeros(1, 1, 64).cuda().expand(1, 4, 64)):
        with pytest.raises(RuntimeError):
            call(key_mass=m)
    with pytest.raises(RuntimeError, match="out must be"):
        call(window=4, out=torch.empty(1, 8, 1, 64, device="cuda"))
    with pytest.raises(NotImplementedError):
        flash_attention(prob["q"], prob["k"][:1], prob["v"][:1], mask=torch.zeros(1, device="cuda"), window=4)
    with pytest.raises(RuntimeError, match="key and value must be"):
        flash_attention(prob["q"], prob["k"], prob["v"], window=4)  # the batch does not match
    mass = torch.zeros(1, 4, 64, device="cuda")
    ev = lambda *a, **kw: evict_tokens(prob["k"], prob["v"], prob["bt"], prob["cl"], mass, *a, **kw)  # noqa: E731
    for a, kw in (((0,), {}), ((8,), dict(sinks=5, recent=4)), ((8,), dict(recent=-1))):
        with pytest.raises(RuntimeError, match="budget"):
            ev(*a, **kw)
    for kw in (dict(mass_out=torch.zeros(1, 4, 63, device="cuda")), dict(page_refcount=torch.zeros(1, dtype=torch.int32).cuda()),
               dict(status=torch.zeros(2, dtype=torch.int32).cuda())):
        with pytest.raises(RuntimeError):
            ev(8, **kw)
    with pytest.raises(RuntimeError, match="contiguous"):
        evict_tokens(prob["k"].transpose(0, 1), prob["v"].transpose(0, 1), prob["bt"], prob["cl"], mass, 8)
    i8 = to_gpu(make_problem(1, [40], 1, 8, 4, 128, 16, I8))
    with pytest.raises(RuntimeError, match="scales"):
        evict_tokens(i8["k"], i8["v"], i8["bt"], i8["cl"], mass, 8)


# ---------------------------------------------------------------------------
# eviction
# ---------------------------------------------------------------------------
def random_mass(gen, B, Hkv, S, kind):
    m = torch.exp(2 * torch.randn(B, Hkv, S, generator=gen))
    if kind == "ties":
        m = torch.randint(0, 4, (B, Hkv, S), generator=gen).float()
    elif kind == "zeros":
        m = torch.where(torch.rand(B, Hkv, S, generator=gen) < 0.5, 0.0, -0.0).float()
    elif kind == "odd values":
        pick = torch.rand(B, Hkv, S, generator=gen)
        m[pick < 0.2] = math.nan
        m[(pick >= 0.2) & (pick < 0.3)] = math.inf
        m[(pick >= 0.3) & (pick < 0.4)] = -math.inf
        m[(pick >= 0.4) & (pick < 0.6)] *= -1e-42  # subnormal, negative
    return m


def equal_or_nan(a, b):
    return torch.equal(a.isnan(), b.isnan()) and torch.equal(a.nan_to_num(7.0, 8.0, 9.0), b.nan_to_num(7.0, 8.0, 9.0))


EVICT_CASES = [  # ctx, Hkv, D, ps, dtype, budget, sinks, recent, kind
    ([20, 5, 9, 8], 2, 128, 16, BF, 8, 0, 0, "plain"),
    ([0, 1, 2], 1, 64, 16, HF, 1, 0, 0, "plain"),
    ([500, 100, 321], 8, 128, 16, BF, 128, 4, 32, "plain"),
    ([500, 130], 4, 128, 16, BF, 100, 0, 0, "ties"),
    ([500, 130], 4, 128, 16, HF, 100, 3, 5, "zeros"),
    ([700, 130, 90], 4, 128, 128, I8, 77, 16, 10, "odd values"),
    ([300], 2, 80, 7, F32, 120, 2, 9, "plain"),
    ([300], 2, 33, 5, BF, 120, 2, 9, "ties"),
    ([300, 299], 3, 33, 24, I8, 64, 64, 0, "plain"),      # nothing but sinks
    ([300, 299], 3, 64, 16, HF, 64, 0, 64, "plain"),      # nothing but the recent
    ([2049, 1025, 1024, 1023], 2, 64, 64, HF, 1023, 1, 100, "plain"),
    ([5000, 4096], 2, 128, 16, BF, 2500, 4, 64, "ties"),
    ([40000], 1, 64, 16, BF, 9000, 4, 64, "plain"),        # longer than a CTA holds in registers
    ([70000, 33000], 1, 64, 16, HF, 40000, 1, 1, "ties"),
]


@pytest.mark.parametrize("case", EVICT_CASES, ids=lambda c: "-".join(str(x).replace("torch.", "") for x in c))
@pytest.mark.parametrize("in_place", [True, False], ids=["in place", "mass out"])
def test_evict(case, in_place):
    ctx, Hkv, D, ps, dt, budget, sinks, recent, kind = case
    prob = make_problem(len(ctx) + budget, ctx, 1, Hkv, Hkv, D, ps, dt)
    gen = torch.Generator().manual_seed(budget)
    S = max(ctx) + 2
    mass = random_mass(gen, len(ctx), Hkv, S, kind)
    keep, kept, dropped, mref, new, bad = evict_reference(prob, mass, budget, sinks, recent)
    assert not bad
    p, gm = to_gpu(prob), mass.cuda()
    out = None if in_place else torch.full_like(gm, -5.0)
    r = evict_tokens(p["k"], p["v"], p["bt"], p["cl"], gm, budget, sinks=sinks, recent=recent, key_scales=p["ks"],
                     value_scales=p["vs"], mass_out=out)
    assert torch.equal(r.keep_index.cpu(), keep)
    assert torch.equal(r.kept.cpu(), kept) and torch.equal(r.dropped.cpu(), dropped) and not r.refused.any()
    got = gm.cpu() if in_place else out.cpu()
    for b, n in enumerate(ctx):
        assert equal_or_nan(got[b, :, :n], mref[b, :, :n])
        assert equal_or_nan(got[b, :, n:], mass[b, :, n:] if in_place else torch.full_like(mass[b, :, n:], -5.0))
    if not in_place:
        assert equal_or_nan(gm.cpu(), mass)
    for x in new:
        assert torch.equal(p[x].cpu(), new[x]), x
    assert torch.equal(p["cl"].cpu(), prob["cl"])


def test_evict_leaves_refused_requests_alone():
    prob = make_problem(8, [100, 100, 100, 20, 100], 1, 2, 2, 64, 16, BF)
    prob["bt"][1, 3] = -1                                  # unmapped
    prob["bt"][4, 0] = prob["k"].shape[0] + 5              # out of range, below the sinks' pages
    ref = torch.ones(prob["k"].shape[0], dtype=torch.int32)
    ref[prob["bt"][0, 0]] = 2                              # shared, but only sinks live there
    ref[prob["bt"][2, 4]] = 2                              # shared
    ref[prob["bt"][3, 0]] = 3                              # shared, but nothing moves
    mass = torch.rand(5, 2, 110)
    keep, kept, dropped, mref, new, bad = evict_reference(prob, mass, 40, 17, 4, ref)
    assert bad and dropped.tolist() == [60, 0, 0, 0, 60]
    p, gm = to_gpu(prob), mass.cuda()
    status = torch.zeros(1, dtype=torch.int32, device="cuda")
    r = evict_tokens(p["k"], p["v"], p["bt"], p["cl"], gm, 40, sinks=17, recent=4, page_refcount=ref.cuda(), status=status)
    assert int(status) != 0 and (r.refused != 0).tolist() == [False, True, True, False, False]
    assert torch.equal(r.keep_index.cpu(), keep) and torch.equal(r.kept.cpu(), kept) and torch.equal(r.dropped.cpu(), dropped)
    assert torch.equal(gm.cpu(), mref)
    assert torch.equal(p["k"].cpu(), new["k"]) and torch.equal(p["v"].cpu(), new["v"])
    short = evict_tokens(p["k"], p["v"], p["bt"], p["cl"], torch.rand(5, 2, 99).cuda(), 40, sinks=17)  # mass too short
    assert (short.refused != 0).tolist() == [True, True, True, False, True] and short.dropped.tolist() == [0, 0, 0, 0, 0]


def test_evict_on_another_stream_and_captured():
    prob = make_problem(5, [400, 300], 1, 4, 4, 128, 16, BF)
    mass = torch.rand(2, 4, 400)
    keep, _, _, mref, new, _ = evict_reference(prob, mass, 128, 4, 16)
    p, gm = to_gpu(prob), mass.cuda()
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        r = evict_tokens(p["k"], p["v"], p["bt"], p["cl"], gm, 128, sinks=4, recent=16)
    side.synchronize()
    assert torch.equal(r.keep_index.cpu(), keep) and torch.equal(p["k"].cpu(), new["k"]) and torch.equal(gm.cpu(), mref)
    p, gm = to_gpu(prob), mass.cuda()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        r = evict_tokens(p["k"], p["v"], p["bt"], p["cl"], gm, 128, sinks=4, recent=16)
    graph.replay()
    torch.cuda.synchronize()
    assert torch.equal(r.keep_index.cpu(), keep) and torch.equal(p["v"].cpu(), new["v"]) and torch.equal(gm.cpu(), mref)


# ---------------------------------------------------------------------------
# graphs, streams, repeatability
# ---------------------------------------------------------------------------
@pytest.mark.parametrize("L", [1, 6, 80])
def test_two_captured_graphs_replayed_side_by_side(L):
    probs = [make_problem(20 + i, [2500, 2900, 1000], L, 64 if L == 1 else 16, 8, 128, 16, BF) for i in range(2)]
    masses = [torch.rand(3, 8, 2900) for _ in range(2)]
    gpu, refs, outs, graphs, gms = [], [], [], [], []
    for prob, mass in zip(probs, masses):
        refs.append(paged_reference(prob, 2000, 4, mass=mass))
        p, gm = to_gpu(prob), mass.cuda()
        run = lambda: paged_attention(p["q"], p["k"], p["v"], p["bt"], p["cl"], 16, mask="causal", window=2000, sinks=4,  # noqa: E731
                                      key_mass=gm)
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            outs.append(run())
        graphs.append(graph)
        gpu.append(p)
        gms.append(gm)
    streams = [torch.cuda.Stream() for _ in range(2)]
    torch.cuda.synchronize()
    for _ in range(20):
        for graph, s, gm, mass in zip(graphs, streams, gms, masses):
            with torch.cuda.stream(s):
                gm.copy_(mass)
                graph.replay()
    torch.cuda.synchronize()
    for (ref, terms, mref, merr), out, gm in zip(refs, outs, gms):
        assert_within(out, ref, out_bound(ref, terms, 128, BF, F32), "out")
        assert_within(gm, mref, merr + 1e-30, "mass")


@pytest.mark.parametrize("L", [1, 6, 80])
def test_graphs_without_a_window_have_workspaces_of_their_own(L):
    """Captured without a warm-up, the second replayed first, then side by side, after an eager call that needs more."""
    probs = [make_problem(25 + i, [2500, 2900, 9000], L, 64 if L == 1 else 16, 8, 128, 16, BF) for i in range(2)]
    gpu = [to_gpu(p) for p in probs]
    refs = [paged_reference(p) for p in probs]
    graphs, outs = [], []
    for p in gpu:
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            outs.append(paged_attention(p["q"], p["k"], p["v"], p["bt"], p["cl"], 16, mask="causal"))
        graphs.append(graph)
    p = gpu[0]
    paged_attention(p["q"], p["k"], p["v"], p["bt"], p["cl"], 16, mask="causal", key_mass=torch.zeros(3, 8, 9000, device="cuda"))
    for i in (1, 0):
        graphs[i].replay()
        torch.cuda.synchronize()
        ref, terms, _, _ = refs[i]
        assert_within(outs[i], ref, out_bound(ref, terms, 128, BF, F32), f"graph {i}")
    streams = [torch.cuda.Stream() for _ in range(2)]
    first = [out.clone() for out in outs]
    torch.cuda.synchronize()
    for _ in range(20):
        for graph, s in zip(graphs, streams):
            with torch.cuda.stream(s):
                graph.replay()
    torch.cuda.synchronize()
    assert all(torch.equal(out, x) for out, x in zip(outs, first))


@pytest.mark.parametrize("L", [1, 6, 80])
def test_two_streams_at_once(L):
    probs = [make_problem(60 + i, [1500, 2900, 700], L, 64 if L == 1 else 16, 8, 128, 16, BF) for i in range(2)]
    masses = [torch.rand(3, 8, 2900) for _ in range(2)]
    refs = [paged_reference(p, 0, 0, mass=m) for p, m in zip(probs, masses)]
    gpu, gms = [to_gpu(p) for p in probs], [m.cuda() for m in masses]
    streams = [torch.cuda.Stream() for _ in range(2)]
    torch.cuda.synchronize()
    outs = [None, None]
    for _ in range(10):
        for i in range(2):
            with torch.cuda.stream(streams[i]):
                gms[i].copy_(masses[i])
                p = gpu[i]
                outs[i] = paged_attention(p["q"], p["k"], p["v"], p["bt"], p["cl"], 16, mask="causal", key_mass=gms[i])
    torch.cuda.synchronize()
    for (ref, terms, mref, merr), out, gm in zip(refs, outs, gms):
        assert_within(out, ref, out_bound(ref, terms, 128, BF, F32), "out")
        assert_within(gm, mref, merr + 1e-30, "mass")


@pytest.mark.parametrize("L", [1, 6, 80])
@pytest.mark.parametrize("kind", ["plain", "window", "dense", "scored"])
def test_first_call_of_a_thread(L, kind):
    """A thread's first call to CUDA may be one of the library's."""
    prob = make_problem(90 + L, [600, 700], L, 16, 8, 128, 16, BF)
    ref, terms, _, _ = paged_reference(prob, 100 if kind == "window" else 0, 4)
    p, got, mass = to_gpu(prob), [], torch.zeros(2, 8, 700, device="cuda")
    dense = torch.randn(2, 8, 300, 128, device="cuda").to(BF)
    want = flash_attention(p["q"], dense, dense, mask="causal", window=50)
    torch.cuda.synchronize()

    def run():
        if kind == "dense":
            got.append(flash_attention(p["q"], dense, dense, mask="causal", window=50))
        else:
            got.append(paged_attention(p["q"], p["k"], p["v"], p["bt"], p["cl"], 16, mask="causal", sinks=4,
                                       window=100 if kind == "window" else None, key_mass=mass if kind == "scored" else None))

    t = threading.Thread(target=run)
    t.start()
    t.join()
    torch.cuda.synchronize()
    assert len(got) == 1, "the call raised"
    if kind == "dense":
        assert torch.equal(got[0], want)
    else:
        assert_within(got[0], ref, out_bound(ref, terms, 128, BF, F32), "out")


@pytest.mark.parametrize("scored", [True, False])
@pytest.mark.parametrize("L", [1, 6, 80])
def test_two_threads_on_one_stream(L, scored):
    probs = [make_problem(70 + i, [1500 + 300 * i, 2900, 700], L, 64 if L == 1 else 16, 8, 128, 16, BF) for i in range(2)]
    masses = [torch.rand(3, 8, 2900) for _ in range(2)]
    refs = [paged_reference(p, 0, 0, mass=m) for p, m in zip(probs, masses)]
    gpu, starts = [to_gpu(p) for p in probs], [m.cuda() for m in masses]
    torch.cuda.synchronize()
    results = [[], []]

    def run(i):
        p = gpu[i]
        for _ in range(100):
            gm = starts[i].clone() if scored else None
            results[i].append((paged_attention(p["q"], p["k"], p["v"], p["bt"], p["cl"], 16, mask="causal", key_mass=gm), gm))

    threads = [threading.Thread(target=run, args=(i,)) for i in range(2)]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    torch.cuda.synchronize()
    for (ref, terms, mref, merr), got in zip(refs, results):
        assert len(got) == 100
        assert all(torch.equal(out, got[0][0]) for out, _ in got)
        assert_within(got[0][0], ref, out_bound(ref, terms, 128, BF, F32), "out")
        if scored:
            assert all(torch.equal(gm, got[0][1]) for _, gm in got)
            assert_within(got[0][1], mref, merr + 1e-30, "mass")


@pytest.mark.parametrize("L", [1, 6, 80])
def test_a_batch_of_empty_contexts_and_the_next_call(L):
    """Nothing is attended or scored, and what follows on the stream comes after it, captured too."""
    empty = to_gpu(make_problem(3, [0, 0, 0], L, 16, 4, 128, 16, BF, spare=40, width_extra=30))
    prob = make_problem(4, [400, 300], L, 16, 4, 128, 16, BF)
    mass, mass0 = torch.rand(2, 4, 400), torch.rand(3, 4, 480).cuda()
    ref, terms, mref, merr = paged_reference(prob, 0, 0, mass=mass)
    p, gm0, gm = to_gpu(prob), mass0.clone(), mass.cuda()
    out0, copy = torch.empty(3, 16, L, 128, device="cuda"), torch.empty(3, 16, L, 128, device="cuda")

    def both():
        paged_attention(empty["q"], empty["k"], empty["v"], empty["bt"], empty["cl"], 16, mask="causal", key_mass=gm0, out=out0)
        copy.copy_(out0)
        return paged_attention(p["q"], p["k"], p["v"], p["bt"], p["cl"], 16, mask="causal", key_mass=gm)

    for _ in range(20):
        out0.fill_(math.nan), gm.copy_(mass)
        got = both()
        assert not copy.any() and torch.equal(gm0, mass0)
    assert_within(got, ref, out_bound(ref, terms, 128, BF, F32), "out")
    assert_within(gm, mref, merr + 1e-30, "mass")
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got = both()
    for _ in range(20):
        out0.fill_(math.nan), gm.copy_(mass)
        graph.replay()
        assert not copy.any() and torch.equal(gm0, mass0)
    assert_within(got, ref, out_bound(ref, terms, 128, BF, F32), "captured")
    assert_within(gm, mref, merr + 1e-30, "mass")


@pytest.mark.parametrize("L", [1, 4, 100])
def test_results_do_not_depend_on_the_run(L, path):
    prob = make_problem(30 + L, [2300, 1700], L, 16, 2, 128, 16, BF)
    p = to_gpu(prob)
    first = None
    for _ in range(4):
        gm = torch.zeros(2, 2, 2304, device="cuda")
        out = paged_attention(p["q"], p["k"], p["v"], p["bt"], p["cl"], 16, mask="causal", key_mass=gm)
        first = first or (out, gm)
        assert torch.equal(out, first[0]) and torch.equal(gm, first[1])


# ---------------------------------------------------------------------------
# the three together, as a decode loop uses them
# ---------------------------------------------------------------------------
def test_decode_loop_with_eviction():
    """Two layers share a page table; every step appends a token, attends with scores, and the
    cache is trimmed when it reaches 48 tokens.  A plain simulation keeps each kv head's tokens
    in lists."""
    gen = torch.Generator().manual_seed(11)
    B, Hq, Hkv, D, ps, layers, budget, sinks, recent = 3, 8, 2, 128, 16, 2, 40, 2, 8
    table = DevicePageTable(B, 8, ps, 32)
    pools = [[torch.zeros(32, Hkv, ps, D, dtype=BF, device="cuda") for _ in range(2)] for _ in range(layers)]
    mass = [torch.full((B, Hkv, 128), math.nan, device="cuda") for _ in range(layers)]  # needs no clearing
    sim = [[[{"k": torch.zeros(0, D, dtype=torch.float64), "v": torch.zeros(0, D, dtype=torch.float64),
              "m": torch.zeros(0, dtype=torch.float64)} for _ in range(Hkv)] for _ in range(B)] for _ in range(layers)]
    for step in range(70):
        L = 30 if step == 0 else 1
        slots = table.append(torch.full((B,), L, dtype=torch.int32, device="cuda"))
        for y in range(layers):
            q = torch.randn(B, Hq, L, D, generator=gen).to(BF)
            k, v = (torch.randn(B * L, Hkv, D, generator=gen).to(BF) for _ in range(2))
            write_slots(k.cuda(), v.cuda(), slots, *pools[y])
            got = paged_attention(q.cuda(), *pools[y], table.block_table, table.context_lens, ps, mask="causal",
                                  key_mass=mass[y]).cpu().double()
            for b in range(B):
                for h in range(Hkv):
                    t = sim[y][b][h]
                    t["k"] = torch.cat([t["k"], k[b * L:(b + 1) * L, h].double()])
                    t["v"] = torch.cat([t["v"], v[b * L:(b + 1) * L, h].double()])
                    t["m"] = torch.cat([t["m"], torch.zeros(L, dtype=torch.float64)])
                    n, g = len(t["m"]), Hq // Hkv
                    z = q[b, h * g:h * g + g].double() @ t["k"].T / math.sqrt(D)
                    w = torch.softmax(z.masked_fill(~visible(n, n, L, 0, 0), -math.inf), -1)
                    t["m"] = t["m"] + w.sum((0, 1))
                    off = (got[b, h * g:h * g + g] - w @ t["v"]).abs().max()
                    assert off <= 2.0 ** -8 * float(t["v"].abs().max()), (step, y, b, h, float(off))
        lens = table.context_lens.tolist()
        if lens[0] >= 48:
            results = table.evict([(*pools[y], mass[y]) for y in range(layers)], budget, sinks=sinks, recent=recent)
            for y in range(layers):
                idx = results[y].keep_index.cpu().long()
                for b in range(B):
                    for h in range(Hkv):
                        t = sim[y][b][h]
                        n = len(t["m"])
                        mid = sorted(range(sinks, n - recent), key=lambda i: -float(t["m"][i]))[:budget - sinks - recent]
                        order = list(range(sinks)) + sorted(mid) + list(range(n - recent, n))
                        if idx[b, h].tolist() != order:  # allowed only where two weights are within rounding
                            theirs = sorted(set(idx[b, h].tolist()) ^ set(order))
                            spread = t["m"][theirs]
                            assert spread.max() - spread.min() <= 1e-4 * spread.max(), (step, y, b, h)
                            order = idx[b, h].tolist()
                        for x in ("k", "v", "m"):
                            t[x] = t[x][order]
            assert table.context_lens.tolist() == [budget] * B
            table.check_status()
    assert table.context_lens.tolist() == [len(sim[0][0][0]["m"])] * B
    assert int(table.free_top) + sum((n + ps - 1) // ps for n in table.context_lens.tolist()) == int(table.num_pages)


def test_table_evict_refuses_shared_prefix_pages():
    table = DevicePageTable(2, 8, 16, 16)
    pages = torch.randn(16, 2, 16, 64, device="cuda").to(BF)
    vals = torch.randn(16, 2, 16, 64, device="cuda").to(BF)
    table.append(torch.tensor([64, 0], dtype=torch.int32, device="cuda"))
    table.attach(torch.tensor([[0, 0], [0, 1]], dtype=torch.int32), torch.tensor([0, 2], dtype=torch.int32))
    table.append(torch.tensor([0, 30], dtype=torch.int32, device="cuda"))
    before = pages.clone()
    mass = torch.rand(2, 2, 128, device="cuda")
    table.evict([(pages, vals, mass)], 40, sinks=4)
    assert table.context_lens.tolist() == [64, 62] and torch.equal(pages, before)
    with pytest.raises(RuntimeError, match="evict refused"):
        table.check_status()
    # past the shared pages, request 1 may be trimmed; request 0's own pages 2 and 3 too
    table.evict([(pages, vals, mass)], 40, sinks=32, recent=2)
    assert table.context_lens.tolist() == [40, 40]
    table.check_status()


def test_an_attached_prefix_starts_without_scores():
    """The slot's last tenant left weights (and NaN) behind; the prefix's tokens are scored by the
    calls that follow alone, and eviction ranks by these."""
    B, Hq, Hkv, D, ps, layers = 3, 8, 2, 128, 16, 2
    table = DevicePageTable(B, 8, ps, 32)
    pools = [torch.randn(32, Hkv, ps, D, device="cuda").to(BF) for _ in range(2)]
    stale = torch.rand(B, Hkv, 128, device="cuda") * 100
    stale[2] = math.nan
    mass = [stale.clone() for _ in range(layers)]
    table.append(torch.tensor([64, 0, 0], dtype=torch.int32, device="cuda"))
    prefix = torch.tensor([[0, 0, 0], [0, 1, 2], [0, 1, 2]], dtype=torch.int32)
    table.attach(prefix, torch.tensor([0, 3, 2], dtype=torch.int32), key_mass=mass)
    table.check_status()
    for m in mass:
        assert torch.equal(m[0], stale[0])  # nothing attached
        assert not m[1, :, :48].any() and torch.equal(m[1, :, 48:], stale[1, :, 48:])
        assert not m[2, :, :32].any() and m[2, :, 32:].isnan().all()
    table.append(torch.tensor([0, 5, 5], dtype=torch.int32, device="cuda"))
    q = torch.randn(B, Hq, 5, D, device="cuda").to(BF)
    paged_attention(q, *pools, table.block_table, table.context_lens, ps, mask="causal", key_mass=mass[0])
    for b, n in ((1, 53), (2, 37)):  # every row's weights sum to one
        total = mass[0][b, :, :n].double().sum().item()
        assert abs(total - Hq * 5) <= 1e-4 * Hq * 5
    # refused: request 0 has tokens, and its scores stay; the table is as it was
    before, lens = mass[0].clone(), table.context_lens.clone()
    table.attach(prefix[:, :1].contiguous(), torch.tensor([1, 0, 0], dtype=torch.int32), key_mass=[mass[0]])
    with pytest.raises(RuntimeError):
        table.check_status()
    assert torch.equal(mass[0][0], before[0]) and torch.equal(table.context_lens, lens)
    for bad in (torch.zeros(2, Hkv, 8, device="cuda"), mass[0].double(), mass[0][0], mass[0].cpu()):
        with pytest.raises(ValueError, match="attach: key_mass"):
            table.attach(prefix, torch.zeros(3, dtype=torch.int32), key_mass=[bad])


def test_table_evict_wants_layers_alike():
    table = DevicePageTable(1, 4, 16, 8)
    pages, mass = torch.zeros(8, 2, 16, 64, device="cuda", dtype=BF), torch.zeros(1, 2, 64, device="cuda")
    table.append(torch.tensor([50], dtype=torch.int32, device="cuda"))
    for bad in ([(pages, pages, mass), (pages, pages, mass[:, :, :40])], [(pages, pages, mass), (pages[:7], pages[:7], mass)],
                [(pages, mass)], [(pages.view(4, 2, 32, 64), pages.view(4, 2, 32, 64), mass)]):
        with pytest.raises(ValueError, match="evict"):
            table.evict(bad, 20)
    assert table.context_lens.tolist() == [50]


def test_table_evict_with_a_faulty_layer_touches_none():
    table = DevicePageTable(1, 4, 16, 8)
    table.append(torch.tensor([50], dtype=torch.int32, device="cuda"))
    layers = [(*(torch.randn(8, 2, 16, 64, device="cuda").to(BF) for _ in range(2)), torch.rand(1, 2, 64, device="cuda"))
              for _ in range(2)]
    before = [[x.clone() for x in layer] for layer in layers]
    (k, v, mass), first = layers[1], layers[0]
    for bad in ((k, v, mass.double()), (k, v, torch.rand(1, 3, 64, device="cuda")), (k, first[1], mass), (k, v, first[2]),
                (k.to(I8), v.to(I8), mass), (k, v, mass.cpu())):
        with pytest.raises((RuntimeError, ValueError), match="evict"):
            table.evict([first, bad], 20)
        assert table.context_lens.tolist() == [50]
        assert all(torch.equal(x, y) for layer, old in zip(layers, before) for x, y in zip(layer, old))
    table.evict(layers, 20)
    assert table.context_lens.tolist() == [20]


def test_request_cache_evict():
    gen = torch.Generator().manual_seed(2)
    pool = TinyKvPagedPool(page_size=16, kv_bits=8)
    cache = TinyKvPagedCache(pool)
    k, v = (torch.randn(1, 2, 100, 64, generator=gen).to(HF).cuda() for _ in range(2))
    cache.update_and_fetch_paged(k, v)
    kq, vq = cache.gather_dense()
    mass = torch.rand(1, 2, 128, generator=gen).cuda()
    r = cache.evict(mass, 50, sinks=3, recent=10)
    assert cache.offset == 50 and cache.num_pages == 4 and pool.num_free_pages == 3
    k2, v2 = cache.gather_dense()
    for h in range(2):
        idx = r.keep_index[0, h].long()
        assert torch.equal(k2[0, h], kq[0, h, idx]) and torch.equal(v2[0, h], vq[0, h, idx])
    meta = cache.update_and_fetch_paged(k[:, :, :1], v[:, :, :1])
    assert int(meta.context_lens) == 51
