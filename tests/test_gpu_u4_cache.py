"""The 4-bit cache on the GPU: what is written, read back and attended to, against the row format in
numpy and attention in 64 bits (tests/u4_reference.py derives the error bounds)."""

import numpy as np
import pytest
import torch

import nano_vllm_b200 as lib
from nano_vllm_b200 import _native as nv
from nano_vllm_b200.layers.qk_prep import qk_norm_rope_write
from nano_vllm_b200.layers.rotary_embedding import RoPE
from u4_reference import attend64, pack, quantise, random_pools, random_table, values64

pytestmark = pytest.mark.gpu
BF, HF, FF = torch.bfloat16, torch.float16, torch.float32


def _empty_pools(P, Hkv, ps, D, dtype, device="cuda"):
    """Pools of a recognisable filler, so that rows that should stay are seen to."""
    kp = torch.full((P, Hkv, ps, D // 2), 0xA5, dtype=torch.uint8, device=device)
    ks = torch.full((P, Hkv, ps, D // 32), 3.0, dtype=dtype, device=device)
    return kp, kp.clone(), ks, ks.clone()


def _expect_rows(rows, slots, pages, scales, ps):
    """pages / scales (on the host, as they were) after rows [T, H, D] were written at slots."""
    packed, sc = pack(*quantise(rows, scales.dtype), scales.dtype)
    pages, scales = pages.clone(), scales.clone()
    for t, slot in enumerate(slots.tolist()):
        if 0 <= slot < pages.shape[0] * ps:
            pages[slot // ps, :, slot % ps] = packed[t]
            scales[slot // ps, :, slot % ps] = sc[t]
    return pages, scales


def _same(got, want):
    got, want = got.cpu(), want
    if got.dtype == torch.uint8:
        assert torch.equal(got, want)
    else:  # by value: an offset of -0.0 and 0.0 are the same
        g, w = got.float(), want.float()
        assert torch.equal(g.isnan(), w.isnan()) and torch.equal(g.nan_to_num(7.0), w.nan_to_num(7.0))


def _slots(gen, T, P, ps, bad=True):
    slots = torch.randperm(P * ps, generator=gen)[:T].to(torch.int64)
    if bad and T > 3:
        slots[1], slots[T - 1] = -1, P * ps + 5
    return slots


@pytest.mark.parametrize("dtype,scale", [(BF, BF), (HF, HF), (FF, BF), (FF, HF), (BF, HF), (HF, BF)])
@pytest.mark.parametrize("D", [64, 128])
@pytest.mark.parametrize("T,Hkv,ps", [(1, 1, 1), (1, 8, 16), (7, 3, 5), (130, 8, 16), (67, 4, 128)])
def test_write(cuda, dtype, scale, D, T, Hkv, ps):
    gen = torch.Generator().manual_seed(T * 7 + D)
    P = (T + 9) // ps + 3
    k = torch.randn(T, Hkv, D, generator=gen) * torch.exp(torch.randn(T, Hkv, 1, generator=gen))
    v = torch.randn(T, Hkv, D, generator=gen) + 3 * torch.randn(T, Hkv, 1, generator=gen)
    k[0, 0, :64] = 1.25  # no span
    if T > 4:
        v[2, 0, 5], v[3, 0, 63], k[4, Hkv - 1, 0] = float("nan"), float("inf"), -float("inf")
    k, v, slots = k.to(dtype), v.to(dtype), _slots(gen, T, P, ps)
    pools = _empty_pools(P, Hkv, ps, D, scale)
    before = [t.cpu() for t in pools]
    lib.write_slots(k.cuda(), v.cuda(), slots.cuda(), *pools)
    for rows, i in ((k, 0), (v, 1)):
        pages, scales = _expect_rows(rows, slots, before[i], before[i + 2], ps)
        _same(pools[i], pages)
        _same(pools[i + 2], scales)


def test_write_strided_rows_and_odd_addresses(cuda):
    """Rows taken out of a fused projection, head-major views, and rows that start on no vector's boundary."""
    gen = torch.Generator().manual_seed(3)
    T, H, D, ps, P = 37, 4, 128, 16, 6
    for make in (lambda x: torch.cat([x, x, x], -1)[..., H * D:2 * H * D].view(T, H, D),
                 lambda x: x.view(T, H, D).transpose(0, 1).contiguous().transpose(0, 1),
                 lambda x: torch.cat([x.new_zeros(3), x.reshape(-1)])[3:].view(T, H, D)):
        base = torch.randn(T, H * D, generator=gen).to(BF).cuda()
        k, v = make(base), make(base * 2)
        slots = _slots(gen, T, P, ps)
        pools = _empty_pools(P, H, ps, D, BF)
        before = [t.cpu() for t in pools]
        lib.write_slots(k, v, slots.cuda(), *pools)
        for rows, i in ((k, 0), (v, 1)):
            pages, scales = _expect_rows(rows, slots, before[i], before[i + 2], ps)
            _same(pools[i], pages)
            _same(pools[i + 2], scales)


@pytest.mark.parametrize("out", [BF, HF, FF])
@pytest.mark.parametrize("scale", [BF, HF])
@pytest.mark.parametrize("D,T,Hkv,ps", [(128, 1, 8, 16), (128, 257, 8, 16), (64, 33, 3, 7), (64, 1, 1, 1), (128, 50, 1, 100)])
def test_read(cuda, out, scale, D, T, Hkv, ps):
    gen = torch.Generator().manual_seed(T + D)
    P = (T + 9) // ps + 3
    kp, vp, ks, vs = random_pools(gen, P, Hkv, ps, D, scale)
    slots = _slots(gen, T, P, ps)
    got = lib.read_slots(slots.cuda(), kp, vp, ks, vs, out)
    for x, pages, scales in zip(got, (kp, vp), (ks, vs)):
        assert x.shape == (T, Hkv, D) and x.dtype == out and x.is_contiguous()
        at = slots.clamp(0, P * ps - 1).cuda()
        want = values64(pages[at // ps, :, at % ps], scales[at // ps, :, at % ps]).float()  # s * code is exact: one rounding
        want[(slots < 0) | (slots >= P * ps)] = 0
        assert torch.equal(x, want.to(out))


@pytest.mark.parametrize("pages", [BF, HF, FF, torch.int8])
@pytest.mark.parametrize("D,T,Hkv,ps", [(128, 70, 8, 16), (80, 9, 3, 5), (4, 6, 2, 4), (1, 3, 1, 2)])
def test_read_other_pages(cuda, pages, D, T, Hkv, ps):
    """What write_slots put there comes back, of any page type."""
    gen = torch.Generator().manual_seed(T)
    P = T // ps + 3
    slots = torch.randperm(P * ps, generator=gen)[:T].cuda()
    dtype = HF if pages == torch.int8 else pages
    k, v = (torch.randn(T, Hkv, D, generator=gen).to(dtype).cuda() for _ in range(2))
    kp, vp = (torch.zeros(P, Hkv, ps, D, dtype=pages, device="cuda") for _ in range(2))
    ks, vs = (torch.ones(P, Hkv, ps, 1, dtype=dtype, device="cuda") for _ in range(2)) if pages == torch.int8 else (None, None)
    lib.write_slots(k, v, slots, kp, vp, ks, vs)
    got = lib.read_slots(slots, kp, vp, ks, vs)
    for x, rows, pool, sc in zip(got, (k, v), (kp, vp), (ks, vs)):
        at = slots.long()
        want = rows if sc is None else (pool[at // ps, :, at % ps].float() * sc[at // ps, :, at % ps].float()).to(dtype)
        assert torch.equal(x, want)
    wide = lib.read_slots(slots, kp, vp, ks, vs, FF)[0]
    assert wide.dtype == FF and torch.equal(wide.to(dtype), got[0])


@pytest.mark.parametrize("dtype", [BF, HF])
@pytest.mark.parametrize("D", [64, 128])
@pytest.mark.parametrize("traditional", [False, True])
@pytest.mark.parametrize("norm", [False, True])
@pytest.mark.parametrize("B,L,Hq,Hkv", [(1, 1, 4, 2), (3, 5, 9, 3), (2, 70, 16, 8), (40, 1, 28, 4)])
def test_append(cuda, dtype, D, traditional, norm, B, L, Hq, Hkv):
    """The fused append leaves the rows that it leaves in 16-bit pages, quantised, and the same q."""
    gen = torch.Generator().manual_seed(B * L)
    ps, T = 16, B * L
    P = T // ps + 4
    qkv = torch.randn(B, L, (Hq + 2 * Hkv) * D, generator=gen).to(dtype).cuda()
    q, k, v = (x.view(B, L, -1, D) for x in qkv.split([Hq * D, Hkv * D, Hkv * D], -1))
    w = [torch.randn(D, generator=gen).to(dtype).cuda() for _ in range(2)] if norm else [None, None]
    rope = RoPE(D, 300, base=1e4, traditional=traditional, device="cuda")
    pos = torch.randint(0, 300, (B, L), generator=gen).int().cuda()
    slots = _slots(gen, T, P, ps, bad=False)
    if T > 3:
        slots[2] = -1
    wide = [torch.zeros(P, Hkv, ps, D, dtype=dtype, device="cuda") for _ in range(2)]
    q16 = qk_norm_rope_write(q, k, v, *w, rope, pos, *wide, slots.cuda())
    pools = _empty_pools(P, Hkv, ps, D, dtype)
    before = [t.cpu() for t in pools]
    q4 = qk_norm_rope_write(q, k, v, *w, rope, pos, *pools[:2], slots.cuda(), key_scales=pools[2], value_scales=pools[3])
    assert torch.equal(q4, q16)
    at = slots.clamp(min=0).cuda()
    for i, pool in enumerate(wide):
        pages, scales = _expect_rows(pool[at // ps, :, at % ps], slots, before[i], before[i + 2], ps)
        _same(pools[i], pages)
        _same(pools[i + 2], scales)
    # the rotation itself, in 64 bits: the fp32 products and sums (3 * 2^-24 of the two terms) and one
    # rounding to the type; norms round once more before the rotation, so they have their own test
    if not norm:
        c, s = rope.cos_freqs[pos.long()].double()[:, :, None], rope.sin_freqs[pos.long()].double()[:, :, None]
        x = q.double()
        a, b = (x[..., 0::2], x[..., 1::2]) if traditional else (x[..., :D // 2], x[..., D // 2:])
        want = [a * c - b * s, a * s + b * c]
        size = [(a * c).abs() + (b * s).abs(), (a * s).abs() + (b * c).abs()]
        join = (lambda y: torch.stack(y, -1).flatten(-2)) if traditional else (lambda y: torch.cat(y, -1))
        got = q4.transpose(1, 2).double()
        tol = join(want).abs() * torch.finfo(dtype).eps / 2 * 1.001 + join(size) * 2.0 ** -22 + 2.0 ** -25
        assert ((got - join(want)).abs() <= tol).all()


@pytest.mark.parametrize("kv", [BF, torch.int8])
def test_append_without_norm_into_other_pages(cuda, kv):
    """Without weights the rows are rotated as they are, whatever the pages hold."""
    gen = torch.Generator().manual_seed(5)
    B, L, Hq, Hkv, D, ps, P = 2, 9, 8, 4, 128, 16, 4
    q, k, v = (torch.randn(B, L, h, D, generator=gen).to(BF).cuda() for h in (Hq, Hkv, Hkv))
    rope = RoPE(D, 64, device="cuda")
    pos = torch.randint(0, 64, (B, L), generator=gen).int().cuda()
    slots = torch.randperm(P * ps, generator=gen)[:B * L].cuda()
    kp, vp = (torch.zeros(P, Hkv, ps, D, dtype=kv, device="cuda") for _ in range(2))
    sc = [torch.ones(P, Hkv, ps, 1, dtype=BF, device="cuda") for _ in range(2)] if kv == torch.int8 else [None, None]
    got = qk_norm_rope_write(q, k, v, None, None, rope, pos, kp, vp, slots, key_scales=sc[0], value_scales=sc[1])
    assert torch.equal(got, rope.apply(q, pos).transpose(1, 2))  # the same fp32 products and sums, one rounding
    want = [torch.zeros_like(kp), torch.zeros_like(vp)]
    wsc = [None if x is None else torch.ones_like(x) for x in sc]
    lib.write_slots(rope.apply(k, pos).flatten(0, 1), v.flatten(0, 1), slots, *want, *wsc)
    assert torch.equal(kp, want[0]) and torch.equal(vp, want[1])
    assert all(x is None or torch.equal(x, y) for x, y in zip(sc, wsc))


def test_append_groups_that_cannot_be_held(cuda):
    for D in (64, 128):
        q = torch.randn(1, 2, 2, D, device="cuda").to(BF)
        v = torch.randn(1, 2, 2, D, device="cuda").to(BF)
        v[0, 0, 1, D - 1], v[0, 1, 0, 7] = float("nan"), -float("inf")
        pools = _empty_pools(1, 2, 4, D, BF)
        rope = RoPE(D, 4, device="cuda")
        qk_norm_rope_write(q, q, v, None, None, rope, torch.zeros(1, 2, dtype=torch.int32, device="cuda"), *pools[:2],
                           torch.tensor([0, 2], device="cuda"), key_scales=pools[2], value_scales=pools[3])
        k, got = lib.read_slots(torch.tensor([0, 2], device="cuda"), *pools)
        bad = torch.zeros(2, 2, D, dtype=torch.bool, device="cuda")
        bad[0, 1, D - 64:], bad[1, 0, :64] = True, True
        assert torch.equal(got.isnan(), bad) and not k.isnan().any()


# ---------------------------------------------------------------------------
# attention
# ---------------------------------------------------------------------------
def _attend(gen, lens, L, Hq, Hkv, D, ps, qdt, sdt, out=None, causal=True, holes=False, scale=None, pools=None, qscale=1.5, **kw):
    P, bt, cl = random_table(gen, lens, ps, holes=holes, **kw)
    kp, vp, ks, vs = random_pools(gen, P, Hkv, ps, D, sdt) if pools is None else pools(P)
    q = (torch.randn(len(lens), Hq, L, D, generator=gen) * qscale).to(qdt).cuda()
    got = lib.paged_attention(q, kp, vp, bt, cl, ps, ks, vs, scale=scale, mask="causal" if causal else None, out_dtype=out or qdt)
    want, bound = attend64(q, kp, vp, ks, vs, bt, cl, ps, scale, causal)
    return got, want, bound


def _close(got, want, bound, what=""):
    half = torch.finfo(got.dtype).eps / 2
    tol = bound + (want.abs() + bound) * half * 1.001 + torch.finfo(got.dtype).smallest_normal * half
    off = (got.double() - want).abs()
    assert not got.isnan().any(), what
    assert (off <= tol).all(), f"{what}: {(off / tol).max().item():.3g} times the bound"


@pytest.mark.parametrize("qdt,sdt", [(BF, BF), (HF, HF), (BF, HF), (HF, BF), (FF, BF)])
@pytest.mark.parametrize("D", [64, 128])
@pytest.mark.parametrize("Hq,Hkv", [(8, 8), (16, 8), (8, 2), (28, 4), (8, 1), (40, 2)])
def test_decode(cuda, qdt, sdt, D, Hq, Hkv):
    gen = torch.Generator().manual_seed(Hq * D)
    lens = [1, 2, 0, 15, 16, 17, 31, 33, 64, 65, 127, 129, 257, 600]
    _close(*_attend(gen, lens, 1, Hq, Hkv, D, 16, qdt, sdt), "16")


@pytest.mark.parametrize("ps", [1, 3, 8, 24, 32, 64, 100, 128, 1000])
@pytest.mark.parametrize("L", [1, 5])
def test_page_sizes(cuda, ps, L):
    gen = torch.Generator().manual_seed(ps)
    lens = [L, 77, 300, ps, 2 * ps + 1 if ps < 500 else 1001]
    _close(*_attend(gen, [max(n, L) for n in lens], L, 8, 2, 128, ps, BF, BF), "causal")
    _close(*_attend(gen, [max(n, L) for n in lens], L, 8, 2, 64, ps, HF, HF, causal=False), "full")


@pytest.mark.parametrize("D", [64, 128])
@pytest.mark.parametrize("qdt", [BF, HF, FF])
@pytest.mark.parametrize("L,Hq,Hkv", [(2, 8, 8), (3, 8, 2), (5, 32, 4), (8, 8, 1), (13, 28, 4), (33, 8, 2), (63, 4, 2), (64, 4, 2),
                                      (100, 8, 2), (200, 4, 1), (129, 16, 2)])
def test_more_tokens(cuda, D, qdt, L, Hq, Hkv):
    gen = torch.Generator().manual_seed(L * D)
    lens = [L, L + 1, L + 40, 3 * L + 100]
    _close(*_attend(gen, lens, L, Hq, Hkv, D, 16, qdt, HF if qdt == HF else BF), "causal")
    _close(*_attend(gen, lens, L, Hq, Hkv, D, 16, qdt, HF if qdt == HF else BF, causal=False), "full")


@pytest.mark.parametrize("L", [1, 4, 70])
def test_holes_empty_rows_and_long_tables(cuda, L):
    """Pages that are missing, requests shorter than the call's tokens (whose first rows see nothing),
    empty requests, tables wider than any request and requests longer than their table."""
    gen = torch.Generator().manual_seed(L)
    lens = [0, 1, L // 2, L, 100, 300]
    for ps in (16, 24):
        got, want, bound = _attend(gen, lens, L, 8, 2, 128, ps, BF, BF, holes=True, width=40)
        _close(got, want, bound, ps)
        assert (got[0] == 0).all()
        if L > 1:
            assert (got[1, :, :L - 1] == 0).all() and (got[1, :, L - 1] != 0).any()
    P, bt, cl = random_table(gen, [100, 50], 16)
    kp, vp, ks, vs = random_pools(gen, P, 2, 16, 128, BF)
    q = torch.randn(2, 8, L, 128, generator=gen).to(BF).cuda()
    cl = torch.tensor([400, 50], dtype=torch.int32, device="cuda")  # the table ends at 112 keys
    got = lib.paged_attention(q, kp, vp, bt, cl, 16, ks, vs, mask="causal", out_dtype=BF)
    _close(got, *attend64(q, kp, vp, ks, vs, bt, cl, 16))
    bt[:, :] = -1
    assert (lib.paged_attention(q, kp, vp, bt, cl, 16, ks, vs, out_dtype=BF) == 0).all()
    bt[:, :] = P  # past the pool
    assert (lib.paged_attention(q, kp, vp, bt, cl, 16, ks, vs, out_dtype=BF) == 0).all()
    with pytest.raises(RuntimeError, match="null tensor pointer"):  # as every page type's table without pages
        lib.paged_attention(q, kp, vp, bt[:, :0].contiguous(), cl, 16, ks, vs, out_dtype=BF)


@pytest.mark.parametrize("L,D", [(1, 128), (1, 64), (5, 128), (66, 128), (66, 64)])
def test_what_no_row_sees_has_no_influence(cuda, L, D):
    """Rows behind the last token, unmapped pages and other requests' pages hold NaN and infinities."""
    gen = torch.Generator().manual_seed(D + L)
    lens = [L, 21 + L, 200, 333]
    P, bt, cl = random_table(gen, lens, 16)
    kp, vp, ks, vs = random_pools(gen, P, 2, 16, D, BF)
    q = torch.randn(4, 8, L, D, generator=gen).to(BF).cuda()
    clean = lib.paged_attention(q, kp, vp, bt, cl, 16, ks, vs, mask="causal", out_dtype=BF)
    used = torch.zeros(P, 16, dtype=torch.bool, device="cuda")
    for b, n in enumerate(lens):
        key = torch.arange(n, device="cuda")
        used[bt[b].long()[key // 16], key % 16] = True
    bad = torch.tensor([float("nan"), float("inf"), -float("inf"), float("nan")], device="cuda").to(BF)
    for x in (ks, vs):
        x.copy_(torch.where(used[:, None, :, None], x, bad[:x.shape[-1]]))
    for x in (kp, vp):
        x.copy_(torch.where(used[:, None, :, None], x, torch.full_like(x, 0xFF)))
    dirty = lib.paged_attention(q, kp, vp, bt, cl, 16, ks, vs, mask="causal", out_dtype=BF)
    assert torch.equal(clean, dirty)


def test_nan_shows_only_where_it_is_seen(cuda):
    gen = torch.Generator().manual_seed(1)
    P, bt, cl = random_table(gen, [90, 90], 16)
    kp, vp, ks, vs = random_pools(gen, P, 2, 16, 128, BF)
    q = torch.randn(2, 4, 1, 128, generator=gen).to(BF).cuda()
    vs[bt[0, 2], 0, 3, 2:] = float("nan")  # request 0, kv head 0, elements 64 and up
    got = lib.paged_attention(q, kp, vp, bt, cl, 16, ks, vs, mask="causal", out_dtype=BF)
    assert got[0, :2, :, 64:].isnan().all() and not got[0, :2, :, :64].isnan().any()
    assert not got[0, 2:].isnan().any() and not got[1].isnan().any()
    ks[bt[1, 1], 1, 0, 0] = float("nan")
    got = lib.paged_attention(q, kp, vp, bt, cl, 16, ks, vs, mask="causal", out_dtype=BF)
    assert got[1, 2:].isnan().all() and not got[1, :2].isnan().any()


@pytest.mark.parametrize("sdt,size", [(BF, 2.0 ** -30), (BF, 2.0 ** 40), (HF, 2.0 ** -12), (HF, 2.0 ** 10)])
def test_values_of_any_size(cuda, sdt, size):
    """The weights held in 16 bits are relative to the largest contribution, not to the largest value."""
    gen = torch.Generator().manual_seed(9)

    def pools(P):
        kp, vp, ks, vs = random_pools(gen, P, 2, 16, 128, FF)
        # tokens whose values differ by 2^20 in size, the small ones far more attended to
        fade = torch.where(torch.rand(P, 1, 16, 1, generator=gen) < 0.5, 1.0, 2.0 ** (-20 if sdt == BF else -6)).cuda()
        return kp, vp, (ks * 0.2).to(sdt), (vs * fade * size).to(sdt)
    for L in (1, 5):
        _close(*_attend(gen, [5, 70, 400], L, 8, 2, 128, 16, BF, sdt, out=FF, pools=pools), f"{L} tokens")


def test_large_and_small_queries(cuda):
    """bf16 queries beyond float16's range on both sides."""
    gen = torch.Generator().manual_seed(11)
    for qscale in (2.0 ** 30, 2.0 ** -30):
        for L in (1, 5, 70):
            got, want, bound = _attend(gen, [L, 150], L, 8, 2, 128, 16, BF, BF, scale=0.1 / qscale, qscale=qscale, out=FF)
            _close(got, want, bound, f"{qscale} {L}")


@pytest.mark.parametrize("scale", [0.0, -0.125, 1.0])
@pytest.mark.parametrize("L", [1, 70])
def test_softmax_scales(cuda, scale, L):
    gen = torch.Generator().manual_seed(13)
    _close(*_attend(gen, [L, 200], L, 8, 2, 128, 16, BF, BF, scale=scale, out=FF), scale)


def test_scores_that_climb_and_fall(cuda):
    """Keys in rising and falling order of their score: the running maximum moves at every step, or never."""
    for sign in (1, -1):
        for L in (1, 4):
            n, D = 1500, 128
            kp = torch.zeros(n // 16 + 1, 1, 16, D // 2, dtype=torch.uint8, device="cuda")
            ramp = torch.arange(kp.shape[0] * 16, device="cuda").float() / n * 40 * sign
            ks = torch.zeros(kp.shape[0], 1, 16, 4, device="cuda", dtype=HF)
            ks[..., 1] = ramp.view(-1, 1, 16) / 64
            gen = torch.Generator().manual_seed(2)
            vp = torch.randint(0, 256, kp.shape, generator=gen, dtype=torch.uint8).cuda()
            vs = torch.rand(ks.shape, generator=gen).to(HF).cuda()
            bt = torch.arange(kp.shape[0], dtype=torch.int32, device="cuda")[None]
            cl = torch.tensor([n], dtype=torch.int32, device="cuda")
            q = torch.ones(1, 4, L, D, device="cuda", dtype=HF)
            got = lib.paged_attention(q, kp, vp, bt, cl, 16, ks, vs, scale=1.0, mask="causal")
            _close(got, *attend64(q, kp, vp, ks, vs, bt, cl, 16, 1.0), f"{sign} {L}")


@pytest.mark.parametrize("B,n,Hq,Hkv,L", [(1, 20000, 8, 1, 1), (2, 9000, 16, 2, 1), (1, 5000, 8, 2, 5), (300, 40, 8, 2, 1)])
def test_long_and_many(cuda, B, n, Hq, Hkv, L):
    gen = torch.Generator().manual_seed(n)
    lens = torch.randint(n // 2, n + 1, (B,), generator=gen).tolist()
    _close(*_attend(gen, lens, L, Hq, Hkv, 128, 16, BF, BF), f"{B} {n}")


def test_same_result_twice(cuda):
    """No sum depends on which thread block is first."""
    gen = torch.Generator().manual_seed(4)
    P, bt, cl = random_table(gen, [6000, 1234, 3000], 16)
    kp, vp, ks, vs = random_pools(gen, P, 4, 16, 128, BF)
    for L in (1, 5):
        q = torch.randn(3, 16, L, 128, generator=gen).to(BF).cuda()
        first = lib.paged_attention(q, kp, vp, bt, cl, 16, ks, vs, mask="causal")
        for _ in range(10):
            assert torch.equal(first, lib.paged_attention(q, kp, vp, bt, cl, 16, ks, vs, mask="causal"))


def test_query_layouts_and_outputs(cuda):
    """q as a transposed view, an output given by the caller, and what is refused."""
    gen = torch.Generator().manual_seed(6)
    P, bt, cl = random_table(gen, [50, 90], 16)
    kp, vp, ks, vs = random_pools(gen, P, 2, 16, 128, BF)
    q = torch.randn(2, 3, 8, 128, generator=gen).to(BF).cuda().transpose(1, 2)
    want = lib.paged_attention(q.contiguous(), kp, vp, bt, cl, 16, ks, vs, mask="causal", out_dtype=BF)
    out = torch.empty_like(want)
    got = lib.paged_attention(q, kp, vp, bt.long(), cl.long(), 16, ks, vs, mask="causal", out=out)
    assert got is out and torch.equal(out, want)
    call = lambda **k: lib.paged_attention(k.get("q", q), k.get("kp", kp), k.get("vp", vp), bt, cl, k.get("ps", 16),  # noqa: E731
                                           k.get("ks", ks), k.get("vs", vs), mask="causal", out=k.get("out"))
    for wrong in (dict(out=out[:, :, :, ::2]), dict(out=out[:1]), dict(ps=32), dict(ks=None), dict(vs=vs[..., :2]),
                  dict(vs=vs.half()), dict(q=q[..., :64]), dict(vp=vp[:-1]), dict(kp=kp.to(torch.int8))):
        with pytest.raises((RuntimeError, AssertionError)):
            call(**wrong)
    x = torch.randn(1, 1, 2, 128, device="cuda").to(BF)
    rope, pos, slot = RoPE(128, 4, device="cuda"), torch.zeros(1, 1, dtype=torch.int32, device="cuda"), torch.zeros(1, device="cuda").long()
    for w, more in (((torch.ones(128, device="cuda"), None), {}), ((None, None), dict(key_scales=ks.half(), value_scales=vs.half())),
                    ((None, None), dict(key_scales=None, value_scales=None))):
        with pytest.raises(RuntimeError):
            qk_norm_rope_write(x, x, x, *w, rope, pos, kp, vp, slot, **{"key_scales": ks, "value_scales": vs, **more})
    with pytest.raises(RuntimeError, match="uint8|evict|pages"):
        lib.evict_tokens(kp, vp, bt, cl, torch.zeros(2, 2, 200, device="cuda"), 8, key_scales=ks, value_scales=vs)
    with pytest.raises(RuntimeError):
        lib.read_slots(torch.zeros(2, 2, device="cuda").long(), kp, vp, ks, vs)
    with pytest.raises(RuntimeError):
        lib.read_slots(slot, kp, vp, ks, vs, torch.int8)
    k, v = lib.read_slots(slot[:0], kp, vp, ks, vs)
    assert k.shape == (0, 2, 128) and k.dtype == BF


def test_other_streams_and_captured_calls(cuda):
    """Append, attention and read back captured into a graph, replayed on new inputs beside another
    graph and after larger eager calls; and on a stream of their own."""
    gen = torch.Generator().manual_seed(8)
    Hq, Hkv, D, ps = 8, 2, 128, 16
    rope = RoPE(D, 4000, device="cuda")

    def problem(n, B):
        P, bt, cl = random_table(gen, [n] * B, ps)
        pools = random_pools(gen, P, Hkv, ps, D, BF)
        qkv = torch.randn(B, 1, (Hq + 2 * Hkv) * D, generator=gen).to(BF).cuda()
        pos = torch.full((B, 1), n - 1, dtype=torch.int32, device="cuda")
        slots = bt.long()[:, (n - 1) // ps] * ps + (n - 1) % ps
        return dict(bt=bt, cl=cl, pools=pools, qkv=qkv, pos=pos, slots=slots)

    def step(x):
        q, k, v = (y.view(y.shape[0], 1, -1, D) for y in x["qkv"].split([Hq * D, Hkv * D, Hkv * D], -1))
        kp, vp, ks, vs = x["pools"]
        q = qk_norm_rope_write(q, k, v, None, None, rope, x["pos"], kp, vp, x["slots"], key_scales=ks, value_scales=vs)
        out = lib.paged_attention(q, kp, vp, x["bt"], x["cl"], ps, ks, vs, mask="causal", out_dtype=BF)
        return out, *lib.read_slots(x["slots"], kp, vp, ks, vs)

    problems = [problem(3000, 2), problem(900, 3)]
    [step(x) for x in problems]
    graphs, outs = [], []
    for x in problems:
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            outs.append(step(x))
        graphs.append(g)
    step(problem(3500, 40))
    for x in problems:
        x["qkv"].copy_(torch.randn(x["qkv"].shape, generator=gen).to(BF))
    torch.cuda.synchronize()
    side = [torch.cuda.Stream() for _ in graphs]
    for _ in range(3):
        for g, s in zip(graphs, side):
            with torch.cuda.stream(s):
                g.replay()
    torch.cuda.synchronize()
    replayed = [[t.clone() for t in o] for o in outs]
    stream = torch.cuda.Stream()
    with torch.cuda.stream(stream):
        eager = [step(x) for x in problems]
    stream.synchronize()
    for r, e in zip(replayed, eager):
        assert all(torch.equal(a, b) for a, b in zip(r, e))


def test_host_caches(cuda):
    """A pool with kv_bits=4: a request cache and a batch of them, prompt then tokens, against the same
    rows attended to in 64 bits."""
    gen = torch.Generator().manual_seed(12)
    H, D, ps = 2, 128, 16
    pool = lib.TinyKvPagedPool(page_size=ps, kv_bits=4, kv_group_size=64, device="cuda")
    caches = [lib.TinyKvPagedCache(pool) for _ in range(2)]
    rows = {0: [], 1: []}
    for i, S in ((0, 37), (1, 18)):
        k, v = (torch.randn(1, H, S, D, generator=gen).to(BF).cuda() for _ in range(2))
        caches[i].update_and_fetch_paged(k, v)
        rows[i].append((k, v))
    batch = lib.BatchingKvCache(2, 100)
    for i in (0, 1):
        batch.add_request(caches[i], i)
    k, v = (torch.randn(2, H, 3, D, generator=gen).to(BF).cuda() for _ in range(2))
    meta = batch.update_and_fetch_paged(k, v, mask="causal")
    for i in (0, 1):
        rows[i].append((k[i:i + 1], v[i:i + 1]))
        dense = [torch.cat([r[j] for r in rows[i]], 2) for j in (0, 1)]
        for got, want in zip(caches[i].gather_dense(), dense):
            held = values64(*pack(*quantise(want, BF), BF)).float()
            assert torch.equal(got.cpu(), held)
    q = torch.randn(2, 8, 3, D, generator=gen).to(BF).cuda()
    out = lib.paged_attention(q, meta.key_pages, meta.value_pages, meta.block_table, meta.context_lens, ps, meta.key_scales,
                              meta.value_scales, mask="causal", out_dtype=BF)
    _close(out, *attend64(q, meta.key_pages, meta.value_pages, meta.key_scales, meta.value_scales, meta.block_table,
                          meta.context_lens, ps))
    with pytest.raises(RuntimeError):
        caches[0].evict(torch.zeros(1, H, 64, device="cuda"), 8)
    assert caches[0].offset == 40


def test_a_generation_over_the_device_table(cuda):
    """Append, attend, verify a few tokens and rewind over a DevicePageTable, all in 4 bits; every step
    against 64 bits over the rows that the pool then holds."""
    gen = torch.Generator().manual_seed(15)
    B, Hq, Hkv, D, ps, cap = 3, 8, 2, 64, 16, 64
    table = lib.DevicePageTable(B, 16, ps, cap)
    kp, vp, ks, vs = _empty_pools(cap, Hkv, ps, D, HF)
    rope = RoPE(D, 300, device="cuda")
    at = torch.zeros(B, dtype=torch.long)
    for L, back in ((70, 0), (1, 0), (1, 0), (5, 3), (1, 0), (4, 1), (1, 0)):
        slots = table.append(torch.full((B,), L, dtype=torch.int32, device="cuda"))
        qkv = torch.randn(B, L, (Hq + 2 * Hkv) * D, generator=gen).to(HF).cuda()
        q, k, v = (x.view(B, L, -1, D) for x in qkv.split([Hq * D, Hkv * D, Hkv * D], -1))
        pos = (at[:, None] + torch.arange(L)).int().cuda()
        q = qk_norm_rope_write(q, k, v, None, None, rope, pos, kp, vp, slots, key_scales=ks, value_scales=vs)
        out = lib.paged_attention(q, kp, vp, table.block_table, table.context_lens, ps, ks, vs, mask="causal", out_dtype=HF)
        _close(out, *attend64(q, kp, vp, ks, vs, table.block_table, table.context_lens, ps), f"{L}")
        held = lib.read_slots(slots, kp, vp, ks, vs)[0]
        _, s, _ = quantise(rope.apply(k, pos).flatten(0, 1), HF)
        step = torch.from_numpy(np.repeat(s, 64, -1)).cuda()
        assert ((held.float() - rope.apply(k, pos).flatten(0, 1).float()).abs() <= step * (0.5 + 2.0 ** -9) + 2.0 ** -8).all()
        table.rewind(torch.full((B,), back, dtype=torch.int32, device="cuda"))
        at += L - back
    table.check_status()
    assert nv.device_error(torch.device("cuda:0")) == 0


# ---------------------------------------------------------------------------
# calls in company, odd addresses, large pools
# ---------------------------------------------------------------------------
@pytest.mark.parametrize("L", [1, 5, 70])
@pytest.mark.parametrize("qdt", [BF, HF, FF])
def test_odd_addresses(cuda, L, qdt):
    """Queries and outputs that start on no vector's boundary."""
    gen = torch.Generator().manual_seed(21)
    P, bt, cl = random_table(gen, [L, 100 + L], 16)
    kp, vp, ks, vs = random_pools(gen, P, 2, 16, 128, HF if qdt == HF else BF)
    n = 2 * 8 * L * 128
    q = torch.randn(n + 3, generator=gen).to(qdt).cuda()[3:].view(2, 8, L, 128)
    out = torch.zeros(n + 5, dtype=qdt, device="cuda")[5:].view(2, 8, L, 128)
    want = attend64(q, kp, vp, ks, vs, bt, cl, 16)
    _close(lib.paged_attention(q, kp, vp, bt, cl, 16, ks, vs, mask="causal", out_dtype=qdt), *want)
    lib.paged_attention(q, kp, vp, bt, cl, 16, ks, vs, mask="causal", out=out)
    _close(out, *want)


@pytest.mark.parametrize("sdt", [BF, HF])
def test_captured_prompts(cuda, sdt):
    """Prompts captured into graphs, replayed on new queries, pages and lengths beside one another."""
    gen = torch.Generator().manual_seed(22)

    def problem(lens, L):
        P, bt, cl = random_table(gen, lens, 16, width=40)
        return [torch.randn(len(lens), 8, L, 128, generator=gen).to(sdt).cuda(), *random_pools(gen, P, 2, 16, 128, sdt), bt, cl]

    def call(x):
        q, kp, vp, ks, vs, bt, cl = x
        return lib.paged_attention(q, kp, vp, bt, cl, 16, ks, vs, mask="causal", out_dtype=sdt)

    problems = [problem([200, 90], 70), problem([600], 300)]
    [call(x) for x in problems]
    graphs, outs = [], []
    for x in problems:
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            outs.append(call(x))
        graphs.append(g)
    call(problem([630, 600, 500, 400], 128))
    for x, n in zip(problems, (150, 333)):
        x[0].copy_(torch.randn(x[0].shape, generator=gen).to(sdt))
        x[3].mul_(1.5)
        x[6][-1] = n
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in graphs]
    for _ in range(3):
        for g, s in zip(graphs, streams):
            with torch.cuda.stream(s):
                g.replay()
    torch.cuda.synchronize()
    for x, o in zip(problems, outs):
        q, kp, vp, ks, vs, bt, cl = x
        _close(o, *attend64(q, kp, vp, ks, vs, bt, cl, 16))


def test_one_workspace_for_every_kind_of_call(cuda):
    """4-bit, 16-bit and scored calls take turns over a stream's workspace: what each leaves, the next finds."""
    gen = torch.Generator().manual_seed(23)
    P, bt, cl = random_table(gen, [2500, 700], 16)
    kp, vp, ks, vs = random_pools(gen, P, 2, 16, 128, BF)
    k16, v16 = (torch.randn(P, 2, 16, 128, generator=gen).to(BF).cuda() for _ in range(2))
    mass = torch.zeros(2, 2, bt.shape[1] * 16, device="cuda")
    calls = []
    for L in (1, 5, 70):
        q = torch.randn(2, 8, L, 128, generator=gen).to(BF).cuda()
        calls += [lambda q=q: lib.paged_attention(q, kp, vp, bt, cl, 16, ks, vs, mask="causal"),
                  lambda q=q: lib.paged_attention(q, k16, v16, bt, cl, 16, mask="causal")]
    calls.append(lambda: lib.paged_attention(q[:, :, :1].contiguous(), k16, v16, bt, cl, 16, mask="causal", key_mass=mass))
    alone = [c() for c in calls]
    for order in range(3):
        for i in torch.randperm(len(calls), generator=gen).tolist():
            assert torch.equal(calls[i](), alone[i]), (order, i)


def test_threads_on_one_stream(cuda):
    import threading

    gen = torch.Generator().manual_seed(24)
    P, bt, cl = random_table(gen, [3000, 2000], 16)
    kp, vp, ks, vs = random_pools(gen, P, 2, 16, 128, BF)
    qs = [torch.randn(2, 8, L, 128, generator=gen).to(BF).cuda() for L in (1, 1, 3, 70)]
    call = lambda q: lib.paged_attention(q, kp, vp, bt, cl, 16, ks, vs, mask="causal")  # noqa: E731
    want, bad = [call(q) for q in qs], []

    def work(i):
        for _ in range(20):
            if not torch.equal(call(qs[i]), want[i]):
                bad.append(i)

    threads = [threading.Thread(target=work, args=(i,)) for i in range(4)]
    [t.start() for t in threads]
    [t.join() for t in threads]
    assert not bad


def test_wide_tables_taken_in_parts(cuda):
    """Tables a million pages wide: the batch is taken in parts, whose requests are found by their own rows."""
    gen = torch.Generator().manual_seed(25)
    B, L, ps, D = 9, 64, 1024, 64
    lens = [64, 100, 65, 1030, 70, 2000, 64, 90, 1500]
    P, bt, cl = random_table(gen, lens, ps, width=1 << 20)
    kp, vp, ks, vs = random_pools(gen, P, 2, ps, D, HF)
    q = torch.randn(B, 8, L, D, generator=gen).to(HF).cuda()
    got = lib.paged_attention(q, kp, vp, bt, cl, ps, ks, vs, mask="causal", out_dtype=HF)
    _close(got, *attend64(q, kp, vp, ks, vs, bt, cl, ps))


def test_pools_past_four_gigabytes(cuda):
    """Rows behind 2^32 bytes and 2^31 elements: append, read back, attention of one token and of many."""
    gen = torch.Generator().manual_seed(26)
    P, Hkv, ps, D, n = 40000, 8, 256, 128, 700
    kp, vp = (torch.empty(P, Hkv, ps, D // 2, dtype=torch.uint8, device="cuda") for _ in range(2))
    ks, vs = (torch.empty(P, Hkv, ps, 4, dtype=BF, device="cuda") for _ in range(2))
    bt = torch.tensor([[P - 1, P - 5, P - 2]], dtype=torch.int32, device="cuda")
    cl = torch.tensor([n], dtype=torch.int32, device="cuda")
    key = torch.arange(n, device="cuda")
    slots = bt[0].long()[key // ps] * ps + key % ps
    q, k, v = (torch.randn(1, n, h, D, generator=gen).to(BF).cuda() for h in (32, Hkv, Hkv))
    rope = RoPE(D, n, device="cuda")
    rq = qk_norm_rope_write(q, k, v, None, None, rope, key.int()[None], kp, vp, slots, key_scales=ks, value_scales=vs)
    at = bt[0].long()
    small = [x[at].contiguous() for x in (kp, vp, ks, vs)]
    near = torch.arange(3, dtype=torch.int32, device="cuda")[None]
    gk, gv = lib.read_slots(slots, kp, vp, ks, vs)
    wk, wv = lib.read_slots(key, *small)
    assert torch.equal(gk, wk) and torch.equal(gv, wv) and (gv.float() - v[0].float()).abs().max() < 0.5
    for L in (1, 3, n):
        x = rq[:, :, n - L:].contiguous()
        far = lib.paged_attention(x, kp, vp, bt, cl, ps, ks, vs, mask="causal", out_dtype=BF)
        assert torch.equal(far, lib.paged_attention(x, *small[:2], near, cl, ps, *small[2:], mask="causal", out_dtype=BF))
    lib.write_slots(v[0], k[0], slots, kp, vp, ks, vs)
    assert torch.equal(lib.read_slots(slots, kp, vp, ks, vs)[0], gv)


def test_positions_and_slots_out_of_range(cuda):
    """Bad positions and slots are skipped and show in the device error word; nothing else is touched."""
    dev = torch.device("cuda:0")
    nv.device_error(dev)
    B, L, Hq, Hkv, D, ps, P = 1, 5, 4, 2, 128, 8, 2
    q, k, v = (torch.randn(B, L, h, D, device="cuda").to(BF) for h in (Hq, Hkv, Hkv))
    rope = RoPE(D, 16, device="cuda")
    pos = torch.tensor([[0, 16, -1, 3, 4]], dtype=torch.int32, device="cuda")
    slots = torch.tensor([3, 4, 5, P * ps, -7], device="cuda")
    pools = _empty_pools(P, Hkv, ps, D, BF)
    out = torch.full((B, Hq, L, D), 9.0, dtype=BF, device="cuda")
    qk_norm_rope_write(q, k, v, None, None, rope, pos, *pools[:2], slots, key_scales=pools[2], value_scales=pools[3], out=out)
    assert nv.device_error(dev) == 7 and nv.device_error(dev) == 0
    good = [0, 3, 4]
    assert torch.equal(out[0, :, good], rope.apply(q, pos.clamp(0, 15))[0, good].transpose(0, 1)) and (out[0, :, 1:3] == 9).all()
    before = [t.cpu() for t in _empty_pools(P, Hkv, ps, D, BF)]
    keys, _ = _expect_rows(rope.apply(k, pos.clamp(0, 15))[0, :1], slots[:1], before[0], before[2], ps)
    values, _ = _expect_rows(v[0, :3], slots[:3], before[1], before[3], ps)
    assert torch.equal(pools[0].cpu(), keys) and torch.equal(pools[1].cpu(), values)


def test_entry_point_without_a_workspace(cuda):
    gen = torch.Generator().manual_seed(27)
    P, bt, cl = random_table(gen, [900, 60], 16)
    kp, vp, ks, vs = random_pools(gen, P, 2, 16, 128, BF)
    for L in (1, 5):
        q = torch.randn(2, 8, L, 128, generator=gen).to(BF).cuda()
        out = torch.empty_like(q)
        nv.check(nv.lib().nvm_paged_attention_noalloc(
            q.data_ptr(), 2, kp.data_ptr(), vp.data_ptr(), nv.NVM_U4, ks.data_ptr(), vs.data_ptr(), 2, bt.data_ptr(),
            cl.data_ptr(), out.data_ptr(), 2, 2, 8, 2, L, 128, P, 16, bt.shape[1], 128 ** -0.5, 1, nv.stream_ptr(cuda)))
        assert torch.equal(out, lib.paged_attention(q, kp, vp, bt, cl, 16, ks, vs, mask="causal", out_dtype=BF))


def test_nan_queries_stay_in_their_rows(cuda):
    gen = torch.Generator().manual_seed(28)
    P, bt, cl = random_table(gen, [300], 16)
    kp, vp, ks, vs = random_pools(gen, P, 2, 16, 128, BF)
    for L in (1, 4):
        q = torch.randn(1, 8, L, 128, generator=gen).to(BF).cuda()
        clean = lib.paged_attention(q, kp, vp, bt, cl, 16, ks, vs, mask="causal")
        q[0, 2, 0, 5], q[0, 5, L - 1, 7] = float("nan"), float("inf")
        got = lib.paged_attention(q, kp, vp, bt, cl, 16, ks, vs, mask="causal")
        bad = torch.zeros(1, 8, L, dtype=torch.bool, device="cuda")
        bad[0, 2, 0], bad[0, 5, L - 1] = True, True
        assert got[bad].isnan().all() and torch.equal(got[~bad], clean[~bad])


@pytest.mark.parametrize("B,L", [(1, 1), (5, 1), (1, 6), (3, 4)])
@pytest.mark.parametrize("kv", ["u4", BF])
def test_fused_projections_are_read_in_place(cuda, B, L, kv, monkeypatch):
    """Views of one projection, of a decode step and of a prompt, are not copied, and give what copies give."""
    gen = torch.Generator().manual_seed(B + L)
    Hq, Hkv, D, ps, P = 8, 2, 128, 16, 4
    views = [x.view(B, L, -1, D) for x in torch.randn(B, L, (Hq + 2 * Hkv) * D, generator=gen).to(BF).cuda()
             .split([Hq * D, Hkv * D, Hkv * D], -1)]
    rope = RoPE(D, 64, device="cuda")
    pos = torch.randint(0, 64, (B, L), generator=gen).int().cuda()
    slots = torch.randperm(P * ps, generator=gen)[:B * L].cuda()

    def call(q, k, v):
        pools = _empty_pools(P, Hkv, ps, D, BF)
        if kv == "u4":
            q = qk_norm_rope_write(q, k, v, None, None, rope, pos, *pools[:2], slots, key_scales=pools[2], value_scales=pools[3])
            return [q, *pools]
        pages = [torch.zeros(P, Hkv, ps, D, dtype=BF, device="cuda") for _ in range(2)]
        return [qk_norm_rope_write(q, k, v, None, None, rope, pos, *pages, slots), *pages]

    want = call(*(x.clone() for x in views))
    from nano_vllm_b200.layers import qk_prep

    whole = qk_prep._token_rows

    def rows(x):
        got = whole(x)
        assert got[0].data_ptr() == x.data_ptr()
        return got

    monkeypatch.setattr(qk_prep, "_token_rows", rows)
    assert all(torch.equal(a, b) for a, b in zip(call(*views), want))


@pytest.mark.parametrize("sdt,qdt", [(BF, BF), (HF, BF), (HF, HF)])
def test_prompts_taken_in_parts(cuda, sdt, qdt):
    """Tables so wide that the unpacked pages of a batch pass the workspace's limit: parts of it, each with its
    own lengths, empty requests and holes among them."""
    gen = torch.Generator().manual_seed(30)
    lens = [128, 700, 0, 129, 400, 2000, 128]
    P, bt, cl = random_table(gen, lens, 32, holes=True, width=2048)
    kp, vp, ks, vs = random_pools(gen, P, 8, 32, 128, sdt)
    q = torch.randn(7, 16, 128, 128, generator=gen).to(qdt).cuda()
    got = lib.paged_attention(q, kp, vp, bt, cl, 32, ks, vs, mask="causal", out_dtype=qdt)
    _close(got, *attend64(q, kp, vp, ks, vs, bt, cl, 32))
    assert (got[2] == 0).all()
