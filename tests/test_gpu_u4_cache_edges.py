"""The 4-bit cache's corners on the GPU."""

import pytest
import torch

import nano_vllm_b200 as lib
from nano_vllm_b200 import _native as nv
from nano_vllm_b200.layers.qk_prep import qk_norm_rope_write
from nano_vllm_b200.layers.rotary_embedding import RoPE
from u4_bounds import attention, close
from u4_reference import random_pools, random_table, values64

pytestmark = pytest.mark.gpu
BF, HF, FF = torch.bfloat16, torch.float16, torch.float32


@pytest.mark.parametrize("L", [1, 64, 512])
def test_empty_batch(cuda, L):
    """No request: an empty result, through the entry with a workspace and the one without."""
    kp, vp, ks, vs = random_pools(torch.Generator().manual_seed(0), 4, 2, 16, 128, BF)
    q = torch.empty(0, 8, L, 128, dtype=BF, device="cuda")
    bt, cl = torch.empty(0, 9, dtype=torch.int32, device="cuda"), torch.empty(0, dtype=torch.int32, device="cuda")
    got = lib.paged_attention(q, kp, vp, bt, cl, 16, ks, vs, mask="causal", out_dtype=BF)
    assert got.shape == q.shape
    assert nv.lib().nvm_paged_attention_noalloc(
        q.data_ptr(), nv.NVM_BF16, kp.data_ptr(), vp.data_ptr(), nv.NVM_U4, ks.data_ptr(), vs.data_ptr(), nv.NVM_BF16,
        bt.data_ptr(), cl.data_ptr(), got.data_ptr(), nv.NVM_BF16, 0, 8, 2, L, 128, 4, 16, 9, 0.1, 1,
        nv.stream_ptr(q.device)) == nv.NVM_OK


@pytest.mark.parametrize("rows", [BF, FF])
@pytest.mark.parametrize("span", [1e36, 2e37, 3e38])
@pytest.mark.parametrize("D", [64, 128])
def test_groups_of_any_span_read_back(cuda, rows, span, D):
    """bfloat16 scales up to the greatest: what is written comes back within half a step."""
    gen = torch.Generator().manual_seed(1)
    T, Hkv, ps = 21, 2, 16
    x = torch.rand(T, Hkv, D, generator=gen)
    x[..., 0], x[..., 1], x[..., D - 2], x[..., D - 1] = 0, 1, 0, 1
    k, v = ((x * span).to(rows).cuda(), ((x - 0.5) * span).to(rows).cuda())
    kp, vp = (torch.zeros(2, Hkv, ps, D // 2, dtype=torch.uint8, device="cuda") for _ in range(2))
    ks, vs = (torch.zeros(2, Hkv, ps, D // 32, dtype=BF, device="cuda") for _ in range(2))
    slots = torch.arange(T, device="cuda")
    lib.write_slots(k, v, slots, kp, vp, ks, vs)
    for got, given, pages, scales in zip(lib.read_slots(slots, kp, vp, ks, vs, FF), (k, v), (kp, vp), (ks, vs)):
        sc = scales[slots // ps, :, slots % ps]
        want = values64(pages[slots // ps, :, slots % ps], sc)
        assert torch.equal(got, want.float())  # s * code + z, rounded once
        step = sc[..., 0::2].double().repeat_interleave(64, -1)
        # and half a step of what was given, but for roundings of the quotient and the span, 45 * 2^-24 of a step
        assert ((want - given.double()).abs() <= step * (0.5 + 45 * 2.0 ** -24)).all()


def test_read_back_over_every_exponent(cuda):
    """A scale of every power of two that bfloat16 has, subnormal ones too, and float16's."""
    for dtype, powers in ((BF, range(-133, 124)), (HF, range(-24, 12))):
        gen = torch.Generator().manual_seed(2)
        s = torch.tensor([2.0 ** e for e in powers], dtype=torch.float64).to(dtype)
        T = s.numel()
        kp = torch.randint(0, 256, (T, 1, 1, 64), generator=gen, dtype=torch.uint8).cuda()
        sc = torch.stack([s, -7 * s, s, torch.zeros_like(s)], -1).view(T, 1, 1, 4).cuda()
        got = lib.read_slots(torch.arange(T, device="cuda"), kp, kp, sc, sc, FF)[0]
        assert torch.equal(got, values64(kp, sc).float()[:, :, 0])


@pytest.mark.parametrize("kv", ["u4", BF, torch.int8])
@pytest.mark.parametrize("D", [64, 128])
@pytest.mark.parametrize("B,L,width,first", [(5, 1, 1, 0), (5, 1, 2, 0), (5, 1, 4, 1), (3, 4, 1, 0), (3, 4, 2, 2), (1, 1, 4, 3), (1, 7, 4, 1)])
def test_append_of_rows_off_the_vectors(cuda, kv, D, B, L, width, first):
    """Rows of a projection with a few more columns than the heads take, or that starts on no vector's boundary,
    give what their copies give."""
    gen = torch.Generator().manual_seed(B * L + D)
    Hq, Hkv, ps, P = 8, 2, 16, 4
    n = (Hq + 2 * Hkv) * D
    wide = torch.randn(B * L * (n + width) + first, generator=gen).to(BF).cuda()[first:].view(B, L, n + width)
    q, k, v = (x.view(B, L, -1, D) for x in wide[..., :n].split([Hq * D, Hkv * D, Hkv * D], -1))
    w = [torch.randn(D, generator=gen).to(BF).cuda() for _ in range(2)]
    rope = RoPE(D, 64, device="cuda")
    pos = torch.randint(0, 64, (B, L), generator=gen).int().cuda()
    slots = torch.randperm(P * ps, generator=gen)[:B * L].cuda()

    def call(q, k, v):
        E = D // 2 if kv == "u4" else D
        pages = [torch.zeros(P, Hkv, ps, E, dtype=torch.uint8 if kv == "u4" else kv, device="cuda") for _ in range(2)]
        sc = [None, None]
        if kv != BF:
            sc = [torch.ones(P, Hkv, ps, D // 32 if kv == "u4" else 1, dtype=BF, device="cuda") for _ in range(2)]
        got = qk_norm_rope_write(q, k, v, *w, rope, pos, *pages, slots, key_scales=sc[0], value_scales=sc[1])
        return [got, *pages, *(x for x in sc if x is not None)]

    for a, b in zip(call(q, k, v), call(q.clone(), k.clone(), v.clone())):
        assert torch.equal(a, b)


@pytest.mark.parametrize("kv", ["u4", BF])
def test_append_of_keys_and_values_laid_out_apart(cuda, kv):
    """Contiguous keys that start on no vector's boundary next to values that are a view of something wider."""
    gen = torch.Generator().manual_seed(6)
    B, L, Hq, Hkv, D, ps = 3, 4, 4, 2, 128, 16
    q = torch.randn(B, L, Hq, D, generator=gen).to(BF).cuda()
    k = torch.randn(B * L * Hkv * D + 1, generator=gen).to(BF).cuda()[1:].view(B, L, Hkv, D)
    v = torch.randn(B, L, 3 * Hkv * D, generator=gen).to(BF).cuda()[..., Hkv * D:2 * Hkv * D].view(B, L, Hkv, D)
    rope, pos = RoPE(D, 16, device="cuda"), torch.arange(L, device="cuda").expand(B, L)

    def call(q, k, v):
        E, dt = (D // 2, torch.uint8) if kv == "u4" else (D, BF)
        pages = [torch.zeros(1, Hkv, ps, E, dtype=dt, device="cuda") for _ in range(2)]
        sc = [torch.ones(1, Hkv, ps, 4, dtype=BF, device="cuda") for _ in range(2)] if kv == "u4" else [None, None]
        return [qk_norm_rope_write(q, k, v, None, None, rope, pos, *pages, torch.arange(B * L, device="cuda"), key_scales=sc[0],
                                   value_scales=sc[1]), *pages]

    for x, y in ((k, v), (v, k)):
        for a, b in zip(call(q, x, y), call(q, x.clone(), y.clone())):
            assert torch.equal(a, b)


def test_append_takes_any_kind_of_number_as_eps(cuda):
    import numpy as np

    x = torch.randn(1, 3, 2, 128, device="cuda").to(BF)
    w = torch.ones(128, dtype=BF, device="cuda")
    rope, pos = RoPE(128, 4, device="cuda"), torch.arange(3, device="cuda")[None]

    def call(eps):
        kp, vp = (torch.zeros(1, 2, 4, 128, dtype=BF, device="cuda") for _ in range(2))
        return qk_norm_rope_write(x, x, x, w, w, rope, pos, kp, vp, torch.arange(3, device="cuda"), eps=eps), kp

    want = call(0.5)
    for eps in (np.float32(0.5), np.float64(0.5), torch.tensor(0.5), np.asarray(0.5)):
        assert all(torch.equal(a, b) for a, b in zip(call(eps), want))


# ---------------------------------------------------------------------------
# attention
# ---------------------------------------------------------------------------
def _call(x, ps=16, causal=True, **kw):
    q, kp, vp, ks, vs, bt, cl = x
    return lib.paged_attention(q, kp, vp, bt, cl, ps, ks, vs, mask="causal" if causal else None, **kw)


def _problem(gen, lens, L, sdt=BF, qdt=None, Hq=8, Hkv=2, D=128, ps=16):
    P, bt, cl = random_table(gen, lens, ps)
    q = torch.randn(len(lens), Hq, L, D, generator=gen).to(qdt or sdt).cuda()
    return [q, *random_pools(gen, P, Hkv, ps, D, sdt), bt, cl]


@pytest.mark.parametrize("L,D", [(1, 128), (5, 128), (5, 64), (70, 64), (70, 128)])
@pytest.mark.parametrize("size", [2.0 ** 20, 2.0 ** 26, 2.0 ** 30, 2.0 ** 60])
@pytest.mark.parametrize("sign", [1, -1])
def test_scores_far_apart(cuda, L, D, size, sign):
    """Scores beyond 2^31, where fp32 has no fractions left: a row is the value of the key with the largest."""
    gen = torch.Generator().manual_seed(41)
    x = _problem(gen, [L, 70 + L, 900], L, BF, FF, D=D)
    x[0] *= size
    got = _call(x, out_dtype=FF, scale=sign * 0.1)
    want, rows, prompts = attention(*x, 16, sign * 0.1)
    # how far a score may be off (2^-20 of its terms, and of a float32 query's 11 bits; from 256 rows a kv head of the
    # keys' too) moves weights between keys that are that close: the output then lies between their values
    t = torch.full_like(want[..., 0], float("inf"))
    for b, n in enumerate([L, 70 + L, 900]):
        key = torch.arange(n, device="cuda")
        page = x[5][b].long()[key // 16]
        for h in range(8):
            k = values64(x[1][page, h // 4, key % 16], x[3][page, h // 4, key % 16])
            s = x[0][b, h].double() @ k.T * (sign * 0.1)
            err = 0.1 * (x[0][b, h].double().abs() @ k.abs().T).amax(-1) * 2.0 ** -9 + 2.0 ** -18 * s.abs().amax(-1)
            s = s.masked_fill(key > torch.arange(L, device="cuda")[:, None] + n - L, float("-inf"))
            two = s.topk(min(2, n), -1).values
            gap = two[:, 0] - two[:, -1] if n > 1 else torch.full_like(err, float("inf"))
            gap[two[:, -1] == float("-inf")] = float("inf")
            t[b, h] = gap - 2 * err - 40
    clear = t > 0  # the largest is alone by more than that: its value, to what a value is held to
    assert clear.float().mean() > 0.1
    # (a scale of at most 0.33 times a code less 8, to 11 bits; or a value and a weight, each to 11 bits)
    close(got[clear], want[clear], 2.0 ** -10 * (want[clear].abs() + 1.4))
    assert got.isfinite().all() and got.abs().max() < 16


# ---------------------------------------------------------------------------
# many query rows (from 256 a kv head the pages are unpacked first)
# ---------------------------------------------------------------------------
@pytest.mark.parametrize("L", [5, 70, 200])
@pytest.mark.parametrize("sdt", [BF, HF])
@pytest.mark.parametrize("what", ["nan", "huge"])
@pytest.mark.parametrize("which", ["k", "v"])
@pytest.mark.parametrize("back", [1, 3])
def test_hidden_keys_have_no_influence_on_a_row(cuda, L, sdt, what, which, back):
    """A late token of a chunk holds NaN, or numbers 2^13 to 2^100 times the others: the rows before it are bit for
    bit what they are without it, those behind it what the definition says."""
    gen = torch.Generator().manual_seed(L + back)
    x = _problem(gen, [L, L + 130, 300], L, sdt)
    clean = _call(x, out_dtype=FF)
    n = L + 130
    page, off = x[5][1, (n - back) // 16].item(), (n - back) % 16
    scales = x[3 if which == "k" else 4]
    if what == "nan":
        scales[page, 0, off, 2:] = float("nan")
    elif which == "k":  # met with small numbers of the queries, so that scores stay ordinary
        scales[page, 0, off, 2:] *= 2.0 ** (20 if sdt == BF else 13)
        x[0][1, :4, :, 64:] *= 2.0 ** (-20 if sdt == BF else -13)
        y = [t.clone() for t in x]
        y[3][page, 0, off, 2:] = 0
        clean[1, :4] = _call(y, out_dtype=FF)[1, :4]
    else:
        scales[page, 0, off, 2:] *= 2.0 ** (100 if sdt == BF else 13)
    got = _call(x, out_dtype=FF)
    hidden = torch.ones(3, 8, L, dtype=torch.bool, device="cuda")
    hidden[1, :4, L - back:] = False
    assert torch.equal(got[hidden], clean[hidden])
    if what == "nan":
        rows = got[1, :4, L - back:]
        assert rows[..., 64:].isnan().all() and (rows.isnan().all() if which == "k" else not rows[..., :64].isnan().any())
    else:
        want, rows, prompts = attention(*x, 16)
        bound = rows if L < 64 or sdt == BF else torch.maximum(rows, prompts)
        close(got[~hidden], want[~hidden], bound[~hidden], "rows that see it")


@pytest.mark.parametrize("L", [5, 70])
@pytest.mark.parametrize("which", ["k", "v"])
def test_largest_float16_groups(cuda, L, which):
    """A group from 0 to 65504 has a scale of 4368 and a top of 65520, past float16's numbers."""
    gen = torch.Generator().manual_seed(3)
    x = _problem(gen, [L, L + 90], L, HF)
    page, off = x[5][1, 2].item(), 5
    i = 1 if which == "k" else 2
    x[i][page, 1, off, :32] = 0xF0
    x[i + 2][page, 1, off, 0], x[i + 2][page, 1, off, 1] = 4368, 0
    if which == "k":
        x[0][1, 4:, :, :64] *= 2.0 ** -14
    got = _call(x, out_dtype=FF)
    want, rows, prompts = attention(*x, 16)
    close(got, want, torch.maximum(rows, prompts))
    sees = torch.arange(L, device="cuda") + 90 >= 37
    close(got[1, 4:, sees], want[1, 4:, sees], rows[1, 4:, sees], "rows that see it")


@pytest.mark.parametrize("L,D", [(1, 128), (5, 128), (5, 64), (70, 128)])
@pytest.mark.parametrize("sdt,size", [(BF, 2.0 ** -90), (BF, 2.0 ** -30), (BF, 2.0 ** 40), (BF, 2.0 ** 100), (HF, 2.0 ** -10), (HF, 2.0 ** 11)])
def test_values_of_any_size_at_any_length(cuda, sdt, size, L, D):
    """Values 2^-20 (float16: 2^-6) of the others' size, and as often attended to."""
    gen = torch.Generator().manual_seed(9)
    x = _problem(gen, [L, 70 + L, 400], L, sdt, BF, D=D)
    small = torch.rand(x[4].shape[0], 1, 16, 1, generator=gen).cuda() < 0.5
    x[4].copy_((x[4].double() * torch.where(small, 2.0 ** (-20 if sdt == BF else -6), 1.0) * size).to(sdt))
    want, rows, prompts = attention(*x, 16)
    close(_call(x, out_dtype=FF), want, rows if L < 70 or sdt == BF else torch.maximum(rows, prompts))


@pytest.mark.parametrize("qdt,qsize", [(BF, 2.0 ** -60), (BF, 2.0 ** 60), (FF, 2.0 ** 60), (HF, 2.0 ** -10), (HF, 2.0 ** 12)])
@pytest.mark.parametrize("sdt", [BF, HF])
def test_some_query_rows_of_another_size(cuda, qdt, qsize, sdt):
    """Rows beyond float16's range, on either side, among ordinary ones leave those alone."""
    gen = torch.Generator().manual_seed(12)
    L = 70
    x = _problem(gen, [L, 150], L, sdt, qdt)
    clean = _call(x, out_dtype=FF)
    x[0][1, 2, 3], x[0][0, 5, 60] = x[0][1, 2, 3] * qsize, x[0][0, 5, 60] * qsize
    got = _call(x, out_dtype=FF)
    other = torch.zeros(2, 8, L, dtype=torch.bool, device="cuda")
    other[1, 2, 3], other[0, 5, 60] = True, True
    assert torch.equal(got[~other], clean[~other])
    want, rows, prompts = attention(*x, 16)
    # scores of 2^60: a row is its largest key's value, whatever the bound on a score's error (which passes 0.05)
    top = torch.maximum(rows, prompts).clamp(max=2.0 ** -8) if qsize > 2.0 ** 20 else torch.maximum(rows, prompts)
    close(got[other], want[other], top[other])


def _far_keys(x, gen, ps, n_keys, requests):
    """Makes some keys' values huge or tiny, some keys huge where the queries are small; returns [B, Hkv] of the first."""
    first = torch.full((x[0].shape[0], x[1].shape[1]), 1 << 30, device="cuda")
    for b in requests:
        n = int(x[6][b])
        for _ in range(n_keys):
            key, h = int(torch.randint(n, (1,), generator=gen)), int(torch.randint(x[1].shape[1], (1,), generator=gen))
            page = int(x[5][b, key // ps])
            if page < 0:
                continue
            x[4][page, h, key % ps] *= [2.0 ** 30, 2.0 ** -40][int(torch.randint(2, (1,), generator=gen))]
            first[b, h] = min(int(first[b, h]), key)
    return first


@pytest.mark.parametrize("L,Hq,Hkv,top", [(33, 16, 2, 3000), (64, 8, 2, 700), (200, 8, 2, 900), (300, 4, 4, 500), (5, 128, 2, 2000)])
@pytest.mark.parametrize("causal", [True, False])
def test_rows_of_either_kernel(cuda, L, Hq, Hkv, top, causal):
    """Some requests have keys that the unpacked pages leave out; calls of few and of many tokens, missing pages,
    eager and replayed from a graph on other keys."""
    gen = torch.Generator().manual_seed(L)
    lens = [top, L, top // 2 + L, 0, top - 77, L + 1]
    P, bt, cl = random_table(gen, lens, 16, holes=True)
    q = torch.randn(len(lens), Hq, L, 128, generator=gen).to(BF).cuda()
    x = [q, *random_pools(gen, P, Hkv, 16, 128, BF), bt, cl]
    plain = [t.clone() for t in x]

    def check(got, first):
        want, rows, prompts = attention(*x, 16, causal=causal)
        last = (torch.arange(L, device="cuda")[None] + cl[:, None] - L) if causal else cl[:, None].expand(-1, L) - 1
        sees = (last[:, None] >= first[:, :, None]).repeat_interleave(Hq // Hkv, 1)  # [B, Hq, L]
        close(got, want, torch.where(sees[..., None], rows, prompts))

    call = lambda: _call(x, out_dtype=FF, causal=causal)  # noqa: E731
    clean = call()
    check(clean, torch.full((len(lens), Hkv), 1 << 30, device="cuda"))
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = call()
    for requests in ((0,), (4, 2), range(len(lens)), ()):
        x[4].copy_(plain[4])
        first = _far_keys(x, gen, 16, 3, requests) if max(requests, default=0) < 3 or len(requests) == 2 else \
            _far_keys(x, gen, 16, 1, [b for b in requests if lens[b]])
        got = call()
        check(got, first)
        graph.replay()
        assert torch.equal(out, got)
    assert torch.equal(call(), clean)


def test_parts_of_a_batch_with_keys_left_out(cuda):
    """The tables are so wide that the batch is unpacked in parts."""
    gen = torch.Generator().manual_seed(43)
    lens = [128, 700, 150, 129, 400, 1000, 128]
    P, bt, cl = random_table(gen, lens, 32, width=2048)
    x = [torch.randn(7, 16, 128, 128, generator=gen).to(BF).cuda(), *random_pools(gen, P, 8, 32, 128, BF), bt, cl]
    first = _far_keys(x, gen, 32, 6, [1, 5, 6])
    x[0][4, 3, 17] *= 2.0 ** 20
    got = _call(x, 32, out_dtype=FF, scale=0.01)
    want, rows, prompts = attention(*x, 32, 0.01)
    last = torch.arange(128, device="cuda")[None] + cl[:, None] - 128
    sees = (last[:, None] >= first[:, :, None]).repeat_interleave(2, 1)
    sees[4, 3, 17] = True
    bound = torch.where(sees[..., None], rows, prompts)
    assert sees.any() and not sees.all()
    far = torch.zeros_like(sees)
    far[4, 3, 17] = True  # scores of 2^17: its own bound passes 0.05, and says nothing
    close(got[~far], want[~far], bound[~far])
    assert got[far].isfinite().all()


def test_more_row_blocks_than_a_launch_counts(cuda):
    """Many tokens under tables a million pages wide: the row blocks are taken in slices."""
    gen = torch.Generator().manual_seed(44)
    L, ps, D, lens = 512, 1024, 64, [512, 1500]
    P, bt, cl = random_table(gen, lens, ps, width=1 << 20)
    x = [torch.randn(2, 8, L, D, generator=gen).to(HF).cuda(), *random_pools(gen, P, 2, ps, D, HF), bt, cl]
    want, rows, _ = attention(*x, ps)
    close(_call(x, ps, out_dtype=HF), want, rows)


def test_prompts_under_tables_too_wide_to_unpack(cuda):
    gen = torch.Generator().manual_seed(45)
    L, ps, lens = 128, 1024, [128, 1500]
    P, bt, cl = random_table(gen, lens, ps, width=1 << 18)
    x = [torch.randn(2, 8, L, 128, generator=gen).to(BF).cuda(), *random_pools(gen, P, 8, ps, 128, BF), bt, cl]
    want, rows, _ = attention(*x, ps)
    close(_call(x, ps, out_dtype=BF), want, rows)


@pytest.mark.parametrize("L", [1, 5, 70])
@pytest.mark.parametrize("key", [3, 130, 394, 398])
def test_nan_of_a_key_with_no_weight_left(cuda, L, key):
    """A value that cannot be held is NaN for every row that sees it, also where its weight is below fp32's numbers."""
    gen = torch.Generator().manual_seed(46)
    x = _problem(gen, [400], L, BF)
    page = x[5][0, key // 16].item()
    x[4][page, 1, key % 16, 0] = float("nan")
    x[1][page, 1, key % 16], x[3][page, 1, key % 16] = 0, torch.tensor([0.0, -1.0] * 2, device="cuda").to(BF)  # K = -1
    x[0][0, 4:] = x[0][0, 4:].abs() + 1  # scores of -128 times the scale and less
    got = _call(x, out_dtype=FF, scale=4.0)
    sees = torch.arange(L, device="cuda") + 400 - L >= key
    assert got[0, 4:, sees, :64].isnan().all() and not got[0, 4:, sees, 64:].isnan().any()
    assert not got[0, 4:, ~sees].isnan().any() and not got[0, :4].isnan().any()


# ---------------------------------------------------------------------------
# groups and keys of unlike size
# ---------------------------------------------------------------------------
@pytest.mark.parametrize("L", [1, 5])
@pytest.mark.parametrize("sdt,ratio", [(BF, 2.0 ** -12), (BF, 2.0 ** -17), (BF, 2.0 ** -24), (BF, 2.0 ** -60), (BF, 2.0 ** 40), (HF, 2.0 ** -9)])
def test_groups_of_unlike_size(cuda, L, sdt, ratio):
    """A value's second group far below or above its first: each keeps its own precision."""
    gen = torch.Generator().manual_seed(31)
    x = _problem(gen, [L, 70, 700], L, sdt)
    x[4][..., 2:] *= ratio
    want, rows, _ = attention(*x, 16)
    close(_call(x, out_dtype=FF), want, rows, ratio)


@pytest.mark.parametrize("L", [1, 5])
def test_groups_whose_ratio_turns(cuda, L):
    """Keys whose first group is 2^30 times the second next to keys of the opposite kind, attended to by turns."""
    gen = torch.Generator().manual_seed(32)
    x = _problem(gen, [900, 300], L, BF)
    turn = torch.rand(x[4].shape[0], 1, 16, 1, generator=gen).cuda() < 0.5
    up = torch.tensor([1.0, 1.0, 2.0 ** -30, 2.0 ** -30], device="cuda")
    x[4].copy_((x[4].float() * torch.where(turn, up, up.flip(0))).to(BF))
    want, rows, _ = attention(*x, 16)
    close(_call(x, out_dtype=FF), want, rows)


@pytest.mark.parametrize("L", [1, 5, 70])
@pytest.mark.parametrize("sdt,value", [(BF, 2.0 ** 40), (BF, 2.0 ** 120), (HF, 30000.0), (BF, -2.0 ** -100)])
@pytest.mark.parametrize("groups", [slice(0, 4), slice(2, 4)])
def test_values_without_a_span(cuda, L, sdt, value, groups):
    """Groups whose elements are all alike have no scale, only an offset, of any size."""
    gen = torch.Generator().manual_seed(33)
    x = _problem(gen, [1000], L, sdt)
    x[4][..., groups] = torch.tensor([0.0, value] * 2, device="cuda")[groups].to(sdt)
    want, rows, prompts = attention(*x, 16)
    close(_call(x, out_dtype=FF), want, torch.maximum(rows, prompts) if L == 70 else rows)


# ---------------------------------------------------------------------------
# prompts in company
# ---------------------------------------------------------------------------
def test_prompts_without_a_workspace(cuda):
    """The entry without a workspace gives what the other one does, keys left out of the unpacked pages among them."""
    gen = torch.Generator().manual_seed(47)
    x = _problem(gen, [900, 130], 70, BF)
    for far in (False, True):
        if far:
            _far_keys(x, gen, 16, 2, [0, 1])
        q, kp, vp, ks, vs, bt, cl = x
        out = torch.empty_like(q)
        nv.check(nv.lib().nvm_paged_attention_noalloc(
            q.data_ptr(), 2, kp.data_ptr(), vp.data_ptr(), nv.NVM_U4, ks.data_ptr(), vs.data_ptr(), 2, bt.data_ptr(),
            cl.data_ptr(), out.data_ptr(), 2, 2, 8, 2, 70, 128, kp.shape[0], 16, bt.shape[1], 128 ** -0.5, 1, nv.stream_ptr(cuda)))
        assert torch.equal(out, _call(x, out_dtype=BF))


@pytest.mark.parametrize("sdt", [BF, HF])
def test_nan_queries_of_a_prompt_stay_in_their_rows(cuda, sdt):
    gen = torch.Generator().manual_seed(48)
    x = _problem(gen, [300, 90], 70, sdt)
    clean = _call(x, out_dtype=FF)
    bad = torch.zeros(2, 8, 70, dtype=torch.bool, device="cuda")
    for b, h, row, value in ((0, 2, 0, "nan"), (0, 5, 69, "inf"), (1, 7, 33, "-inf"), (1, 0, 64, "nan")):
        x[0][b, h, row, 5 * h] = float(value)
        bad[b, h, row] = True
    got = _call(x, out_dtype=FF)
    assert got[bad].isnan().all() and torch.equal(got[~bad], clean[~bad])


def test_prompts_of_both_kinds_take_turns(cuda):
    """Calls with and without keys left out, of other shapes and page types, over one workspace."""
    gen = torch.Generator().manual_seed(49)
    problems = [_problem(gen, [700, 90, 200], 70), _problem(gen, [2500], 300), _problem(gen, [1500, 64], 64, HF), _problem(gen, [400], 5)]
    _far_keys(problems[0], gen, 16, 3, [0, 2])
    _far_keys(problems[1], gen, 16, 1, [0])
    k16, v16 = (torch.randn(problems[0][1].shape[0], 2, 16, 128, generator=gen).to(BF).cuda() for _ in range(2))
    calls = [lambda x=x: _call(x, out_dtype=FF) for x in problems]
    calls.append(lambda: lib.paged_attention(problems[0][0], k16, v16, *problems[0][5:], 16, mask="causal"))
    alone = [c() for c in calls]
    for _ in range(4):
        for i in torch.randperm(len(calls), generator=gen).tolist():
            assert torch.equal(calls[i](), alone[i])
    streams = [torch.cuda.Stream() for _ in calls]
    for _ in range(3):
        outs = []
        for s, c in zip(streams, calls):
            s.wait_stream(torch.cuda.current_stream())
            with torch.cuda.stream(s):
                outs.append(c())
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(outs, alone))


def test_large_value_behind_a_far_score(cuda):
    """Scores of 2^28: a key 96 below the first, with values 2^120 times finer held before it, takes nothing from it."""
    B, D, ps = 300, 128, 16
    kp = torch.zeros(9, 1, ps, D // 2, dtype=torch.uint8, device="cuda")
    vp = kp.clone()
    ks = torch.zeros(9, 1, ps, 4, dtype=BF, device="cuda")
    vs = ks.clone()
    for page in (0, 8):  # keys 0 and 128, which one warp meets one after the other
        ks[page, 0, 0] = torch.tensor([1.0, 2.0 ** 21] * 2, device="cuda")
        vp[page, 0, 0] = 0x88
        vs[page, 0, 0] = torch.tensor([2.0 ** (-60 if page == 0 else 60), 2.0 ** 40 if page == 0 else 0.0] * 2, device="cuda")
    kp[0, 0, 0, :32] = 0x21  # 32 times 1 and 2
    bt = torch.arange(9, dtype=torch.int32, device="cuda").expand(B, -1)
    cl = torch.full((B,), 129, dtype=torch.int32, device="cuda")
    for L in (1, 5):
        q = torch.ones(B, 2, L, D, dtype=BF, device="cuda")
        got = lib.paged_attention(q, kp, vp, bt, cl, ps, ks, vs, scale=0.6931472, mask=None, out_dtype=FF)
        assert (got == 2.0 ** 40).all()
