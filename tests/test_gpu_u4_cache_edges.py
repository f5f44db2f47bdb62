"""The 4-bit cache's corners on the GPU."""

import pytest
import torch

import nano_vllm_b200 as lib
from nano_vllm_b200 import _native as nv
from nano_vllm_b200.layers.qk_prep import qk_norm_rope_write
from nano_vllm_b200.layers.rotary_embedding import RoPE
from u4_reference import random_pools, values64

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
