"""The 4-bit cache's corners on the GPU."""

import pytest
import torch

import nano_vllm_b200 as lib
from nano_vllm_b200 import _native as nv
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
