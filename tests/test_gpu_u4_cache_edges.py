"""The 4-bit cache's corners on the GPU."""

import pytest
import torch

import nano_vllm_b200 as lib
from nano_vllm_b200 import _native as nv
from u4_reference import random_pools

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
