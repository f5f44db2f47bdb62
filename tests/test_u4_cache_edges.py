"""The 4-bit cache's corners without a GPU."""

import pytest
import torch

import nano_vllm_b200 as lib
from nano_vllm_b200 import _native as nv


@pytest.mark.parametrize("L", [1, 64, 512])
@pytest.mark.parametrize("D", [64, 128])
def test_workspace_of_an_empty_batch(L, D):
    """Any number of query rows, the ones that go through unpacked pages among them (from 256 a kv head)."""
    size = nv.lib().nvm_paged_attention_workspace_size
    empty, one = (size(B, 32, 8, L, D, 16, 500, nv.NVM_U4) for B in (0, 1))
    assert 0 <= empty <= one


@pytest.mark.parametrize("first,then", [(torch.float16, torch.bfloat16), (torch.bfloat16, torch.float16), (torch.bfloat16, torch.float32)])
@pytest.mark.parametrize("reserve", [None, 2])
def test_growth_keeps_scales_as_they_are(first, then, reserve):
    """Rows of another type do not change the type of the scales that are there: rounded to it they would stand
    for other values."""
    pool = lib.TinyKvPagedPool(page_size=4, kv_bits=4, kv_group_size=64, device="cpu", reserve_pages=reserve)
    pool.allocate_page()
    pool.grow()
    pool._ensure_page_storage(torch.zeros(1, 2, 1, 128, dtype=first))
    one = 1 + torch.finfo(first).eps
    pool.key_scales.fill_(one)
    pool.value_scales.fill_(-one)
    for _ in range(3):
        pool.allocate_page()
        pool.grow()
        pool._ensure_page_storage(torch.zeros(1, 2, 1, 128, dtype=then))
        assert pool.key_scales.dtype == pool.value_scales.dtype == first
        assert (pool.key_scales[0] == one).all() and (pool.value_scales[0] == -one).all()


@pytest.mark.parametrize("width", [1, 1000, 1 << 16, 1 << 20, (1 << 21) - 64])
@pytest.mark.parametrize("B", [1, 3, 64, 1 << 20])
def test_workspace_of_wide_tables(width, B):
    """Unpacked pages take at most 1 GiB of a batch and 8 GiB of one request, whatever the tables have room for."""
    rows = 16 * 128 * 128 * 2 + 16 * 128  # a request's queries, and a mark for each
    most = max(8 << 30, (1 << 30) + B * rows) + (16 << 20) + B * 64 + B * width * 256
    assert nv.lib().nvm_paged_attention_workspace_size(B, 16, 8, 128, 128, 1024, width, nv.NVM_U4) <= most
