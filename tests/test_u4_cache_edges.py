"""The 4-bit cache's corners without a GPU."""

import pytest

from nano_vllm_b200 import _native as nv


@pytest.mark.parametrize("L", [1, 64, 512])
@pytest.mark.parametrize("D", [64, 128])
def test_workspace_of_an_empty_batch(L, D):
    """Any number of query rows, the ones that go through unpacked pages among them (from 256 a kv head)."""
    size = nv.lib().nvm_paged_attention_workspace_size
    empty, one = (size(B, 32, 8, L, D, 16, 500, nv.NVM_U4) for B in (0, 1))
    assert 0 <= empty <= one
