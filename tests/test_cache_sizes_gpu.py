"""Rows of expanded tensors, more than 32 bits count: refused, not cut off."""
import pytest
import torch

import flash_attn_with_score_b200 as F

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("M", [2 ** 31, 2 ** 32 + 1, 2 ** 30 + 1])
def test_rows_beyond_32_bits(M):
    cache = F.KVCache4(2, 16, 2, 64)
    table = torch.arange(2, dtype=torch.int32, device="cuda").view(1, 2)
    lengths = torch.full((1,), 20, dtype=torch.int32, device="cuda")
    x = torch.ones((1, 2, 1, 64), dtype=torch.float16, device="cuda").expand(1, 2, M, 64)
    with pytest.raises((AssertionError, RuntimeError)):
        F.kv_cache_write(cache, x, x, table, lengths)
    with pytest.raises(AssertionError):
        F.kv_cache_read(cache, table, lengths, 2 ** 32 + 1)
    with pytest.raises(AssertionError):
        F.kv_cache_write(cache, x[:, :, :1], x[:, :, :1], table[:, :1].expand(1, 2 ** 32 + 2), lengths)
    torch.cuda.synchronize()
    assert not bool(cache.k_codes.any()) and not bool(cache.k_scales.any())
