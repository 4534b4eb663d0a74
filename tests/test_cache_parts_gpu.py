"""A cache keeps what it was made with: its calls go by the tensors' addresses."""
import pytest
import torch

import flash_attn_with_score_b200 as F

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("name", ["k_codes", "v_codes", "k_scales", "v_scales", "pages", "heads", "dtype", "device", "_struct", "_plain"])
def test_parts_cannot_be_deleted(name):
    cache = F.KVCache4(2, 16, 2, 64)
    part = getattr(cache, name)
    with pytest.raises(AttributeError, match=name):
        delattr(cache, name)
    assert getattr(cache, name) is part
    x = torch.ones((1, 2, 3, 64), dtype=torch.float16, device="cuda")
    table, lengths = torch.zeros((1, 1), dtype=torch.int32, device="cuda"), torch.full((1,), 3, dtype=torch.int32, device="cuda")
    F.kv_cache_write(cache, x, x, table, lengths)
    # 7 codes of bf16(1 / 7) = 0.142578125, in fp16
    want = torch.full_like(x, 7 * 0.142578125)
    assert all(torch.equal(got, want) for got in F.kv_cache_read(cache, table, lengths, 3))
