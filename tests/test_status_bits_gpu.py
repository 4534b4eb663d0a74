"""The bits of the status word: what raises one leaves the other as it is."""
import ctypes as C

import pytest
import torch

import flash_attn_with_score_b200 as F
from flash_attn_with_score_b200 import _lib

pytestmark = pytest.mark.gpu


def _bad_page():
    cache = F.KVCache4(2, 16, 1, 64)
    F.kv_cache_read(cache, torch.full((1, 1), 9, dtype=torch.int32, device="cuda"), torch.ones(1, dtype=torch.int32, device="cuda"), 1)


def _give_up():
    assert _lib.load().faws_selftest_wait_give_up(C.c_void_p(torch.cuda.current_stream().cuda_stream)) == 0


@pytest.mark.parametrize("first,then", [(_bad_page, _give_up), (_give_up, _bad_page)])
def test_both_bits(first, then):
    assert F.device_status() == 0
    first()
    one = F.device_status(reset=False)
    then()
    assert one in (1, 2) and F.device_status() == 3
    assert F.device_status() == 0
