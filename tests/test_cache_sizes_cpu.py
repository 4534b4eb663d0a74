"""Sizes of a call on the 4-bit cache that 32 bits or a grid do not count: refused before anything is launched."""
import ctypes as C

import pytest


@pytest.fixture(scope="module")
def lib():
    from flash_attn_with_score_b200 import build, _lib
    build.build()
    return _lib.load()


@pytest.mark.parametrize("B,Hk,rows,D", [
    (2 ** 30, 4, 1, 16), (2 ** 30 + 1, 4, 1, 128), (2 ** 31 - 1, 2, 1, 64), (2 ** 29, 4, 16, 128), (2 ** 31 - 1, 8, 3, 16),
    (2 ** 20, 2 ** 11, 129, 16), (2 ** 10, 2 ** 6, 2 ** 26, 128), (1, 2 ** 31 - 1, 129, 16)])
def test_more_blocks_than_a_grid_has(lib, B, Hk, rows, D):
    """A block of its own for each sequence and head, 8192 elements of its rows to a block at most."""
    from flash_attn_with_score_b200 import _lib
    assert B * Hk * -(-rows * D // 8192) > 2 ** 31 - 1 or B * Hk * -(-rows * D // 2048) > 2 ** 31 - 1
    cache = _lib.KVCache(4096, 4096, 4096, 4096, 4, 16, Hk, D, 0)
    batch = _lib.CacheBatch(4096, 4096, 0, B, 2)
    t = _lib.Tensor(4096, 0, 0, 0)
    for fn in (lib.faws_kv_cache_write, lib.faws_kv_cache_read):
        assert fn(C.byref(cache), C.byref(batch), C.byref(t), C.byref(t), rows, None) == -1
    p = _lib.Problem(B=B, Hq=Hk, Hk=Hk, M=rows, N=1, D=D, dtype=0, m_end=rows, sm_scale=1.0, q=t, out=t)
    assert lib.faws_attention_with_kv_cache(C.byref(p), C.byref(cache), C.byref(batch), 0, 0, 4096, 1 << 30, None) == -1
