"""Refusals of the 4-bit cache's operators, which need no GPU: nothing is launched for a bad argument."""
import ctypes as C

import pytest
import torch


@pytest.fixture(scope="module")
def lib():
    from flash_attn_with_score_b200 import build, _lib
    build.build()
    return _lib.load()


def _structs(**over):
    from flash_attn_with_score_b200 import _lib
    cache = dict(k_codes=4096, v_codes=4096, k_scales=4096, v_scales=4096, pages=4, page_size=16, Hk=2, D=64, dtype=0)
    batch = dict(page_table=4096, lengths=4096, table_stride=2, B=3, max_pages=2)
    prob = dict(B=3, Hq=4, Hk=2, M=1, N=1, D=64, dtype=0, m_end=1, sm_scale=1.0,
                q=_lib.Tensor(4096, 256, 64, 64), out=_lib.Tensor(4096, 256, 64, 64))
    for name, value in over.items():
        for d in (cache, batch, prob):
            if name in d:
                d[name] = value
                break
        else:
            raise KeyError(name)
    return _lib.KVCache(**cache), _lib.CacheBatch(**batch), _lib.Problem(**prob)


@pytest.mark.parametrize("over,status", [
    (dict(pages=0), -1), (dict(page_size=24), -1), (dict(page_size=8), -1), (dict(page_size=1 << 17), -1), (dict(k_codes=None), -1),
    (dict(v_scales=4104), -1), (dict(page_table=None), -1), (dict(lengths=None), -1), (dict(max_pages=0), -1),
    (dict(table_stride=-1), -1)])
def test_bad_cache_or_batch(lib, over, status):
    from flash_attn_with_score_b200 import _lib
    cache, batch, p = _structs(**over)
    t = _lib.Tensor(4096, 256, 64, 64)
    for fn in (lib.faws_kv_cache_write, lib.faws_kv_cache_read):
        assert fn(C.byref(cache), C.byref(batch), C.byref(t), C.byref(t), 1, None) == status
    assert lib.faws_attention_with_kv_cache(C.byref(p), C.byref(cache), C.byref(batch), 0, 0, 4096, 1 << 30, None) == status


def test_bad_head_dim_and_dtype(lib):
    from flash_attn_with_score_b200 import _lib
    t = _lib.Tensor(4096, 256, 64, 64)
    for field, value in (("D", 48), ("dtype", 2)):
        cache, batch, p = _structs()
        setattr(cache, field, value)
        assert lib.faws_kv_cache_write(C.byref(cache), C.byref(batch), C.byref(t), C.byref(t), 1, None) == -2


def test_bad_rows_and_attention_arguments(lib):
    from flash_attn_with_score_b200 import _lib
    cache, batch, p = _structs()
    t, none = _lib.Tensor(4096, 256, 64, 64), _lib.Tensor(None, 256, 64, 64)
    call = lambda q=p, window=0, sinks=0, ws=4096, n=1 << 30: lib.faws_attention_with_kv_cache(
        C.byref(q), C.byref(cache), C.byref(batch), window, sinks, ws, n, None)
    assert lib.faws_kv_cache_write(C.byref(cache), C.byref(batch), C.byref(t), C.byref(t), 0, None) == -1
    assert lib.faws_kv_cache_read(C.byref(cache), C.byref(batch), C.byref(none), C.byref(t), 1, None) == -1
    assert lib.faws_kv_cache_write(None, C.byref(batch), C.byref(t), C.byref(t), 1, None) == -1
    assert call(window=-1) == -1 and call(sinks=-1) == -1
    assert call(n=lib.faws_kv_cache_workspace_bytes(C.byref(p)) - 1) == -3
    assert call(ws=None) == -3 and call(ws=4100) == -3
    for over in (dict(Hq=3), dict(M=0), dict(q=none)):
        _, _, q = _structs(**over)
        assert call(q) == -1
    q = _structs()[2]
    q.Hk = 4  # not the cache's
    assert call(q) == -1
    q = _structs()[2]
    q.dtype = 1
    assert call(q) == -1


def test_more_rows_than_are_counted(lib):
    """B 1, two heads: 2^30 rows are the most, and the elements of a call's grid are bounded."""
    from flash_attn_with_score_b200 import _lib
    cache, batch, p = _structs(B=1, D=16)
    p.B, p.D = 1, 16
    t = _lib.Tensor(4096, 0, 0, 0)
    for rows in (2 ** 30 + 1, 2 ** 31 - 1):
        for fn in (lib.faws_kv_cache_write, lib.faws_kv_cache_read):
            assert fn(C.byref(cache), C.byref(batch), C.byref(t), C.byref(t), rows, None) == -1
        p.M = p.m_end = rows
        p.Hq = 2
        assert lib.faws_attention_with_kv_cache(C.byref(p), C.byref(cache), C.byref(batch), 0, 0, 4096, 1 << 30, None) == -1


def test_python_refusals():
    import flash_attn_with_score_b200 as F
    with pytest.raises(RuntimeError, match="CUDA"):
        F.KVCache4(2, 16, 2, 64, device="cpu")
    with pytest.raises(AssertionError, match="page_size"):
        F.KVCache4(2, 24, 2, 64, device="cpu")
    with pytest.raises(AssertionError, match="head_dim"):
        F.KVCache4(2, 16, 2, 48, device="cpu")
    with pytest.raises(TypeError, match="dtype"):
        F.KVCache4(2, 16, 2, 64, dtype=torch.float32, device="cpu")
    with pytest.raises(TypeError, match="KVCache4"):
        F.kv_cache_read(None, torch.zeros((1, 1), dtype=torch.int32), torch.zeros(1, dtype=torch.int32), 1)
