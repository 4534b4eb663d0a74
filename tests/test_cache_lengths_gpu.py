"""Lengths that the page table has no room for: positions stay what they are, those behind the table do not exist."""
import pytest
import torch

from test_kv_cache_gpu import BF16, F16, Setup, _values

pytestmark = pytest.mark.gpu
PAGE = 16


def _tensors(cache):
    return cache.k_codes, cache.v_codes, cache.k_scales, cache.v_scales


@pytest.mark.parametrize("dtype,D", [(F16, 128), (BF16, 64), (BF16, 32), (F16, 16)])
@pytest.mark.parametrize("M,beyond", [(1, 1), (3, 1), (5, 3), (5, 5), (4, 9), (40, 2), (300, 290), (300, 1), (1, 2 ** 31 - 1 - 640)])
def test_rows_behind_the_table(dtype, D, M, beyond):
    """640 positions a sequence; the second sequence's last row is the table's last, the first one's lie up to `beyond` behind it."""
    import flash_attn_with_score_b200 as F
    cap, Hk = 640, 3
    s = Setup([cap, cap], Hk, D, dtype, PAGE)
    before = [t.clone() for t in _tensors(s.cache)]
    lengths = torch.tensor([cap + beyond, cap], dtype=torch.int32, device="cuda")
    g = torch.Generator().manual_seed(3)
    new = [torch.randn((2, Hk, M, D), generator=g).to(dtype).cuda() for _ in range(2)]
    F.kv_cache_write(s.cache, *new, s.table, lengths)
    assert F.device_status() == 2
    # rows on pages of the table are written where they belong, and nothing else is
    kept = max(0, M - beyond)  # of sequence 0, from position cap - kept on
    want = [t.clone() for t in (s.k, s.v)]
    for w, n in zip(want, new):
        w[0, :, cap - kept:] = n[0, :, :kept]
        w[1, :, cap - M:] = n[1]
    full = torch.full((2,), cap, dtype=torch.int32, device="cuda")
    for got, w in zip(F.kv_cache_read(s.cache, s.table, full, cap), want):
        assert torch.equal(got, _values(w).to(dtype))
    assert F.device_status() == 0
    same = torch.ones((s.cache.pages, PAGE), dtype=torch.bool, device="cuda")
    for b, first, n in ((0, cap - kept, kept), (1, cap - M, M)):
        for pos in range(first, first + n):
            same[s.table[b, pos // PAGE].long(), pos % PAGE] = False
    for was, now in zip(before, _tensors(s.cache)):
        assert torch.equal(was.transpose(1, 2)[same], now.transpose(1, 2)[same])
    # read back: NaN behind the table, every other row its own position's
    for got, w in zip(F.kv_cache_read(s.cache, s.table, lengths, M), want):
        assert bool(got[0, :, kept:].isnan().all())
        assert torch.equal(got[0, :, :kept], _values(w[0, :, cap - kept:cap]).to(dtype))
        assert torch.equal(got[1], _values(w[1, :, cap - M:]).to(dtype))
    assert F.device_status() == 2


@pytest.mark.parametrize("window,sinks", [(None, 0), (7, 0), (100, 20), (1, 0)])
@pytest.mark.parametrize("M,beyond", [(1, 1), (5, 3), (5, 5), (4, 900), (40, 2)])
def test_queries_behind_the_table(M, beyond, window, sinks):
    """They see a key that does not exist, their own: NaN.  Queries at positions of the table are what they are without them."""
    import flash_attn_with_score_b200 as F
    cap = 640
    s = Setup([cap, cap], 2, 64, F16, PAGE)
    q = torch.randn((2, 8, M, 64), generator=torch.Generator().manual_seed(1)).half().cuda()
    lengths = torch.tensor([cap + beyond, cap], dtype=torch.int32, device="cuda")
    out, L = F.attention_with_kv_cache(q, s.cache, s.table, lengths, window, sinks, return_log_normalizer=True)
    assert F.device_status() == 2
    kept = max(0, M - beyond)
    assert bool(out[0, :, kept:].isnan().all()) and bool(L[0, :, kept:].isnan().all())
    alone = torch.tensor([cap], dtype=torch.int32, device="cuda")
    parts = [(0, kept), (1, M)]
    for b, n in parts:
        if n == 0:
            continue
        w, Lw = F.attention_with_kv_cache(q[b:b + 1, :, :n], s.cache, s.table[b:b + 1], alone, window, sinks, return_log_normalizer=True)
        # The scores are the same, shares may be cut elsewhere.  On either side, of max |v|: 2^-11 by the weights and as much by the
        # output, 2^-10.9 / 7 by the products' alignment and 640 15 2^-24 / 7 by subnormal weights (_reference): 1.24 2^-10.
        # Of L: 40 sums of 2^-24 and 2^-21 of each weight.
        tol = 2.5 * 2.0 ** -10 * s.v[b].abs().amax().double()
        assert bool(((out[b:b + 1, :, :n].double() - w.double()).abs() <= tol).all())
        assert bool(((L[b:b + 1, :, :n] - Lw).abs() <= 2.0 ** -16 * (1 + Lw.abs())).all())
    assert F.device_status() == 0
