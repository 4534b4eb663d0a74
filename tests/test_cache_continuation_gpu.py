"""The cache as a decoding loop uses it, against the definition in 64 bits, with bounds that a wrong answer does not keep."""
import pytest
import torch

from test_kv_cache_gpu import BF16, F16, Setup, _reference, _values

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("dtype", [F16, BF16])
@pytest.mark.parametrize("window,sinks", [(128, 4), (None, 0), (40, 0)])
def test_continuation_row_by_row_and_at_once(dtype, window, sinks):
    """Rows appended and attended to one by one, and all of them in one call."""
    import flash_attn_with_score_b200 as F
    B, Hq, Hk, S, T, D = 2, 8, 2, 500, 6, 64
    s = Setup([S, S], Hk, D, dtype, 64)
    g = torch.Generator().manual_seed(2)
    make = lambda h: torch.randn((B, h, T, D), generator=g).to(dtype).cuda()  # noqa: E731
    q, k, v = make(Hq), make(Hk), make(Hk)
    free = sorted(set(range(s.cache.pages)) - set(s.table.flatten().tolist()))[:B]
    s.table = torch.cat([s.table, torch.tensor(free, dtype=torch.int32, device="cuda")[:, None]], 1)
    s.k, s.v = torch.cat([s.k, k], 2), torch.cat([s.v, v], 2)

    def near(got, q, n):
        s.lens = [n] * B
        ref, _, tol, _ = _reference(s, q, window, sinks, D ** -0.5)
        assert float(tol.max()) < 0.05 * float(ref.abs().max()) and float(tol.mean()) < 0.05 * float(ref.abs().mean())
        err = (got.double() - ref).abs()
        assert bool((err <= tol).all()), f"{float((err / tol).max()):.3g} of what rounding explains"

    for t in range(T):
        s.lengths += 1
        F.kv_cache_write(s.cache, k[:, :, t:t + 1], v[:, :, t:t + 1], s.table, s.lengths)
        near(F.attention_with_kv_cache(q[:, :, t:t + 1], s.cache, s.table, s.lengths, window, sinks), q[:, :, t:t + 1], S + t + 1)
    near(F.attention_with_kv_cache(q, s.cache, s.table, s.lengths, window, sinks), q, S + T)
    assert F.device_status() == 0


@pytest.mark.parametrize("dtype,D", [(F16, 128), (BF16, 16)])
@pytest.mark.parametrize("page", [-1, 2 ** 31 - 1, -0x7fffffff])
def test_rows_beside_a_missing_page(dtype, D, page):
    """The other rows of the call are written all the same, and nothing else is."""
    import flash_attn_with_score_b200 as F
    n, Hk, M = 100, 2, 70
    s = Setup([n, n], Hk, D, dtype, 16)
    before = [t.clone() for t in (s.cache.k_codes, s.cache.v_codes, s.cache.k_scales, s.cache.v_scales)]
    bad = s.table.clone()
    bad[1, 3] = page  # positions 48 .. 63
    g = torch.Generator().manual_seed(4)
    new = [torch.randn((2, Hk, M, D), generator=g).to(dtype).cuda() for _ in range(2)]
    F.kv_cache_write(s.cache, *new, bad, s.lengths)
    assert F.device_status() == 2
    want = [t.clone() for t in (s.k, s.v)]
    for w, x in zip(want, new):
        w[0, :, n - M:] = x[0]
        w[1, :, n - M:48], w[1, :, 64:] = x[1, :, :48 - (n - M)], x[1, :, 64 - (n - M):]
    for got, w in zip(F.kv_cache_read(s.cache, s.table, s.lengths, n), want):
        assert torch.equal(got, _values(w).to(dtype))
    same = torch.ones((s.cache.pages, 16), dtype=torch.bool, device="cuda")
    for b in range(2):
        for pos in range(n - M, n):
            if b == 0 or not 48 <= pos < 64:
                same[s.table[b, pos // 16].long(), pos % 16] = False
    for was, now in zip(before, (s.cache.k_codes, s.cache.v_codes, s.cache.k_scales, s.cache.v_scales)):
        assert torch.equal(was.transpose(1, 2)[same], now.transpose(1, 2)[same])
    assert F.device_status() == 0
