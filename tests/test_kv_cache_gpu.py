"""The 4-bit cache against its definition in 64 bits: what a write leaves, what a read returns, attention over it."""
import math

import pytest
import torch

pytestmark = pytest.mark.gpu
F16, BF16 = torch.float16, torch.bfloat16


def _values(x):
    """What the cache holds of x (float64)."""
    D = x.shape[-1]
    g = min(32, D)
    xg = x.double().unflatten(-1, (D // g, g))
    s = (xg.abs().amax(-1, keepdim=True) / 7).to(BF16).double()
    s = torch.where(s < 2.0 ** -126, 0.0, s)
    c = torch.sign(xg) * torch.floor(xg.abs() / s + 0.5)
    v = torch.where(s > 0, c * s, 0.0)
    v = torch.where(torch.isfinite(xg).all(-1, keepdim=True), v, float("nan"))
    return v.flatten(-2)


class Setup:
    """A cache with the rows of a batch written in pages of no order."""

    def __init__(self, lens, Hk, D, dtype, page, seed=0, spread=True):
        import flash_attn_with_score_b200 as F
        g = torch.Generator().manual_seed(seed)
        self.lens, B, N = lens, len(lens), max(max(lens), 1)
        P = (N + page - 1) // page
        self.k, self.v = (torch.randn((B, Hk, N, D), generator=g).to(dtype).cuda() for _ in range(2))
        if spread:  # rows and channels of unlike size
            self.k *= torch.exp(torch.randn((1, Hk, 1, D), generator=g)).to(dtype).cuda()
            self.v *= torch.exp(2 * torch.randn((B, Hk, N, 1), generator=g)).to(dtype).cuda()
        self.table = torch.randperm(B * P + 3, generator=g)[:B * P].view(B, P).int().cuda()
        self.lengths = torch.tensor(lens, dtype=torch.int32, device="cuda")
        self.cache = F.KVCache4(B * P + 3, page, Hk, D, dtype=dtype)
        for b, n in enumerate(lens):
            if n > 0:
                F.kv_cache_write(self.cache, self.k[b:b + 1, :, :n], self.v[b:b + 1, :, :n], self.table[b:b + 1], self.lengths[b:b + 1])


def _reference(s, q, window, sinks, scale):
    """Output, log-normaliser and the largest error that rounding may make, float64.

    Errors of an output: its own rounding; 2^-11 of each weight, which is fp16; 2 eS of each weight, eS being the score's error;
    the weights that fp16 flushes, 2^-24 of the largest weighted scale each, times codes up to 15; and the sums.
    The matrix instructions take codes as c + 8 in subnormal halves, n 2^-22, aligned like 2^-14, that is like 2^8 codes.  Of the
    17 numbers that one adds each may lose 2^-24 of the largest: 17 2^-24 2^8 < 2^-11.9 of the largest factor
    next to the codes.  Scores: two instructions a group, for which the factor is at most max |q| s.  Outputs: one per 16 tokens
    and another for the sum of 8 P s, so 2^-10.9 of the sum of the largest P s of each 16, at most of sum P s; and
    the running sums, up to 15 sum P s, lose 2^-23 of themselves at each of n / 16 instructions, twice.  Other fp32 steps of a
    score are 2^-22 of sum |q| |k|."""
    B, Hq, M, D = q.shape
    Hk = s.k.shape[1]
    out = torch.zeros((B, Hq, M, D), dtype=torch.float64, device="cuda")
    L = torch.full((B, Hq, M), -float("inf"), dtype=torch.float64, device="cuda")
    tol, tolL = torch.zeros_like(out), torch.zeros_like(L)
    for b, n in enumerate(s.lens):
        if n == 0:
            continue
        k, v = _values(s.k[b, :, :n]), _values(s.v[b, :, :n])
        k, v = (x.repeat_interleave(Hq // Hk, 0) for x in (k, v))
        sc = q[b].double() @ k.mT * scale
        p, j = torch.arange(n - M, n, device="cuda")[:, None], torch.arange(n, device="cuda")[None, :]
        see = j <= p
        if window:
            see = see & ((j > p - window) | (j < sinks))
        sc = torch.where(see, sc, -float("inf"))
        some = see.any(-1)
        L[b] = torch.logsumexp(sc, -1)
        w = torch.where(some[:, None], torch.exp(sc - torch.where(some, L[b], 0.0)[..., None]), 0.0)
        broken, v = v.isnan(), v.nan_to_num()  # values that a row sees make its output NaN, others do not
        out[b] = torch.where(see.double() @ broken.double() > 0, float("nan"), w @ v)
        ks = k.abs().unflatten(-1, (D // min(32, D), min(32, D))).amax(-1, keepdim=True) / 7  # scales
        qa = q[b].double().abs()
        eS = abs(scale) * (2.0 ** -22 * qa @ k.abs().mT + 2 * 2.0 ** -11.9 * qa.amax(-1, keepdim=True) * ks.amax(-1).sum(-1)[:, None, :])
        tol[b] = (w * (2.0 ** -11 + 2 * eS)) @ v.abs() * 1.01 + (2 * (w * eS).sum(-1, keepdim=True)) * out[b].nan_to_num().abs()
        ws = w * v.abs().amax(-1)[:, None, :] / 7
        tol[b] += 15 * 2.0 ** -24 * n * ws.amax(-1, keepdim=True)
        tol[b] += (2.0 ** -10.9 + 2 * 15 * 2.0 ** -23 * (n / 16 + 1)) * ws.sum(-1, keepdim=True)
        tolL[b] = torch.where(see, eS, 0.0).amax(-1) + 2.0 ** -20 * (1 + torch.where(some, L[b], 0.0).abs())
    tol += torch.finfo(q.dtype).eps / 2 * (out.nan_to_num().abs() + tol) + torch.finfo(q.dtype).smallest_normal * torch.finfo(q.dtype).eps
    return out, L, tol, tolL


def _check(s, Hq, M, window=None, sinks=0, scale=None, seed=1):
    import flash_attn_with_score_b200 as F
    B, Hk, _, D = s.k.shape
    q = torch.randn((B, Hq, M, D), generator=torch.Generator().manual_seed(seed)).to(s.k.dtype).cuda()
    out, L = F.attention_with_kv_cache(q, s.cache, s.table, s.lengths, window, sinks, scale, return_log_normalizer=True)
    ref, Lr, tol, tolL = _reference(s, q, window, sinks, D ** -0.5 if scale is None else scale)
    assert out.dtype == q.dtype and out.shape == q.shape
    assert torch.equal(out.isnan(), ref.isnan())
    err = torch.where(ref.isnan(), 0.0, (out.double() - ref).abs())
    assert bool((err <= torch.where(ref.isnan(), 0.0, tol)).all()), f"worst {float((err / tol).nan_to_num().max()):.3g} of what rounding explains"
    none = Lr == -float("inf")
    assert bool((L[none] == -float("inf")).all()) and bool((out[none] == 0).all())
    assert bool(((L.double() - Lr).abs()[~none] <= tolL[~none]).all())
    assert F.device_status() == 0
    return out


@pytest.mark.parametrize("dtype", [F16, BF16])
@pytest.mark.parametrize("D", [16, 32, 64, 128])
@pytest.mark.parametrize("page", [16, 64, 256])
def test_read_returns_the_values(dtype, D, page):
    import flash_attn_with_score_b200 as F
    s = Setup([1, 16, 17, 300], 3, D, dtype, page)
    rows = 310  # more than any sequence has
    k, v = F.kv_cache_read(s.cache, s.table, s.lengths, rows)
    for got, x in ((k, s.k), (v, s.v)):
        assert got.shape == (4, 3, rows, D) and got.dtype == dtype
        for b, n in enumerate(s.lens):
            assert bool((got[b, :, :rows - n] == 0).all())
            assert torch.equal(got[b, :, rows - n:], _values(x[b, :, :n]).to(dtype))
    assert F.device_status() == 0


@pytest.mark.parametrize("dtype", [F16, BF16])
def test_borders_of_the_codes(dtype):
    """Halves, the largest and smallest numbers, groups of zeros, infinities and NaN."""
    import flash_attn_with_score_b200 as F
    D, n = 128, 256
    g = torch.Generator().manual_seed(5)
    x = torch.randn((1, 2, n, D), generator=g)
    step = torch.exp2(torch.randint(-12, 8, (1, 2, n, D // 32, 1), generator=g).float())
    halves = torch.randint(-14, 15, (1, 2, n, D // 32, 32), generator=g).float() / 2  # multiples of half a step, 7 among them
    halves[..., 0] = 7.0
    x[:, :, :100] = (halves * step).flatten(-2)[:, :, :100]
    x = x.to(dtype)
    big, small = torch.finfo(dtype).max, torch.finfo(dtype).smallest_normal
    x[0, 0, 100] = big
    x[0, 0, 101, ::2], x[0, 0, 101, 1::2] = -big, small
    x[0, 0, 102] = 0
    x[0, 0, 103] = small
    x[0, 0, 104] = small * torch.finfo(dtype).eps  # the smallest number
    x[0, 0, 105, 5], x[0, 0, 106, 70], x[0, 0, 107, 127] = float("inf"), -float("inf"), float("nan")
    x = x.cuda()
    table = torch.arange(n // 64, dtype=torch.int32, device="cuda")[None]
    lengths = torch.tensor([n], dtype=torch.int32, device="cuda")
    cache = F.KVCache4(n // 64, 64, 2, D, dtype=dtype)
    F.kv_cache_write(cache, x, x.flip(2), table, lengths)
    k, v = F.kv_cache_read(cache, table, lengths, n)
    want = _values(x).to(dtype)
    torch.testing.assert_close(k, want, rtol=0, atol=0, equal_nan=True)
    torch.testing.assert_close(v, want.flip(2), rtol=0, atol=0, equal_nan=True)


SHAPES = [  # lens, Hq, Hk, M, page, window, sinks
    ([1], 1, 1, 1, 16, None, 0),
    ([785], 28, 4, 1, 64, None, 0),
    ([0, 1, 15, 16, 17, 127, 128, 129, 400], 4, 2, 1, 16, None, 0),
    ([0, 1, 3, 64, 200, 1000], 8, 8, 5, 32, None, 0),           # more rows than tokens
    ([2100, 37, 900], 32, 8, 4, 128, None, 0),                  # two blocks of rows
    ([500, 129], 28, 4, 4, 64, None, 0),                        # 28 rows
    ([1500, 3, 700, 257], 16, 4, 1, 16, 100, 4),
    ([1500, 3, 700, 257], 16, 4, 3, 64, 128, 130),              # sinks over a tile
    ([600, 130], 8, 2, 2, 256, 1, 0),                           # one key a row
    ([600, 130], 8, 2, 2, 32, 1, 1),
    ([600, 350], 4, 4, 64, 16, 5000, 9),                        # a window longer than the sequences
    ([(7 * i) % 300 + (i % 3 == 0) * 500 for i in range(70)], 8, 2, 1, 16, None, 0),  # more sequences than lanes
    ([20000, 5], 8, 2, 1, 64, None, 0),                         # many shares to an item
    ([20000, 5], 8, 1, 2, 64, 9000, 64),
]


@pytest.mark.parametrize("shape", SHAPES, ids=lambda s: f"B{len(s[0])}n{max(s[0])}h{s[1]}-{s[2]}m{s[3]}p{s[4]}w{s[5]}s{s[6]}")
@pytest.mark.parametrize("dtype,D", [(F16, 128), (BF16, 128), (F16, 64), (BF16, 32), (F16, 16)])
def test_attention(shape, dtype, D):
    lens, Hq, Hk, M, page, window, sinks = shape
    _check(Setup(lens, Hk, D, dtype, page), Hq, M, window, sinks)


@pytest.mark.parametrize("scale", [0.0, -0.05, 3.0])
def test_scales(scale):
    _check(Setup([300, 70], 2, 64, BF16, 16, spread=False), 4, 2, None, 0, scale)


@pytest.mark.parametrize("size", [1e-30, 1e-6, 1e4, 1e30])
def test_values_of_any_size(size):
    """bf16 values beyond what fp16 holds, next to others of ordinary size."""
    import flash_attn_with_score_b200 as F
    s = Setup([400], 2, 64, BF16, 16)
    s.v[:, :, 100:] *= size
    F.kv_cache_write(s.cache, s.k, s.v, s.table, s.lengths)
    _check(s, 4, 1)


@pytest.mark.parametrize("size", [1e-25, 1e-5, 1e5, 1e30])
def test_values_all_of_one_size(size):
    import flash_attn_with_score_b200 as F
    s = Setup([400], 2, 64, BF16, 16)
    s.v *= size
    F.kv_cache_write(s.cache, s.k, s.v, s.table, s.lengths)
    _check(s, 4, 1)


@pytest.mark.parametrize("Hq,Hk,M,D", [(4, 4, 1, 64), (6, 2, 300, 16), (3, 1, 1001, 128), (32, 8, 700, 32)])
def test_empty_sequences_of_any_number_of_rows(Hq, Hk, M, D):
    """Zeros and -inf in every row of them, whatever lay in the memory of the outputs."""
    import flash_attn_with_score_b200 as F
    s = Setup([0, 30, 0, 1, 0], Hk, D, F16, 16)
    poison = [torch.full((5, Hq, M, *d), float("nan"), dtype=t, device="cuda") for d, t in (((D,), F16), ((), torch.float32))]
    del poison
    q = torch.randn((5, Hq, M, D), generator=torch.Generator().manual_seed(1)).half().cuda()
    for _ in range(4):
        out, L = F.attention_with_kv_cache(q, s.cache, s.table, s.lengths, return_log_normalizer=True)
        assert bool((out[::2] == 0).all()) and bool((L[::2] == -float("inf")).all())
        out.fill_(float("nan")), L.fill_(float("nan"))
    _check(s, Hq, M)


def test_unwritten_rows_of_a_page_do_not_matter():
    import flash_attn_with_score_b200 as F
    s = Setup([130, 40], 2, 128, F16, 64)
    want = _check(s, 8, 3, 60, 2)
    used = [(int(s.table[b, n // 64]), n % 64) for b, m in enumerate(s.lens) for n in range(m)]
    free = torch.ones((s.cache.pages, 64), dtype=torch.bool)
    for at in used:
        free[at] = False
    free = free.cuda()
    for codes, scales in ((s.cache.k_codes, s.cache.k_scales), (s.cache.v_codes, s.cache.v_scales)):
        codes.transpose(1, 2)[free] = 0x5A
        for fill in (float("nan"), float("inf"), -float("inf")):
            scales.transpose(1, 2)[free] = fill
            assert torch.equal(_check(s, 8, 3, 60, 2), want)


def test_non_finite_values_reach_only_who_sees_them():
    import flash_attn_with_score_b200 as F
    s = Setup([300], 2, 64, F16, 16, spread=False)
    s.v[0, 0, 50, 3] = float("inf")   # group 0 of head 0
    s.k[0, 1, 200, 40] = float("nan")  # head 1
    F.kv_cache_write(s.cache, s.k, s.v, s.table, s.lengths)
    q = torch.randn((1, 4, 20, 64), device="cuda").half()
    out = F.attention_with_kv_cache(q, s.cache, s.table, s.lengths, 85, 0)
    # rows 0..19 stand at 280..299 and see from 196 + row on: all but rows 0..4 are past key 200
    assert bool(out[0, 2:, :5].isnan().all()) and not bool(out[0, 2:, 5:].isnan().any())
    assert not bool(out[0, :2].isnan().any())
    out = F.attention_with_kv_cache(q, s.cache, s.table, s.lengths, 1, 51)
    assert bool(out[0, :2, :, :32].isnan().all()) and not bool(out[0, :2, :, 32:].isnan().any())


def test_strided_inputs():
    import flash_attn_with_score_b200 as F
    s = Setup([200, 90], 2, 64, BF16, 16, spread=False)
    want = _check(s, 4, 1)
    q = torch.randn((2, 4, 1, 64), generator=torch.Generator().manual_seed(1)).to(BF16).cuda()
    odd = torch.zeros((2, 1, 4, 67), dtype=BF16, device="cuda")[..., 1:65].transpose(1, 2)  # (B, H, M, D), rows off 16 bytes
    odd.copy_(q)
    table = torch.full((2, s.table.shape[1] + 5), -7, dtype=torch.int32, device="cuda")
    table[:, :s.table.shape[1]] = s.table
    view = table[:, :s.table.shape[1]]
    assert torch.equal(F.attention_with_kv_cache(odd, s.cache, view, s.lengths), want)
    other = F.KVCache4(s.cache.pages, 16, 2, 64, dtype=BF16)
    kv = torch.zeros((2, 200, 2, 2, 65), dtype=BF16, device="cuda")[..., 1:]
    k, v = kv[:, :, 0].transpose(1, 2), kv[:, :, 1].transpose(1, 2)
    for b, n in enumerate(s.lens):  # sequence 1 with padding before it
        k[b, :, 200 - n:], v[b, :, 200 - n:] = s.k[b, :, :n], s.v[b, :, :n]
    F.kv_cache_write(other, k, v, view, s.lengths)
    for a, b in zip(F.kv_cache_read(other, view, s.lengths, 200), F.kv_cache_read(s.cache, view, s.lengths, 200)):
        assert torch.equal(a, b)


def test_written_rows_only():
    """Rows of other positions, pages and heads stay as they were."""
    import flash_attn_with_score_b200 as F
    s = Setup([70, 33], 2, 128, F16, 16)
    before = [t.clone() for t in (s.cache.k_codes, s.cache.v_codes, s.cache.k_scales, s.cache.v_scales)]
    new = torch.randn((2, 2, 3, 128), device="cuda").half()
    F.kv_cache_write(s.cache, new, new, s.table, s.lengths)
    mask = torch.ones((s.cache.pages, 16), dtype=torch.bool, device="cuda")
    for b, n in enumerate(s.lens):
        for pos in range(n - 3, n):
            mask[s.table[b, pos // 16].long(), pos % 16] = False
    for was, now in zip(before, (s.cache.k_codes, s.cache.v_codes, s.cache.k_scales, s.cache.v_scales)):
        assert torch.equal(was.transpose(1, 2)[mask], now.transpose(1, 2)[mask])


def test_cache_beyond_32_bits():
    """Rows behind the first 4 GB of the codes."""
    import flash_attn_with_score_b200 as F
    pages = 36000  # x 16 heads x 128 tokens x 64 bytes: 4.7 GB of codes for the keys
    cache = F.KVCache4(pages, 128, 16, 128, dtype=F16)
    table = torch.tensor([[pages - 1, 3]], dtype=torch.int32, device="cuda")
    lengths = torch.tensor([200], dtype=torch.int32, device="cuda")
    x = torch.randn((1, 16, 200, 128), device="cuda").half()
    F.kv_cache_write(cache, x, x, table, lengths)
    assert torch.equal(F.kv_cache_read(cache, table, lengths, 200)[0], _values(x).half())
    q = torch.randn((1, 16, 1, 128), device="cuda").half()
    out = F.attention_with_kv_cache(q, cache, table, lengths)
    v = _values(x)
    want = torch.softmax(q.double() @ v.mT * 128 ** -0.5, -1) @ v
    assert float((out.double() - want).abs().max()) < 2e-3  # |out| < 1, weights and output rounded to 2^-11


def test_what_the_cache_does_not_have():
    """Pages and lengths out of range: nothing is touched, the status says so."""
    import flash_attn_with_score_b200 as F
    s = Setup([100, 100], 2, 64, F16, 16)
    want = _check(s, 4, 1)
    q = torch.randn((2, 4, 1, 64), generator=torch.Generator().manual_seed(1)).half().cuda()
    bad = s.table.clone()
    for page in (s.cache.pages, -1, 2 ** 31 - 1, -2 ** 31):
        bad[1, 2] = page
        out = F.attention_with_kv_cache(q, s.cache, bad, s.lengths)
        assert torch.equal(out[0], want[0]) and bool(out[1].isnan().all())
        assert F.device_status() == 2 and F.device_status() == 0
        k, v = F.kv_cache_read(s.cache, bad, s.lengths, 100)
        assert bool(k[1, :, 32:48].isnan().all()) and not bool(k[1, :, :32].isnan().any()) and not bool(v[0].isnan().any())
        assert F.device_status() == 2
        before = s.cache.k_codes.clone()
        new = torch.randn((2, 2, 100, 64), device="cuda").half()
        keep = s.cache.k_codes[:, :, :].clone()
        F.kv_cache_write(s.cache, s.k, s.v, bad, s.lengths)
        assert torch.equal(before, s.cache.k_codes) and F.device_status() == 2
    # an unused entry may be anything
    wide = torch.cat([s.table, torch.full((2, 3), -1, dtype=torch.int32, device="cuda")], 1)
    assert torch.equal(F.attention_with_kv_cache(q, s.cache, wide, s.lengths), want) and F.device_status() == 0
    long = torch.tensor([10 ** 9, -5], dtype=torch.int32, device="cuda")
    out = F.attention_with_kv_cache(q, s.cache, s.table, long)
    assert bool((out[1] == 0).all()) and F.device_status() == 2


def test_graph_stream_and_two_at_once():
    import flash_attn_with_score_b200 as F
    s = Setup([900, 333, 12], 4, 128, BF16, 64)
    q = torch.randn((3, 16, 1, 128), device="cuda").to(BF16)
    new = torch.randn((3, 4, 1, 128), device="cuda").to(BF16)

    def step():
        F.kv_cache_write(s.cache, new, new, s.table, s.lengths)
        return F.attention_with_kv_cache(q, s.cache, s.table, s.lengths)

    want = step().clone()
    again = step()
    assert torch.equal(want, again)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        other = step()
    torch.cuda.synchronize()
    assert torch.equal(want, other)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        captured = step()
    # replayed with other rows, lengths and pages in place
    new.normal_()
    q.normal_()
    s.lengths.copy_(torch.tensor([700, 332, 13], dtype=torch.int32))
    graph.replay()
    torch.cuda.synchronize()
    assert torch.equal(captured, step())
    # two calls at once
    F.kv_cache_write(s.cache, new, new, s.table, s.lengths)
    side.wait_stream(torch.cuda.current_stream())
    outs = []
    for x in range(6):
        with torch.cuda.stream(side if x & 1 else torch.cuda.current_stream()):
            outs.append(F.attention_with_kv_cache(q, s.cache, s.table, s.lengths))
    torch.cuda.synchronize()
    assert all(torch.equal(o, outs[0]) for o in outs)
    assert F.device_status() == 0


def test_a_cache_stays_what_it_is():
    import copy
    s = Setup([64], 2, 64, F16, 16)
    for name in ("k_codes", "v_codes", "k_scales", "v_scales", "pages", "page_size", "heads", "head_dim", "dtype"):
        with pytest.raises(AttributeError, match=name):
            setattr(s.cache, name, getattr(s.cache, name))
    with pytest.raises(ValueError):  # two caches that say to be apart and share their memory
        copy.deepcopy(s.cache)
    _check(s, 4, 1)


def test_refusals():
    import flash_attn_with_score_b200 as F
    s = Setup([64], 2, 64, F16, 16)
    q = torch.zeros((1, 4, 1, 64), dtype=F16, device="cuda")
    call = lambda q=q, table=s.table, lens=s.lengths, **kw: F.attention_with_kv_cache(q, s.cache, table, lens, **kw)
    with pytest.raises(TypeError):
        call(q.bfloat16())
    with pytest.raises(TypeError):
        call(table=s.table.long())
    with pytest.raises(AssertionError):
        call(q[..., :32])
    with pytest.raises(AssertionError):
        call(q[:, :3])
    with pytest.raises(AssertionError):
        call(window=0)
    with pytest.raises(AssertionError):
        call(sinks=-1)
    with pytest.raises(AssertionError):
        call(lens=s.lengths.cpu())
    with pytest.raises(AssertionError):
        call(table=s.table[:, :0])
    with pytest.raises(RuntimeError, match="backward"):
        call(q.clone().requires_grad_())
    with pytest.raises(AssertionError):
        F.kv_cache_write(s.cache, s.k[:, :1], s.v[:, :1], s.table, s.lengths)
    with pytest.raises(TypeError):
        F.kv_cache_write(s.cache, s.k.bfloat16(), s.v.bfloat16(), s.table, s.lengths)
    # nothing to do
    F.kv_cache_write(s.cache, s.k[:, :, :0], s.v[:, :, :0], s.table, s.lengths)
    assert call(q[:, :, :0]).shape == (1, 4, 0, 64)
    assert F.kv_cache_read(s.cache, s.table, s.lengths, 0)[0].shape == (1, 2, 0, 64)
