"""attention_with_window and the cache's operators: the native call from Python against the long way, which a torch function mode
forces, and what is not for the native call."""
import sys

import pytest
import torch
from torch.overrides import TorchFunctionMode

import flash_attn_with_score_b200 as F
from flash_attn_with_score_b200 import _lib

pytestmark = pytest.mark.gpu


class _LongWay(TorchFunctionMode):
    def __torch_function__(self, func, types, args=(), kwargs=None):
        return func(*args, **(kwargs or {}))


@pytest.fixture
def natives(monkeypatch):
    """What each native call of the test returned."""
    seen, plain = [], _lib.plain
    monkeypatch.setattr(_lib, "plain", lambda *a: seen.append(plain(*a)) or seen[-1])
    return seen


def _inputs(M, N, D, dtype, heads_last=False, B=2, H=4, Hk=2):
    g = torch.Generator().manual_seed(M + N)
    make = lambda h, s: (torch.randn((B, s, h, D), generator=g).transpose(1, 2) if heads_last else torch.randn((B, h, s, D), generator=g)).to(dtype).cuda()  # noqa: E731
    return make(H, M), make(Hk, N), make(Hk, N), make(H, M)


def _same(a, b):
    assert a.dtype == b.dtype and a.shape == b.shape and a.stride() == b.stride() and a.requires_grad == b.requires_grad
    assert torch.equal(a, b)


@pytest.mark.parametrize("M,N,D,dtype,heads_last", [
    (300, 300, 64, torch.float16, False), (129, 700, 128, torch.bfloat16, True), (1, 3000, 128, torch.bfloat16, False),
    (50, 77, 16, torch.float16, False)])
@pytest.mark.parametrize("want_L", [False, True])
def test_window(natives, M, N, D, dtype, heads_last, want_L):
    q, k, v, g = _inputs(M, N, D, dtype, heads_last)
    call = lambda: F.attention_with_window(q, k, v, 60, 3, 0.2, return_log_normalizer=want_L)  # noqa: E731
    short = call()
    with _LongWay():
        long = call()
    assert natives[0] is not None and natives[1] is None
    for a, b in zip(*(x if want_L else (x,) for x in (short, long))):
        _same(a, b)
    for t in (q, k, v):
        t.requires_grad_()
    short = call()
    with _LongWay():
        long = call()
    assert natives[2] is not None and natives[3] is None
    short, long = ((x if want_L else (x,)) for x in (short, long))
    for a, b in zip(short, long):
        _same(a, b)
    for a, b in zip(torch.autograd.grad(short[0], (q, k, v), g), torch.autograd.grad(long[0], (q, k, v), g)):
        _same(a, b)


def test_gradients_that_are_out_of_the_ordinary(natives):
    q, k, v, g = _inputs(200, 200, 64, torch.float16)
    xs = [t.requires_grad_() for t in (q, k, v)]
    out = F.attention_with_window(q, k, v, 50, 2)
    assert natives[-1] is not None
    want = torch.autograd.grad(out, xs, g, retain_graph=True)
    for other in (g.transpose(2, 3).contiguous().transpose(2, 3), torch.zeros(2, 4, 200, 65, dtype=g.dtype, device="cuda")[..., 1:].copy_(g)):
        for a, b in zip(torch.autograd.grad(out, xs, other, retain_graph=True), want):
            assert float((a.double() - b.double()).abs().max()) <= 2.0 ** -8 * float(b.abs().max())  # another kernel family maybe
    expanded = torch.autograd.grad(out.sum(), xs, retain_graph=True)
    ones = torch.autograd.grad(out, xs, torch.ones_like(out))
    for a, b in zip(expanded, ones):
        assert float((a.double() - b.double()).abs().max()) <= 2.0 ** -8 * float(b.abs().max())
    # only some of the inputs want a gradient; L has none
    out, L = F.attention_with_window(q, k.detach(), v.detach(), 50, 2, return_log_normalizer=True)
    assert not L.requires_grad and out.requires_grad
    assert torch.equal(torch.autograd.grad(out, q, g)[0], want[0])
    # saved tensors that are packed away come back elsewhere
    with torch.autograd.graph.save_on_cpu():
        out = F.attention_with_window(q, k, v, 50, 2)
    for a, b in zip(torch.autograd.grad(out, xs, g), want):
        assert torch.equal(a, b)
    with torch.no_grad():
        assert not F.attention_with_window(q, k, v, 50, 2).requires_grad
    with torch.inference_mode():
        assert torch.equal(F.attention_with_window(q, k, v, 50, 2), F.attention_with_window(q.detach(), k, v, 50, 2))


def test_in_place_changes_of_what_was_saved_are_noticed():
    q, k, v, g = _inputs(64, 64, 64, torch.float16)
    q.requires_grad_()
    out = F.attention_with_window(q, k, v, 50, 2)
    k.add_(1)
    with pytest.raises(RuntimeError, match="modified by an inplace operation"):
        torch.autograd.grad(out, q, g)


@pytest.mark.parametrize("dtype,D", [(torch.float16, 128), (torch.bfloat16, 16)])
def test_cache(natives, dtype, D):
    q, k, v, _ = _inputs(3, 90, D, dtype)
    table = torch.randperm(14, generator=torch.Generator().manual_seed(1))[:12].view(2, 6).int().cuda()
    lengths = torch.tensor([90, 33], dtype=torch.int32, device="cuda")
    got = []
    for mode in (False, True):
        cache = F.KVCache4(14, 16, 2, D, dtype=dtype)
        with _LongWay() if mode else torch.no_grad():
            F.kv_cache_write(cache, k, v, table, lengths)
            got.append((cache.k_codes, cache.v_codes, cache.k_scales, cache.v_scales, *F.kv_cache_read(cache, table, lengths, 95),
                        *F.attention_with_kv_cache(q, cache, table, lengths, 40, 2, return_log_normalizer=True),
                        F.attention_with_kv_cache(q, cache, table, lengths, sm_scale=0.1)))
    assert all(x is not None for x in natives[:4]) and all(x is None for x in natives[4:]) and len(natives) == 8
    for a, b in zip(*got):
        _same(a, b)


def test_what_is_not_plain(natives):
    q, k, v, _ = _inputs(3, 90, 64, torch.float16)
    table = torch.arange(12, dtype=torch.int32, device="cuda").view(2, 6)
    lengths = torch.tensor([90, 33], dtype=torch.int32, device="cuda")
    cache = F.KVCache4(12, 16, 2, 64)
    F.kv_cache_write(cache, k, v, table, lengths)
    assert natives[-1] is True
    want = F.attention_with_kv_cache(q, cache, table, lengths)
    wide = torch.zeros((2, 12), dtype=torch.int32, device="cuda")
    wide[:, ::2] = table
    assert torch.equal(F.attention_with_kv_cache(q, cache, wide[:, ::2], lengths), want) and natives[-1] is None
    twice = torch.stack([lengths, lengths], 1)[:, 0]
    assert torch.equal(F.attention_with_kv_cache(q, cache, table, twice), want) and natives[-1] is None
    assert torch.equal(F.attention_with_kv_cache(q, cache, table, lengths, sm_scale="0.125"), want) and natives[-1] is None

    class Mine(F.KVCache4):
        pass
    mine = Mine(12, 16, 2, 64)
    before = len(natives)
    F.kv_cache_write(mine, k, v, table, lengths)
    assert torch.equal(F.attention_with_kv_cache(q, mine, table, lengths), want) and len(natives) == before


def test_without_the_module(monkeypatch):
    q, k, v, g = _inputs(100, 100, 64, torch.float16)
    want = F.attention_with_window(q, k, v, 30, 1)
    monkeypatch.setattr(_lib, "_plain", None)
    monkeypatch.delattr(F, "_plain", raising=False)
    monkeypatch.setitem(sys.modules, "flash_attn_with_score_b200._plain", None)
    assert torch.equal(F.attention_with_window(q, k, v, 30, 1), want) and _lib._plain is False
