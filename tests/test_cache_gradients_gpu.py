"""Derivatives that the operators do not have are refused, not dropped."""
import pytest
import torch
import torch.autograd.forward_ad as forward_ad
from torch.overrides import TorchFunctionMode

import flash_attn_with_score_b200 as F

pytestmark = pytest.mark.gpu


class _LongWay(TorchFunctionMode):
    def __torch_function__(self, func, types, args=(), kwargs=None):
        return func(*args, **(kwargs or {}))


def _cache():
    cache = F.KVCache4(4, 16, 2, 64)
    return cache, torch.arange(4, dtype=torch.int32, device="cuda").view(1, 4), torch.full((1,), 40, dtype=torch.int32, device="cuda")


@pytest.mark.parametrize("which", ["k", "v"])
@pytest.mark.parametrize("long", [False, True])
def test_written_rows_that_want_gradients(which, long):
    cache, table, lengths = _cache()
    x = torch.randn((1, 2, 5, 64), device="cuda").half()
    leaf = x.clone().requires_grad_()
    k, v = (leaf * 2, x) if which == "k" else (x, leaf * 2)
    before = cache.k_codes.clone()

    def refused():
        with pytest.raises(RuntimeError, match="backward"):
            F.kv_cache_write(cache, k, v, table, lengths)

    if long:
        with _LongWay():
            refused()
    else:
        refused()
    assert torch.equal(cache.k_codes, before)
    with torch.no_grad():
        F.kv_cache_write(cache, k, v, table, lengths)
    assert not torch.equal(cache.k_codes, before)
    written = cache.k_codes.clone()
    F.kv_cache_write(cache, k.detach(), v.detach(), table, lengths)
    assert torch.equal(cache.k_codes, written) and not cache.k_codes.requires_grad


@pytest.mark.parametrize("long", [False, True])
@pytest.mark.parametrize("at", [0, 1, 2])
def test_forward_mode_of_windows(at, long):
    xs = [torch.randn((1, 2, 70, 64), device="cuda").half() for _ in range(3)]
    tangent = torch.randn_like(xs[at])
    want = F.attention_with_window(*xs, 20, 1)

    def refused():
        duals = list(xs)
        duals[at] = forward_ad.make_dual(xs[at], tangent)
        for leaf in (False, True):
            if leaf:
                duals[(at + 1) % 3] = duals[(at + 1) % 3].clone().requires_grad_()
            with pytest.raises(RuntimeError, match="forward-mode"):
                F.attention_with_window(*duals, 20, 1)
        assert torch.equal(F.attention_with_window(*xs, 20, 1), want)  # no tangent, nothing to lose

    with forward_ad.dual_level():
        if long:
            with _LongWay():
                refused()
        else:
            refused()
    assert torch.equal(F.attention_with_window(*xs, 20, 1), want)


@pytest.mark.parametrize("long", [False, True])
def test_forward_mode_of_the_cache(long):
    cache, table, lengths = _cache()
    x = torch.randn((1, 2, 5, 64), device="cuda").half()
    F.kv_cache_write(cache, x, x, table, lengths)
    before = cache.k_codes.clone()

    def refused():
        dual = forward_ad.make_dual(x * 2, x)
        for call in (lambda: F.kv_cache_write(cache, dual, x, table, lengths), lambda: F.kv_cache_write(cache, x, dual, table, lengths),
                     lambda: F.attention_with_kv_cache(dual, cache, table, lengths)):
            with pytest.raises(RuntimeError, match="forward-mode"):
                call()

    with forward_ad.dual_level():
        if long:
            with _LongWay():
                refused()
        else:
            refused()
    assert torch.equal(cache.k_codes, before)
