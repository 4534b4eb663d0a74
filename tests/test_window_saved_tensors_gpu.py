"""attention_with_window's backward pass on what saved-tensor hooks make of the tensors that it kept."""
import pytest
import torch

import flash_attn_with_score_b200 as F

pytestmark = pytest.mark.gpu


def _inputs(D, dtype):
    g = torch.Generator().manual_seed(1)
    make = lambda h: torch.randn((2, h, 150, D), generator=g).to(dtype).cuda()  # noqa: E731
    return [make(4).requires_grad_(), make(2).requires_grad_(), make(2).requires_grad_()], make(4)


@pytest.mark.parametrize("kv_splits", [None, 1])  # the native call, and the long way
@pytest.mark.parametrize("D,dtype", [(64, torch.float16), (128, torch.bfloat16), (16, torch.float16)])
def test_other_strides(kv_splits, D, dtype):
    xs, g = _inputs(D, dtype)
    call = lambda: F.attention_with_window(*xs, 40, 2, kv_splits=kv_splits)  # noqa: E731
    want = torch.autograd.grad(call(), xs, g)
    turn = lambda t: t.transpose(-1, -2).contiguous()  # noqa: E731
    wide = lambda t: torch.stack([t, t], -1)  # noqa: E731
    for pack, unpack in ((turn, lambda t: t.transpose(-1, -2)), (wide, lambda t: t[..., 1])):
        with torch.autograd.graph.saved_tensors_hooks(pack, unpack):
            out = call()
        for a, b in zip(torch.autograd.grad(out, xs, g), want):
            assert a.shape == b.shape and torch.equal(a, b)
    assert F.device_status() == 0


@pytest.mark.parametrize("kv_splits", [None, 1])
@pytest.mark.parametrize("unpack", [lambda t: t.double(), lambda t: t.cpu(), lambda t: t[..., :8], lambda t: t[:1]])
def test_other_tensors_are_refused(kv_splits, unpack):
    xs, g = _inputs(64, torch.float16)
    with torch.autograd.graph.saved_tensors_hooks(lambda t: t, unpack):
        out = F.attention_with_window(*xs, 40, 2, kv_splits=kv_splits)
    with pytest.raises((RuntimeError, TypeError, AssertionError)):
        torch.autograd.grad(out, xs, g)
    # one of them alone
    for at in range(5):
        count = iter(range(100))
        with torch.autograd.graph.saved_tensors_hooks(lambda t: (next(count), t), lambda p: unpack(p[1]) if p[0] == at else p[1]):
            out = F.attention_with_window(*xs, 40, 2, kv_splits=kv_splits)
        with pytest.raises((RuntimeError, TypeError, AssertionError)):
            torch.autograd.grad(out, xs, g)
    assert F.device_status() == 0
