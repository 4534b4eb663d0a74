"""attention_with_window against its definition in 64 bits: forward, backward, both kernel families, few rows and many."""
import time

import pytest
import torch

pytestmark = pytest.mark.gpu
F16, BF16 = torch.float16, torch.bfloat16


@pytest.fixture(scope="module", autouse=True)
def _engine_at_rest():
    """The autograd engine's thread lets go of the last gradients a moment after a backward pass has returned (14 % of the passes
    of test_expanded_inputs, up to 0.5 ms); tests that count the memory in use may come next."""
    yield
    time.sleep(0.5)


def _inputs(B, Hq, Hk, M, N, D, dtype, seed=0):
    g = torch.Generator().manual_seed(seed)
    make = lambda h, n: torch.randn((B, h, n, D), generator=g).to(dtype).cuda()
    return make(Hq, M), make(Hk, N), make(Hk, N), make(Hq, M)


def _see(M, N, window, sinks):
    p, j = torch.arange(M, device="cuda")[:, None] + (N - M), torch.arange(N, device="cuda")[None, :]
    return (j <= p) & ((j > p - window) | (j < sinks))


class Reference:
    """out, L, dq, dk, dv of one call in 64 bits, and what rounding may make of each.

    u = eps / 2 of the 16-bit type.  eS, the error of a score: 2^-20 sum |q||k| scale (fp32 sums of products).  A weight is off by
    2 eS P (score and normaliser), and by u P more where it is a 16-bit operand, with 2^-25 of 2^8 times it at most (the running
    maximum lags by up to 2^8) where fp16 makes it a subnormal: 2^-16 of the largest weight, 1.
    out: u |out| + (u + 2 eS) sum P |v| + 2^-24 sum |v| over visible keys (subnormal weights, relative to a maximum weight).
    delta: what out is off by, times |dout|, and 2^-20 sum |out dout|.
    dS: (u + 2 eS) |dS| + P (delta's error + 2^-20 sum |dout||v|), and half the smallest fp16 number.
    dq, dk, dv: those through the products, u of the result and (grouped heads: 16-bit partial sums) u of each head's part."""

    def __init__(self, q, k, v, window, sinks, scale=None, dout=None):
        B, Hq, M, D = q.shape
        Hk, N = k.shape[1], k.shape[2]
        G = Hq // Hk
        scale = D ** -0.5 if scale is None else scale
        u = torch.finfo(q.dtype).eps / 2
        sub = 2.0 ** -25 if q.dtype == F16 else 0.0
        see = _see(M, N, window, sinks)
        some = see.any(-1)
        d = lambda t: torch.zeros(t, dtype=torch.float64, device="cuda")
        self.out, self.L, self.tout, self.tL = d(q.shape), d((B, Hq, M)), d(q.shape), d((B, Hq, M))
        self.dq, self.tdq = d(q.shape), d(q.shape)
        self.dk, self.dv, self.tdk, self.tdv = d(k.shape), d(k.shape), d(k.shape), d(k.shape)
        for b in range(B):
            for h in range(Hq):
                qq, kk, vv = q[b, h].double(), k[b, h // G].double(), v[b, h // G].double()
                s = torch.where(see, qq @ kk.mT * scale, -float("inf"))
                L = torch.logsumexp(s, -1)
                p = torch.where(some[:, None], torch.exp(s - torch.where(some, L, 0.0)[:, None]), 0.0)
                eS = 2.0 ** -20 * (qq.abs() @ kk.abs().mT) * abs(scale)
                o = p @ vv
                to = (p * (u + 2 * eS)) @ vv.abs() + sub * 2 * (see.double() @ vv.abs())
                to = to + u * (o.abs() + to) + 2 * sub
                self.out[b, h], self.L[b, h], self.tout[b, h] = o, L, to
                self.tL[b, h] = torch.where(see, eS, 0.0).amax(-1) + 2.0 ** -20 * (1 + torch.where(some, L, 0.0).abs())
                if dout is None:
                    continue
                g = dout[b, h].double()
                delta = (o * g).sum(-1, keepdim=True)
                dp = g @ vv.mT
                ds = p * (dp - delta)
                ed = (to * g.abs()).sum(-1, keepdim=True) + 2.0 ** -20 * (o * g).abs().sum(-1, keepdim=True)
                eds = torch.where(see, (u + 2 * eS) * ds.abs() + p * (ed + 2.0 ** -20 * (g.abs() @ vv.abs().mT)) + sub, 0.0)
                dq, dk, dv = ds @ kk * scale, ds.mT @ qq * scale, p.mT @ g
                self.dq[b, h] = dq
                self.tdq[b, h] = (eds @ kk.abs()) * abs(scale) * (1 + u) + u * dq.abs() + 2 * sub
                self.dk[b, h // G] += dk
                self.dv[b, h // G] += dv
                self.tdk[b, h // G] += (eds.mT @ qq.abs()) * abs(scale) * (1 + u) + u * dk.abs() + 2 * sub
                ep = torch.where(see, p * (u + 2 * eS) + sub, 0.0)
                self.tdv[b, h // G] += (ep.mT @ g.abs()) * (1 + u) + u * dv.abs() + 2 * sub
        self.tdk += u * (self.dk.abs() + self.tdk)
        self.tdv += u * (self.dv.abs() + self.tdv)


def _near(name, got, want, tol):
    err = (got.double() - want).abs()
    assert bool((err <= tol).all()), f"{name}: {float((err / tol).nan_to_num().max()):.3g} of what rounding explains"


def _check(shape, dtype, backend=None, backward=True, kv_splits=None, scale=None):
    import flash_attn_with_score_b200 as F
    B, Hq, Hk, M, N, D, window, sinks = shape
    q, k, v, g = _inputs(B, Hq, Hk, M, N, D, dtype)
    ref = Reference(q, k, v, window, sinks, scale, g if backward else None)
    kw = dict(sinks=sinks, sm_scale=scale, backend=backend, kv_splits=kv_splits)
    out, L = F.attention_with_window(q, k, v, window, return_log_normalizer=True, **kw)
    _near("out", out, ref.out, ref.tout)
    none = ref.L == -float("inf")
    assert torch.equal(L == -float("inf"), none) and bool((out[none] == 0).all())
    assert bool(((L.double() - ref.L).abs()[~none] <= ref.tL[~none]).all())
    assert torch.equal(F.attention_with_window(q, k, v, window, **kw), out)
    if backward:
        for t in (q, k, v):
            t.requires_grad_()
        got = F.attention_with_window(q, k, v, window, **kw)
        assert torch.equal(got.detach(), out)
        dq, dk, dv = torch.autograd.grad(got, (q, k, v), g)
        assert dk.shape == k.shape and dv.shape == v.shape
        _near("dq", dq, ref.dq, ref.tdq)
        _near("dk", dk, ref.dk, ref.tdk)
        _near("dv", dv, ref.dv, ref.tdv)
    assert F.device_status() == 0
    return out


SHAPES = [  # B, Hq, Hk, M, N, window, sinks
    (1, 1, 1, 1, 1, 1, 0),
    (1, 2, 1, 3, 3, 1, 1),
    (1, 4, 4, 129, 129, 1, 0),             # only itself
    (2, 4, 2, 128, 128, 64, 4),
    (1, 4, 2, 300, 300, 64, 7),
    (2, 3, 3, 257, 700, 128, 0),           # continues a sequence
    (1, 2, 2, 1000, 1000, 128, 4),
    (1, 2, 1, 1000, 1000, 200, 130),       # sinks of two tiles
    (1, 4, 1, 640, 640, 100, 300),         # more sinks than window
    (1, 2, 2, 500, 200, 50, 3),            # rows before the first key
    (1, 2, 2, 700, 300, 1000, 0),
    (1, 2, 2, 2048, 2048, 512, 64),
    (1, 7, 1, 897, 897, 129, 1),
    (1, 2, 2, 385, 385, 10 ** 9, 10 ** 9),  # all of it
]


@pytest.mark.parametrize("shape", SHAPES, ids=lambda s: "b%dh%d-%dm%dn%dw%ds%d" % s)
@pytest.mark.parametrize("dtype,D", [(F16, 128), (BF16, 128), (F16, 64), (BF16, 64), (F16, 32), (BF16, 16)])
def test_window(shape, dtype, D):
    _check((*shape[:5], D, *shape[5:]), dtype)


@pytest.mark.parametrize("shape", SHAPES, ids=lambda s: "b%dh%d-%dm%dn%dw%ds%d" % s)
@pytest.mark.parametrize("dtype,D", [(F16, 64), (BF16, 32)])
def test_window_on_the_cuda_core_kernels(shape, dtype, D):
    _check((*shape[:5], D, *shape[5:]), dtype, backend="generic")


@pytest.mark.parametrize("shape", [
    (2, 32, 8, 1, 1500, 128, 400, 4), (1, 28, 4, 1, 3000, 128, 2900, 0), (3, 4, 4, 1, 777, 64, 100, 4), (1, 8, 2, 16, 3000, 64, 1500, 64),
    (2, 28, 4, 4, 2000, 128, 300, 130), (1, 16, 4, 32, 32, 64, 8, 2), (1, 8, 1, 17, 900, 128, 256, 1), (1, 2, 1, 64, 5000, 32, 4096, 7),
    (1, 4, 2, 5, 130, 64, 1000, 0), (4, 8, 8, 2, 129, 128, 1, 1), (1, 2, 2, 200, 4000, 128, 3000, 4)],
    ids=lambda s: "b%dh%d-%dm%dn%dd%dw%ds%d" % s)
@pytest.mark.parametrize("dtype", [F16, BF16])
def test_few_rows(shape, dtype):
    want = _check(shape, dtype, backward=False)
    nkt = (shape[4] + 127) // 128
    for splits in {1, 2, min(5, nkt), nkt}:
        if splits <= nkt:
            _check(shape, dtype, backward=False, kv_splits=splits)
    assert want.shape[2] == shape[3]


@pytest.mark.parametrize("shape", [(1, 40, 40, 1500, 1500, 64, 300, 7), (2, 37, 37, 600, 600, 128, 130, 0), (1, 75, 75, 513, 2000, 64, 700, 4),
                                   (3, 32, 8, 700, 700, 128, 256, 4), (1, 600, 600, 1000, 1000, 64, 100, 4)],
                         ids=lambda s: "b%dh%d-%dm%dn%dd%dw%ds%d" % s)
def test_many_row_blocks(shape):
    """Launches of more CTAs than SMs, which walk lists of row blocks, and of 256-row CTAs."""
    _check(shape, F16, backward=shape[1] < 100)


@pytest.mark.parametrize("shape", [
    (8, 4, 2, 1100, 1100, 64, 64, 4),      # a group's heads in one CTA, the tile with sinks in parts of heads and query ranges
    (4, 14, 2, 1700, 1700, 64, 60, 200),   # two tiles with sinks
    (1, 3, 3, 2500, 2500, 64, 90, 300),    # three, each in five ranges
    (2, 16, 4, 900, 900, 128, 100, 0),     # none
    (2, 6, 2, 300, 1200, 128, 50, 140),    # queries that begin behind the tiles with sinks
    (2, 6, 2, 700, 300, 64, 50, 140),      # and before the first key
    (1, 8, 2, 1100, 1100, 128, 64, 600),   # too many sinks for parts
    (3, 32, 8, 300, 300, 64, 256, 4)],
    ids=lambda s: "b%dh%d-%dm%dn%dd%dw%ds%d" % s)
@pytest.mark.parametrize("dtype", [F16, BF16])
def test_backward_of_groups_and_sinks(shape, dtype):
    _check(shape, dtype)


@pytest.mark.parametrize("scale", [0.3, 0.0, -0.1])
def test_scales(scale):
    """(0 and below: the CUDA-core kernels)"""
    _check((1, 2, 1, 200, 200, 64, 50, 3), BF16, scale=scale)


def test_equals_causal_attention_where_the_window_holds_everything():
    import flash_attn_with_score_b200 as F
    for shape in ((2, 8, 2, 600, 600, 128), (1, 4, 4, 100, 700, 64)):
        q, k, v, g = _inputs(*shape, BF16)
        ref = Reference(q, k, v, 10 ** 6, 0)
        _near("out", F.attention(q, k, v, causal=True), ref.out, ref.tout)
        _near("out", F.attention_with_window(q, k, v, shape[4]), ref.out, ref.tout)


def test_hidden_keys_do_not_matter():
    """Keys and values that no query of a call sees may hold anything finite; those outside the visited tiles anything at all."""
    import flash_attn_with_score_b200 as F
    q, k, v, g = _inputs(1, 4, 2, 100, 2000, 64, F16)
    want = F.attention_with_window(q, k, v, 300, 4)
    k[:, :, 128:1400], v[:, :, 128:1400] = float("nan"), float("inf")
    assert torch.equal(F.attention_with_window(q, k, v, 300, 4), want)
    k[:, :, 4:1601], v[:, :, 4:1601] = 60000.0, -60000.0
    assert torch.equal(F.attention_with_window(q, k, v, 300, 4), want)


def test_strided_views_and_gradients_of_views():
    import flash_attn_with_score_b200 as F
    B, H, S, D = 2, 4, 300, 64
    packed = torch.randn((B, S, 3, H, D), generator=torch.Generator().manual_seed(3)).half().cuda().requires_grad_()
    q, k, v = (packed[:, :, x].transpose(1, 2) for x in range(3))
    ref = Reference(q.detach(), k.detach(), v.detach(), 70, 5, None, torch.ones_like(q))
    out = F.attention_with_window(q, k, v, 70, 5)
    _near("out", out.detach(), ref.out, ref.tout)
    out.backward(torch.ones_like(out))  # an expanded gradient would do too
    for x, (want, tol) in enumerate(((ref.dq, ref.tdq), (ref.dk, ref.tdk), (ref.dv, ref.tdv))):
        _near("grad", packed.grad[:, :, x].transpose(1, 2), want, tol)
    odd = torch.zeros((1, 2, 130, 65), dtype=F16, device="cuda")[..., 1:]
    odd.copy_(torch.randn(odd.shape, generator=torch.Generator().manual_seed(4)))
    ref = Reference(odd, odd, odd, 33, 1)
    _near("out", F.attention_with_window(odd, odd, odd, 33, 1), ref.out, ref.tout)
    assert F.last_backend() == "generic"


def test_differences():
    """The gradient against differences of the kernel's own outputs, along the gradient; what rounding and the third derivative may
    add is bounded in 64 bits."""
    import flash_attn_with_score_b200 as F
    q, k, v, g = _inputs(1, 2, 1, 96, 96, 64, F16, seed=2)
    window, sinks = 20, 3
    q, k, v = q * 2, k, v
    xs = [t.clone().requires_grad_() for t in (q, k, v)]
    grads = torch.autograd.grad(F.attention_with_window(*xs, window, sinks), xs, g)
    ref = Reference(q, k, v, window, sinks, None, g)
    for n, (name, gk, g64, tol) in enumerate((("q", grads[0], ref.dq, ref.tdq), ("k", grads[1], ref.dk, ref.tdk), ("v", grads[2], ref.dv, ref.tdv))):
        step = (g64 * (0.25 / float(g64.abs().max()))).half()
        plus, minus = [q, k, v], [q, k, v]
        plus[n], minus[n] = plus[n] + step, minus[n] - step
        move = plus[n].double() - minus[n].double()  # as the 16-bit sums came out
        r1, r0 = Reference(*plus, window, sinks), Reference(*minus, window, sinks)
        diff = ((F.attention_with_window(*plus, window, sinks).double() - F.attention_with_window(*minus, window, sinks).double()) * g).sum()
        curve = (((r1.out - r0.out) * g).sum() - (g64 * move).sum()).abs()
        bound = ((r1.tout + r0.tout) * g.abs()).sum() + curve + (tol * move.abs()).sum()
        slope = (gk.double() * move).sum()
        assert float((diff - slope).abs()) <= float(bound), name
        assert float(bound) < 0.5 * float(slope.abs()), name  # the comparison says something


def test_graphs_streams_and_a_backward_pass_captured():
    import flash_attn_with_score_b200 as F
    q, k, v, g = _inputs(2, 8, 2, 400, 400, 64, BF16)
    xs = [t.requires_grad_() for t in (q, k, v)]

    def step():
        out = F.attention_with_window(*xs, 100, 4)
        # (detached: torch refuses to capture a backward pass while an eager graph of the same leaves lives)
        return (out.detach(), *torch.autograd.grad(out, xs, g))

    want = [t.clone() for t in step()]
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        for _ in range(3):
            other = step()
    torch.cuda.current_stream().wait_stream(side)
    torch.cuda.synchronize()
    assert all(torch.equal(a, b) for a, b in zip(want, other))
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        captured = step()
    with torch.no_grad():
        for t in xs:
            t.copy_(torch.randn_like(t))
    graph.replay()
    torch.cuda.synchronize()
    assert all(torch.equal(a, b) for a, b in zip(captured, step()))
    assert F.device_status() == 0


def test_together_window_prefill_then_cache():
    """A prompt is attended to with the window, goes into the 4-bit cache, and is continued token by token over it: the rows of
    the continuation are those of one windowed call on the values that the cache holds."""
    import flash_attn_with_score_b200 as F
    B, Hq, Hk, S, T, D, window, sinks = 2, 8, 2, 500, 6, 64, 128, 4
    q, k, v, _ = _inputs(B, Hq, Hk, S + T, S + T, D, BF16)
    cache = F.KVCache4(40, 64, Hk, D, dtype=BF16)
    table = torch.randperm(40, generator=torch.Generator().manual_seed(1))[:2 * 8].view(2, 8).int().cuda()
    lengths = torch.full((B,), S, dtype=torch.int32, device="cuda")
    first = F.attention_with_window(q[:, :, :S], k[:, :, :S], v[:, :, :S], window, sinks)
    ref = Reference(q[:, :, :S], k[:, :, :S], v[:, :, :S], window, sinks)
    _near("prompt", first, ref.out, ref.tout)
    F.kv_cache_write(cache, k[:, :, :S], v[:, :, :S], table, lengths)
    rows = []
    for t in range(S, S + T):
        lengths += 1
        F.kv_cache_write(cache, k[:, :, t:t + 1], v[:, :, t:t + 1], table, lengths)
        rows.append(F.attention_with_kv_cache(q[:, :, t:t + 1], cache, table, lengths, window, sinks))
    rows = torch.cat(rows, 2)
    again = F.attention_with_kv_cache(q[:, :, S:], cache, table, lengths, window, sinks)
    kc, vc = F.kv_cache_read(cache, table, lengths, S + T)
    # (bf16 values are within 2^-9 of what the cache holds)
    ref = Reference(q[:, :, S:], kc, vc, window, sinks)
    slack = 2.0 ** -8 * (1 + (q[:, :, S:].double().abs().amax() * kc.double().abs().amax()) * D ** 0.5) * vc.double().abs().amax()
    assert float((rows.double() - ref.out).abs().max()) <= float(slack) and float((again.double() - ref.out).abs().max()) <= float(slack)
    # the same rows, in one call or six: fp16 weights, outputs rounded once
    assert float((rows.double() - again.double()).abs().max()) <= 2 * (2.0 ** -8 + 2.0 ** -10) * float(vc.double().abs().amax())
    via_window = F.attention_with_window(q[:, :, S:], kc, vc, window, sinks)
    _near("window over the values read back", via_window, ref.out, ref.tout)
    assert F.device_status() == 0


@pytest.mark.parametrize("kv_splits", [None, 1])
def test_no_second_derivative(kv_splits):
    """Refused, where a gradient without a graph would drop terms silently."""
    import flash_attn_with_score_b200 as F
    q = torch.randn((1, 2, 40, 64), device="cuda").half().requires_grad_()
    out = F.attention_with_window(q, q, q, 10, kv_splits=kv_splits).float().sum()
    with pytest.raises(RuntimeError, match="second derivative"):
        torch.autograd.grad(out, q, create_graph=True, retain_graph=True)
    want, = torch.autograd.grad(out, q)
    y = torch.utils.checkpoint.checkpoint(lambda x: F.attention_with_window(x, x, x, 10, kv_splits=kv_splits), q, use_reentrant=False)
    assert torch.equal(torch.autograd.grad(y.float().sum(), q)[0], want)


@pytest.mark.parametrize("D", [64, 128])
def test_expanded_inputs(D):
    """Heads, sequences and rows that are one in memory, and their gradients: the sums over what shares them."""
    import flash_attn_with_score_b200 as F
    B, H, N = 2, 4, 300
    g = torch.Generator().manual_seed(5)
    make = lambda *s: torch.randn(s, generator=g).half().cuda()  # noqa: E731
    q, do = make(B, H, N, D), make(B, H, N, D)
    for shape in ((B, 1, N, D), (1, H, N, D), (1, 1, N, D), (B, H, 1, D)):
        k, v = make(*shape), make(*shape)
        grads = []
        for whole in (False, True):
            xs = [x.clone().requires_grad_() for x in (q, k, v)]
            wide = [x.expand(B, H, N, D) for x in xs]
            out = F.attention_with_window(*([x.contiguous() for x in wide] if whole else wide), 64, 3)
            grads.append((out, *torch.autograd.grad(out, wide, do)))
        for a, b in zip(*grads):
            assert torch.equal(a, b)


def test_refusals():
    import flash_attn_with_score_b200 as F
    q, k, v, _ = _inputs(1, 4, 2, 64, 64, 64, F16)
    for bad in (dict(window=0), dict(window=-3), dict(window=5, sinks=-1)):
        with pytest.raises(AssertionError):
            F.attention_with_window(q, k, v, **bad)
    with pytest.raises(AssertionError):
        F.attention_with_window(q[:, :3], k, v, 5)
    with pytest.raises(TypeError):
        F.attention_with_window(q.float(), k.float(), v.float(), 5)
    with pytest.raises(RuntimeError):
        F.attention_with_window(q, k, v, 5, kv_splits=9)  # more ranges than key tiles
    with pytest.raises(ValueError):
        F.attention_with_window(q, k, v, 5, backend="other")
    with pytest.raises(RuntimeError):
        F.attention_with_window(q.cpu(), k.cpu(), v.cpu(), 5)
