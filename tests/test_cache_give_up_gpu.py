"""Attention over the 4-bit cache where its waits run out: reported, and nothing but the outputs is touched."""
import ctypes as C

import pytest
import torch

from test_kv_cache_gpu import BF16, F16, Setup, _check

pytestmark = pytest.mark.gpu
POISON = 77.0


class Call:
    """The C call with buffers of the test's own; outputs lie between guards."""

    def __init__(self, s, Hq, M):
        from flash_attn_with_score_b200 import _lib
        from flash_attn_with_score_b200.api import _DTYPES, _tensor
        self.lib, self.s = _lib.load(), s
        B, Hk, _, D = s.k.shape
        self.q = torch.randn((B, Hq, M, D), generator=torch.Generator().manual_seed(1)).to(s.k.dtype).cuda()
        self.all = torch.full((3 * B, Hq, M, D), POISON, dtype=s.k.dtype, device="cuda")
        self.all_L = torch.full((3 * B, Hq, M), POISON, device="cuda")
        self.out, self.L = self.all[B:2 * B], self.all_L[B:2 * B]
        self.p = _lib.Problem(B=B, Hq=Hq, Hk=Hk, M=M, N=1, D=D, dtype=_DTYPES[s.k.dtype], causal=1, sm_scale=D ** -0.5, m_end=M,
                              q=_tensor(self.q), out=_tensor(self.out), log_normalizer=self.L.data_ptr())
        self.batch = _lib.CacheBatch(s.table.data_ptr(), s.lengths.data_ptr(), s.table.stride(0), B, s.table.shape[1])
        n = self.lib.faws_kv_cache_workspace_bytes(C.byref(self.p))
        self.grid = n // (16 + 2 * 8 * (D + 4) * 4)  # (fewer than 16 bytes of a share are alignment's)
        self.ws = torch.zeros(n + 512, dtype=torch.uint8, device="cuda")
        self.ws[n:] = 0x7F
        self.n = n

    def headers(self):
        """(grid, 4) int32: sequence, item, unused, last share."""
        return self.ws[:16 * self.grid].view(torch.int32).view(self.grid, 4)

    def run(self, tiles=None):
        stream = C.c_void_p(torch.cuda.current_stream().cuda_stream)
        args = (C.byref(self.p), C.byref(self.s.cache._struct), C.byref(self.batch), 0, 0)
        ws = (C.c_void_p(self.ws.data_ptr()), self.n, stream)
        if tiles is None:
            assert self.lib.faws_attention_with_kv_cache(*args, *ws) == 0
        else:
            assert self.lib.faws_selftest_kv_cache_give_up(*args, tiles, *ws) == 0
        torch.cuda.synchronize()
        B = self.q.shape[0]
        for t in (self.all, self.all_L):
            assert bool((t[:B] == POISON).all()) and bool((t[2 * B:] == POISON).all())
        assert bool((self.ws[self.n:] == 0x7F).all())


LENS = [700, 130, 1, 0, 300, 129] * 12  # 72 sequences x 8 heads: three tiles to a share, of several items


@pytest.mark.parametrize("dtype,D", [(F16, 128), (BF16, 64), (F16, 16)])
@pytest.mark.parametrize("tiles", [0, 1, 3])
def test_waits_that_run_out(dtype, D, tiles):
    import flash_attn_with_score_b200 as F
    s = Setup(LENS, 8, D, dtype, 16)
    call = Call(s, 16, 2)
    call.run()
    want, want_L = call.out.clone(), call.L.clone()
    assert F.device_status() == 0
    for garbage in (0x7F7F7F7F, -0x01010102, 5):
        call.headers().fill_(garbage)
        t0, t1 = (torch.cuda.Event(enable_timing=True) for _ in range(2))
        t0.record()
        call.run(tiles)
        t1.record()
        torch.cuda.synchronize()
        assert t0.elapsed_time(t1) < 200.0, "the give-up limit is about a millisecond"
        assert F.device_status() == 1
        # nothing to join, or what the share was to begin (its parts are no good, but they are the call's own)
        seq, item, _, last = call.headers().unbind(1)
        begun = last != -1
        assert bool((last < call.grid).all()) and bool((last[begun] > begun.nonzero()[:, 0]).all())
        assert bool(((seq >= 0) & (seq < len(LENS)) & (item >= 0) & (item < 8))[begun].all())
    # the same buffers serve the next call
    call.run()
    assert torch.equal(call.out, want) and torch.equal(call.L, want_L) and F.device_status() == 0
    _check(s, 16, 2)


def test_enough_tiles_are_an_ordinary_call():
    import flash_attn_with_score_b200 as F
    s = Setup(LENS, 8, 64, F16, 64)
    call = Call(s, 16, 2)
    call.run()
    want = call.out.clone()
    call.out.fill_(POISON)
    call.run(10 ** 6)
    assert torch.equal(call.out, want) and F.device_status() == 0


def test_join_of_what_no_call_leaves():
    """Headers out of range: passed over, with the rest joined as ever."""
    import flash_attn_with_score_b200 as F
    s = Setup([3000, 2000], 2, 64, F16, 64)
    call = Call(s, 4, 1)
    call.run()
    want, kept = call.out.clone(), call.headers().clone()
    assert int((kept[:, 3] > torch.arange(call.grid, device="cuda")).sum()) >= 2  # items of several shares
    free = (kept[:, 3] == -1).nonzero()[:, 0].tolist()
    first = torch.arange(call.grid, device="cuda").int()
    big = 2 ** 31 - 1
    bad = [(2, 0, "next"), (-1, 0, "next"), (big, 0, "next"), (-big - 1, 0, "next"), (0, 2, "next"), (0, -1, "next"), (1, big, "next"),
           (0, 0, call.grid), (0, 0, big), (0, 0, -5), (0, 0, -big - 1), (0, 0, "same")]
    for x, (b, item, last) in enumerate(bad):
        for at in free[x::len(bad)]:
            end = at + 1 if last == "next" else at if last == "same" else last
            if last == "next" and end >= call.grid:
                continue
            call.headers()[at] = torch.tensor([b, item, 0, end], dtype=torch.int32, device="cuda")
    assert len(free) >= 2 * len(bad)
    call.out.fill_(POISON)
    call.run(-1)
    joined = (kept[:, 3] > first).nonzero()[:, 0].tolist()
    done = torch.zeros((2, 4), dtype=torch.bool, device="cuda")
    for at in joined:
        b, hk = int(kept[at, 0]), int(kept[at, 1])
        done[b, 2 * hk:2 * hk + 2] = True
    assert bool(done.any())
    assert torch.equal(call.out[done], want[done]) and bool((call.out[~done] == POISON).all())
    assert F.device_status() == 0
