"""A paged cache of keys and values in 4 bits, and the operators on it: writing rows, reading them back, and attention over it.

The operators take sequences as the rest of the package does: tensors (B, H, rows, D) whose rows are the *last* ones of each
sequence.  ``lengths[b]`` counts the tokens of sequence b, those of the call among them, so row m of M stands for position
``lengths[b] - M + m``; rows before position 0 are padding.  ``page_table[b, n // page_size]`` is the page that holds position n.
Both are int32 tensors on the cache's device, so that a decoding step can be captured in a graph and replayed with
others in place (between calls, in stream order: while one runs they stay as they are).

Positions, pages and lengths are known to the device alone.  What does not exist there is never touched: rows on a page outside
the cache, or at a position behind the table's last page, are not written and read as NaN, as do outputs that see such keys (a
row at such a position sees its own); a length below 0 is taken as 0.  ``device_status()`` then has bit 1 set.
"""
from __future__ import annotations

import ctypes as C
import math

import torch

from . import _lib
from .api import _DTYPES, _NO_LIMIT, _no_tangents, _raw_stream, _tensor, maybe_contiguous


class KVCache4:
    """``pages`` pages of ``page_size`` tokens (a power of two, 16 to 65536) for ``heads`` kv heads of ``head_dim``
    (16, 32, 64 or 128), rows of ``dtype`` (float16 or bfloat16): 9/16 of a byte an element (10/16 at head dim 16).

    A row of a head is held in groups of min(32, head_dim) neighbouring elements: a scale bf16(amax / 7) and codes from -7 to
    7, halves rounded away from zero.  A group that holds an infinity or a NaN reads as NaN.  ``k_codes``, ``v_codes`` (pages,
    heads, page_size, head_dim / 2) uint8 and ``k_scales``, ``v_scales`` (pages, heads, page_size, groups) bfloat16 may be copied
    page by page; how codes lie within a row is the library's affair.  The tensors themselves are the cache's for good.

    Attention weights its values in fp16, relative to the largest group of a token's value: groups within 2^-12 of their neighbours
    lose nothing by it, one 2^-16 of them keeps 7 bits, one 2^-20 three."""

    def __init__(self, pages, page_size, heads, head_dim, dtype=torch.float16, device="cuda"):
        if dtype not in _DTYPES:
            raise TypeError(f"dtype must be float16 or bfloat16, got {dtype}")
        assert head_dim in {16, 32, 64, 128}, f"Unsupported head_dim: {head_dim}"
        assert pages > 0 and heads > 0, "pages and heads must be positive"
        assert 16 <= page_size <= 65536 and page_size & (page_size - 1) == 0, "page_size must be a power of two from 16 to 65536"
        self.pages, self.page_size, self.heads, self.head_dim, self.dtype = pages, page_size, heads, head_dim, dtype
        rows = (pages, heads, page_size)
        self.k_codes = torch.zeros((*rows, head_dim // 2), dtype=torch.uint8, device=device)
        self.v_codes = torch.zeros_like(self.k_codes)
        self.k_scales = torch.zeros((*rows, max(1, head_dim // 32)), dtype=torch.bfloat16, device=device)
        self.v_scales = torch.zeros_like(self.k_scales)
        self.device = self.k_codes.device
        if not self.k_codes.is_cuda:
            raise RuntimeError("flash_attn_with_score_b200 runs on CUDA tensors only (no CPU fallback)")
        self._struct = _lib.KVCache(self.k_codes.data_ptr(), self.v_codes.data_ptr(), self.k_scales.data_ptr(),
                                    self.v_scales.data_ptr(), pages, page_size, heads, head_dim, _DTYPES[dtype])
        self._plain = (C.addressof(self._struct), self.device.index)

    def __setattr__(self, name, value):
        if name in self.__dict__:  # (calls go by what the cache was made with)
            raise AttributeError(f"a cache's {name} cannot be replaced: copy into its tensors, or make another cache")
        super().__setattr__(name, value)

    def __delattr__(self, name):  # (nor without)
        raise AttributeError(f"a cache's {name} cannot be deleted: calls go by its tensors' memory")


def _batch(cache, page_table, lengths, B, rows):
    if not isinstance(cache, KVCache4):
        raise TypeError("cache must be a KVCache4")
    assert page_table.dim() == 2 and page_table.shape[0] == B and page_table.shape[1] > 0, (
        f"page_table must be ({B}, pages of a sequence), got {tuple(page_table.shape)}")
    assert lengths.shape == (B,), f"lengths must be ({B},), got {tuple(lengths.shape)}"
    assert max(B, rows, page_table.shape[1]) < 2 ** 31, "sequences, rows and pages of a sequence are counted in 32 bits"
    if page_table.dtype != torch.int32 or lengths.dtype != torch.int32:
        raise TypeError("page_table and lengths must be int32")
    assert page_table.device == cache.device and lengths.device == cache.device, "page_table and lengths must be on the cache's device"
    page_table, lengths = maybe_contiguous(page_table), lengths.contiguous()
    return page_table, lengths, _lib.CacheBatch(page_table.data_ptr(), lengths.data_ptr(), page_table.stride(0), B,
                                                page_table.shape[1])


def _run(cache, name, *args):
    fn, index = getattr(_lib.load(), name), cache.device.index
    if index == torch.cuda.current_device():
        st = fn(*args, _raw_stream(index))
    else:
        with torch.cuda.device(cache.device):
            st = fn(*args, _raw_stream(index))
    _lib.check(st, name)


def kv_cache_write(cache, k, v, page_table, lengths):
    """Quantises k and v (B, Hk, M, D), the last M rows of each sequence, into the cache; padding rows are skipped.  Rows of one
    call are to go to different places (a page that several sequences share may be read by all, written by none).  No gradients: k and v
    that want one are refused."""
    _no_tangents("kv_cache_write", k, v)
    if type(cache) is KVCache4 and _lib.plain("cache_write", *cache._plain, k, v, page_table, lengths):
        return
    assert k.dim() == 4 and k.shape == v.shape, "k and v must have the same (B, Hk, M, D)"
    B, Hk, M, D = k.shape
    table, lens, batch = _batch(cache, page_table, lengths, B, M)
    assert Hk == cache.heads and D == cache.head_dim, f"rows are ({Hk}, {D}) heads and dims, the cache has ({cache.heads}, {cache.head_dim})"
    if k.dtype != cache.dtype or v.dtype != cache.dtype:
        raise TypeError(f"k and v must be {cache.dtype} as the cache is, got {k.dtype}, {v.dtype}")
    assert k.device == cache.device and v.device == cache.device, "k and v must be on the cache's device"
    if torch.is_grad_enabled() and (k.requires_grad or v.requires_grad):
        raise RuntimeError("kv_cache_write has no backward pass: call it under torch.no_grad(), or with detached k and v")
    if B == 0 or M == 0:
        return
    k, v = maybe_contiguous(k), maybe_contiguous(v)
    _run(cache, "faws_kv_cache_write", C.byref(cache._struct), C.byref(batch), C.byref(_tensor(k)), C.byref(_tensor(v)), M)


def kv_cache_read(cache, page_table, lengths, rows):
    """``(k, v)``, each (B, Hk, rows, D) in the cache's dtype: the values that the cache holds of the last ``rows`` positions of each
    sequence, zeros in padding rows."""
    if type(cache) is KVCache4:
        got = _lib.plain("cache_read", *cache._plain, page_table, lengths, rows)
        if got is not None:
            return got
    B = lengths.shape[0]
    table, lens, batch = _batch(cache, page_table, lengths, B, rows)
    assert rows >= 0, "rows must not be negative"
    shape = (B, cache.heads, rows, cache.head_dim)
    k, v = (torch.empty(shape, dtype=cache.dtype, device=cache.device) for _ in range(2))
    if k.numel() > 0:
        _run(cache, "faws_kv_cache_read", C.byref(cache._struct), C.byref(batch), C.byref(_tensor(k)), C.byref(_tensor(v)), rows)
    return k, v


def attention_with_kv_cache(q, cache, page_table, lengths, window=None, sinks=0, sm_scale=None,
                            return_log_normalizer=False):
    """Causal attention of q (B, Hq, M, D), the last M rows of each sequence, over the cache, which holds these rows' keys already.

    A row sees the keys up to its own position; with ``window`` the last ``window`` of them (its own among them) and the
    first ``sinks`` of the sequence.  Rows that see nothing (padding, empty sequences) become 0, their log-normaliser -inf.
    Returns ``out`` (B, Hq, M, D), or ``(out, log_normalizer)``, the latter (B, Hq, M) fp32.  Forward only; any M, made for few rows."""
    assert window is None or window >= 1, "window must be at least 1"
    assert sinks >= 0, "sinks must not be negative"
    window, sinks = min(int(window), _NO_LIMIT) if window is not None else 0, min(int(sinks), _NO_LIMIT)
    _no_tangents("attention_with_kv_cache", q)
    if type(cache) is KVCache4:
        got = _lib.plain("cache_attention", *cache._plain, q, page_table, lengths, window, sinks, sm_scale, return_log_normalizer)
        if got is not None:
            return got
    assert q.dim() == 4, "q must be (B, Hq, M, D)"
    B, H, M, D = q.shape
    table, lens, batch = _batch(cache, page_table, lengths, B, max(H, M))
    assert D == cache.head_dim, f"feature size of q is {D}, the cache's {cache.head_dim}"
    assert H > 0 and H % cache.heads == 0, "number of heads in q must be a multiple of that in the cache"
    if q.dtype != cache.dtype:
        raise TypeError(f"q must be {cache.dtype} as the cache is, got {q.dtype}")
    assert q.device == cache.device, "q must be on the cache's device"
    if torch.is_grad_enabled() and q.requires_grad:
        raise RuntimeError("attention_with_kv_cache has no backward pass: call it under torch.no_grad()")
    q = maybe_contiguous(q)
    out = torch.empty((B, H, M, D), dtype=q.dtype, device=q.device)
    L = torch.empty((B, H, M), dtype=torch.float32, device=q.device) if return_log_normalizer else None
    if out.numel() > 0:
        p = _lib.Problem(B=B, Hq=H, Hk=cache.heads, M=M, N=1, D=D, dtype=_DTYPES[q.dtype], causal=1,
                         sm_scale=float(1.0 / math.sqrt(D) if sm_scale is None else sm_scale), m_begin=0, m_end=M,
                         q=_tensor(q), out=_tensor(out), log_normalizer=L.data_ptr() if L is not None else None)
        with torch.cuda.device(cache.device):  # (as many shares as that device has room for)
            n = _lib.load().faws_kv_cache_workspace_bytes(C.byref(p))
        ws = torch.empty(n, device=q.device, dtype=torch.uint8)
        _run(cache, "faws_attention_with_kv_cache", C.byref(p), C.byref(cache._struct), C.byref(batch),
             window, sinks, C.c_void_p(ws.data_ptr()), n)
    return (out, L) if return_log_normalizer else out
