"""The operators that serve and train with a bounded context, and the 4-bit cache: what is measured of them.

A case is a dict of plain values; ``op`` says which operator:
  window   ``attention_with_window``: causal attention to the last ``window`` keys and the first ``sinks``, forward
  train    the same, forward and backward: output and the three gradients
  rewrite  ``kv_cache_write`` of ``M`` new tokens per sequence, then ``kv_cache_read`` of the same tokens
  cache    ``attention_with_kv_cache``: ``M`` query rows per sequence over a paged 4-bit cache (``window`` 0: all of it)

The ranges that the listed cases stand for, and that ``draw`` spreads its cases over: batch 1 to 64; 4 to 32 query heads,
multi-head or grouped up to seven to a kv head; head dimension 32, 64, 128; prefills and training steps of 128 to 16384
tokens with windows of 64 to 4096 and 0 to 64 sinks; continuations of 1 to 64 rows; caches of 64 to 16384 tokens a sequence in
pages of 16 to 128 tokens, sequences of unlike length; fp16 and bf16.  Lengths are odd as often as round.
"""
import math

import torch

own = False

_HEADS = [(4, 4), (8, 8), (12, 12), (16, 16), (32, 32), (32, 8), (28, 4), (16, 4), (16, 8)]
_DTYPES = {"float16": torch.float16, "bfloat16": torch.bfloat16}


def _case(op, dtype, B, Hq, Hk, M, N, D, window=0, sinks=0, page=0, name=None):
    c = dict(op=op, dtype=dtype, B=B, Hq=Hq, Hk=Hk, M=M, N=N, D=D, window=window, sinks=sinks, page=page)
    return c if name is None else dict(c, name=name)


def listed():
    return [
        # Decoding with a bounded 16-bit cache: one new row per sequence.  Launch and host time count.
        _case("window", "bfloat16", 4, 32, 8, 1, 4096, 128, 1024, 4, name="window_token"),
        # An ordinary prefill of a small grouped-query model.
        _case("window", "float16", 2, 16, 4, 2048, 2048, 64, 512, 4, name="window_prefill"),
        # The largest: a long prompt of a large model.
        _case("window", "bfloat16", 1, 32, 8, 16384, 16384, 128, 4096, 4, name="window_prefill_long"),
        # A training step on texts of whatever length, every size odd.
        _case("train", "float16", 2, 12, 12, 1531, 1531, 64, 300, 7, name="window_train_ragged"),
        # A training step of a grouped-query layer on long texts.
        _case("train", "bfloat16", 1, 28, 4, 8192, 8192, 128, 1024, 4, name="window_train_gqa"),
        # Decoding: one new token per sequence goes into the cache, and is looked at.  Launch time counts.
        _case("rewrite", "float16", 32, 32, 8, 1, 2048, 128, page=64, name="cache_append"),
        # A prompt goes into the cache; its values as the cache holds them come back for the prompt's own attention.
        _case("rewrite", "bfloat16", 4, 32, 8, 8192, 8192, 128, page=64, name="cache_prefill"),
        # The same of a multi-head model with small pages and a ragged batch, some of whose rows are padding.
        _case("rewrite", "float16", 3, 12, 12, 1531, 1531, 64, page=16, name="cache_prefill_ragged"),
        # The smallest: one sequence, one token.
        _case("cache", "bfloat16", 1, 28, 4, 1, 785, 128, page=64, name="cache_token"),
        # Ordinary decoding: sequences of unlike length.
        _case("cache", "bfloat16", 32, 32, 8, 1, 9001, 128, page=64, name="cache_decode"),
        # The largest: long contexts, many of them.
        _case("cache", "float16", 64, 32, 8, 1, 16384, 128, page=128, name="cache_decode_long"),
        # A few drafted tokens a sequence are verified with a window, on a model with seven query heads to a kv head.
        _case("cache", "bfloat16", 16, 28, 4, 4, 8192, 128, 1024, 4, page=16, name="cache_window_draft"),
    ]


def _log_int(rng, lo, hi):
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    while True:
        op = rng.choice(("window", "window", "train", "rewrite", "cache", "cache"))
        dtype = rng.choice(("float16", "bfloat16"))
        Hq, Hk = rng.choice(_HEADS)
        D = rng.choice((32, 64, 128, 128))
        window, sinks, page = _log_int(rng, 64, 4096), rng.choice((0, 1, 4, 4, 7, 16, 64)), 0
        if op in ("window", "train"):
            B = _log_int(rng, 1, 8)
            M = _log_int(rng, 128, 16384)
            N = M
            if op == "window" and rng.random() < 0.4:  # a continuation
                M, N = _log_int(rng, 1, 64), _log_int(rng, 64, 16384)
                N = max(N, M)
        else:
            B = _log_int(rng, 1, 64)
            page = rng.choice((16, 32, 64, 128))
            N = _log_int(rng, 64, 16384)
            if op == "rewrite":
                M = rng.choice((1, 1, N))
                window = sinks = 0
            else:
                M = rng.choice((1, 1, 1, _log_int(rng, 2, 8)))
                if rng.random() < 0.6:
                    window = sinks = 0
        c = _case(op, dtype, B, Hq, Hk, M, N, D, window, sinks, page)
        most = work(max((x for x in listed() if x["op"] == op), key=lambda x: work(x)["flops"] + work(x)["bytes"] * 250))
        w = work(c)
        if w["flops"] <= most["flops"] and w["bytes"] <= most["bytes"]:
            return c


def _lengths(case):
    """Tokens of each sequence, the new ones among them: from a quarter of N up to N, the first has N."""
    return [max(1, int(case["N"] * (1.0 - 0.75 * ((b * 0.6180339887498949) % 1.0)))) for b in range(case["B"])]


def _visible(n_keys, rows, window, sinks):
    """Visible (row, key) pairs of the last ``rows`` rows of a sequence of ``n_keys``."""
    total = 0
    for p in range(max(0, n_keys - rows), n_keys):
        w = min(window or n_keys, p + 1)
        total += w + min(sinks, p + 1 - w)
    return total


def _keys_read(n_keys, rows, window, sinks):
    """Keys that any of those rows sees."""
    w = min(n_keys, (window or n_keys) + rows - 1)
    return w + min(sinks, n_keys - w)


def work(case):
    op, B, Hq, Hk, M, N, D = (case[x] for x in ("op", "B", "Hq", "Hk", "M", "N", "D"))
    window, sinks = case["window"], case["sinks"]
    if op in ("window", "train"):
        pairs = B * Hq * _visible(N, M, window, sinks)
        q, kv = B * Hq * M * D * 2, B * Hk * _keys_read(N, M, window, sinks) * D * 2
        if op == "window":
            return {"bytes": 2 * q + 2 * kv, "flops": 4 * D * pairs}
        # q, dout in, out, dq out; k, v in, dk, dv out
        return {"bytes": 4 * q + 4 * kv, "flops": 14 * D * pairs}
    cached = D // 2 + 2 * (D // min(32, D))  # bytes of a cached row
    if op == "rewrite":
        rows = Hk * sum(min(M, n) for n in _lengths(case))
        return {"bytes": 2 * (rows * (D * 2 + cached) + rows * cached + B * Hk * M * D * 2), "flops": 6 * rows * D}
    lens = _lengths(case)
    keys = Hk * sum(_keys_read(n, M, window, sinks) for n in lens)
    pairs = Hq * sum(_visible(n, M, window, sinks) for n in lens)
    return {"bytes": 2 * keys * cached + 2 * B * Hq * M * D * 2, "flops": 4 * D * pairs}


# ---------------------------------------------------------------------------------------------- inputs
def _generator(seed, salt):
    g = torch.Generator(device="cuda")
    g.manual_seed((int(seed) * 1000003 + salt) & 0x7FFFFFFF)
    return g


def _normal(shape, dtype, seed, salt):
    return torch.randn(shape, generator=_generator(seed, salt), device="cuda", dtype=torch.float32).to(dtype)


def _history(case, seed, b):
    """Keys and values (1, Hk, N, D) of sequence b: normal, with the outliers of some channels and rows."""
    n, Hk, D, dtype = _lengths(case)[b], case["Hk"], case["D"], _DTYPES[case["dtype"]]
    g = _generator(seed, 100 + b)
    k, v = (torch.randn((1, Hk, n, D), generator=g, device="cuda") for _ in range(2))
    k = k * (1.0 + 3.0 * (torch.rand((1, Hk, 1, D), generator=g, device="cuda") > 0.95))
    v = v * (1.0 + 3.0 * (torch.rand((1, Hk, n, 1), generator=g, device="cuda") > 0.98))
    return k.to(dtype), v.to(dtype)


def _new_rows(case, seed):
    shape = (case["B"], case["Hk"], case["M"], case["D"])
    return (_normal(shape, _DTYPES[case["dtype"]], seed, 11), _normal(shape, _DTYPES[case["dtype"]], seed, 12))


def _pages(case, seed):
    """A page table (B, P) of pages in no order, and how many pages there are."""
    per = (case["N"] + case["page"] - 1) // case["page"]
    order = torch.randperm(case["B"] * per, generator=_generator(seed, 7), device="cuda")
    return order.view(case["B"], per).to(torch.int32), case["B"] * per


def prepare(case, seed):
    op, B, Hq, Hk, M, N, D = (case[x] for x in ("op", "B", "Hq", "Hk", "M", "N", "D"))
    dtype = _DTYPES[case["dtype"]]
    st = {"case": case}
    if op in ("window", "train"):
        st["q"] = _normal((B, Hq, M, D), dtype, seed, 1)
        st["k"], st["v"] = _normal((B, Hk, N, D), dtype, seed, 2), _normal((B, Hk, N, D), dtype, seed, 3)
        if op == "train":
            st["dout"] = _normal((B, Hq, M, D), dtype, seed, 4)
            if own:
                for x in ("q", "k", "v"):
                    st[x].requires_grad_(True)
        return st
    st["table"], n_pages = _pages(case, seed)
    st["lengths"] = torch.tensor(_lengths(case), dtype=torch.int32, device="cuda")
    if own:
        from flash_attn_with_score_b200 import KVCache4, kv_cache_write
        st["cache"] = KVCache4(n_pages, case["page"], Hk, D, dtype=dtype, device="cuda")
    else:  # codes and scales, a row of a head after the other
        g = min(32, D)
        st["cache"] = [(torch.zeros((n_pages, case["page"], Hk, D), dtype=torch.int8, device="cuda"),
                        torch.zeros((n_pages, case["page"], Hk, D // g), dtype=torch.bfloat16, device="cuda")) for _ in range(2)]
    if op == "rewrite":
        st["k"], st["v"] = _new_rows(case, seed)
        return st
    st["q"] = _normal((B, Hq, M, D), dtype, seed, 1)
    for b in range(B):
        k, v = _history(case, seed, b)
        if own:
            kv_cache_write(st["cache"], k, v, st["table"][b:b + 1], st["lengths"][b:b + 1])
        else:
            _plain_write(st["cache"], k, v, st["table"][b:b + 1], st["lengths"][b:b + 1])
    return st


# ---------------------------------------------------------------------------------------------- plain forms
def _plain_window(q, k, v, window, sinks, dout=None):
    """Blocks of query rows against the keys that any of them sees; gradients by the formulas."""
    B, Hq, M, D = q.shape
    Hk, N = k.shape[1], k.shape[2]
    G, scale = Hq // Hk, 1.0 / math.sqrt(D)
    qf, kf, vf = q.float().view(B, Hk, G, M, D), k.float(), v.float()
    out = torch.empty((B, Hk, G, M, D), device=q.device)
    if dout is not None:
        gf, dq, dk, dv = dout.float().view(B, Hk, G, M, D), torch.empty_like(qf), torch.zeros_like(kf), torch.zeros_like(vf)
    step = 512
    for r in range(0, M, step):
        e = min(M, r + step)
        pos = torch.arange(r, e, device=q.device) + (N - M)
        lo, hi = max(0, r + N - M - window + 1), e + N - M
        head = min(sinks, lo)
        keys = torch.cat([torch.arange(0, head, device=q.device), torch.arange(lo, hi, device=q.device)])
        kb, vb = kf[:, :, keys].unsqueeze(2), vf[:, :, keys].unsqueeze(2)
        s = torch.matmul(qf[:, :, :, r:e], kb.transpose(-1, -2)) * scale
        see = (keys[None, :] <= pos[:, None]) & ((keys[None, :] > pos[:, None] - window) | (keys[None, :] < sinks))
        s = torch.where(see, s, torch.full_like(s, -float("inf")))
        p = torch.exp(s - s.amax(-1, keepdim=True))
        p = p / p.sum(-1, keepdim=True)
        o = torch.matmul(p, vb)
        out[:, :, :, r:e] = o
        if dout is not None:
            g = gf[:, :, :, r:e]
            ds = p * (torch.matmul(g, vb.transpose(-1, -2)) - (o * g).sum(-1, keepdim=True))
            dq[:, :, :, r:e] = torch.matmul(ds, kb) * scale
            dk_b = torch.matmul(ds.transpose(-1, -2), qf[:, :, :, r:e]).sum(2) * scale
            dv_b = torch.matmul(p.transpose(-1, -2), g).sum(2)
            dk[:, :, :head] += dk_b[:, :, :head]
            dk[:, :, lo:hi] += dk_b[:, :, head:]
            dv[:, :, :head] += dv_b[:, :, :head]
            dv[:, :, lo:hi] += dv_b[:, :, head:]
    out = out.view(B, Hq, M, D).to(q.dtype)
    if dout is None:
        return out
    return out, dq.view(B, Hq, M, D).to(q.dtype), dk.to(k.dtype), dv.to(v.dtype)


def _quantise(x):
    """Codes (int8) and scales (bf16) of rows in groups of up to 32: halves go away from zero."""
    D = x.shape[-1]
    g = min(32, D)
    xg = x.float().view(*x.shape[:-1], D // g, g)
    s = (xg.abs().amax(-1) / 7.0).to(torch.bfloat16)
    s = torch.where(s.float() < 2.0 ** -126, torch.zeros_like(s), s)
    sf = s.float().unsqueeze(-1)
    c = torch.where(sf > 0, torch.floor(xg.abs() / sf + 0.5), torch.zeros_like(xg)) * torch.sign(xg)
    return c.to(torch.int8).view(x.shape), s


def _slots(table, lengths, rows, page):
    """Page and place in it of the last ``rows`` positions of each sequence, and which of them exist."""
    pos = lengths.long()[:, None] - rows + torch.arange(rows, device=table.device)[None, :]
    real = pos >= 0
    at = pos.clamp(min=0)
    return torch.gather(table.long(), 1, at // page), at % page, real


def _plain_write(cache, k, v, table, lengths):
    page, place, real = _slots(table, lengths, k.shape[2], cache[0][0].shape[1])
    for x, (codes, scales) in ((k, cache[0]), (v, cache[1])):
        c, s = _quantise(x)
        codes[page[real], place[real]] = c.transpose(1, 2)[real]
        scales[page[real], place[real]] = s.transpose(1, 2)[real]


def _values(codes, scales):
    D = codes.shape[-1]
    g = D // scales.shape[-1]
    return (codes.float().view(*codes.shape[:-1], D // g, g) * scales.float().unsqueeze(-1)).view(codes.shape)


def _plain_read(cache, table, lengths, rows, dtype):
    page, place, real = _slots(table, lengths, rows, cache[0][0].shape[1])
    got = []
    for codes, scales in cache:
        x = _values(codes[page, place], scales[page, place])
        x = torch.where(real[:, :, None, None], x, torch.zeros_like(x))
        got.append(x.transpose(1, 2).contiguous().to(dtype))
    return got


def _plain_cache_attention(q, cache, table, lengths, lens, window, sinks):
    B, Hq, M, D = q.shape
    out = torch.zeros((B, Hq, M, D), device=q.device)
    page_size = cache[0][0].shape[1]
    for b in range(B):
        n = lens[b]
        lo = max(0, n - M - (window or n) + 1)
        head = min(sinks, lo)
        keys = torch.cat([torch.arange(0, head, device=q.device), torch.arange(lo, n, device=q.device)])
        page, place = table[b].long()[keys // page_size], keys % page_size
        k, v = (_values(codes[page, place], scales[page, place]).transpose(0, 1) for codes, scales in cache)
        G = Hq // k.shape[0]
        pos = torch.arange(n - M, n, device=q.device)
        s = torch.matmul(q[b].float().view(-1, G * M, D), k.transpose(-1, -2)) / math.sqrt(D)
        see = keys[None, :] <= pos[:, None]
        if window:
            see = see & ((keys[None, :] > pos[:, None] - window) | (keys[None, :] < sinks))
        s = torch.where(see.repeat(G, 1), s, torch.full_like(s, -float("inf")))
        top = s.amax(-1, keepdim=True)
        p = torch.exp(s - torch.where(top > -float("inf"), top, torch.zeros_like(top)))
        o = torch.matmul(p, v)
        total = p.sum(-1, keepdim=True)
        out[b] = torch.where(total > 0, o / total, torch.zeros_like(o)).view(Hq, M, D)
    return out.to(q.dtype)


def run(state):
    case = state["case"]
    op, window, sinks = case["op"], case["window"], case["sinks"]
    if own:
        import flash_attn_with_score_b200 as F
        if op == "window":
            return F.attention_with_window(state["q"], state["k"], state["v"], window, sinks)
        if op == "train":
            out = F.attention_with_window(state["q"], state["k"], state["v"], window, sinks)
            return (out.detach(), *torch.autograd.grad(out, (state["q"], state["k"], state["v"]), state["dout"]))
        if op == "rewrite":
            F.kv_cache_write(state["cache"], state["k"], state["v"], state["table"], state["lengths"])
            return F.kv_cache_read(state["cache"], state["table"], state["lengths"], case["M"])
        return F.attention_with_kv_cache(state["q"], state["cache"], state["table"], state["lengths"], window or None, sinks)
    if op == "window":
        return _plain_window(state["q"], state["k"], state["v"], window, sinks)
    if op == "train":
        return _plain_window(state["q"], state["k"], state["v"], window, sinks, state["dout"])
    if op == "rewrite":
        _plain_write(state["cache"], state["k"], state["v"], state["table"], state["lengths"])
        return tuple(_plain_read(state["cache"], state["table"], state["lengths"], case["M"], _DTYPES[case["dtype"]]))
    return _plain_cache_attention(state["q"], state["cache"], state["table"], state["lengths"], _lengths(case), window, sinks)


# ---------------------------------------------------------------------------------------------- 64 bits
def _exact_head(q, k, v, window, sinks):
    """One head in 64 bits: the whole score matrix."""
    M, N = q.shape[0], k.shape[0]
    i = torch.arange(M, device=q.device, dtype=torch.float64)[:, None] + float(N - M)
    j = torch.arange(N, device=q.device, dtype=torch.float64)[None, :]
    hidden = (j > i) | ((i - j >= float(window or N + 1)) & (j >= float(sinks)))
    s = (q @ k.mT).mul_(q.shape[-1] ** -0.5).masked_fill_(hidden, -1.0e300)
    # (a row that sees nothing has equal weights until its output is cleared)
    w = torch.softmax(s, -1)
    return (w @ v).masked_fill(hidden.all(-1, keepdim=True), 0.0)


def _exact_values(x):
    """What the cache holds of x, in 64 bits."""
    D = x.shape[-1]
    g = min(32, D)
    xs = torch.stack(x.double().split(g, -1), -2)
    s = xs.abs().max(-1, keepdim=True).values.div(7).to(torch.bfloat16).double()
    s[s < 2.0 ** -126] = 0.0
    q = torch.trunc(xs / s + torch.copysign(torch.full_like(xs, 0.5), xs))
    return torch.where(s > 0, q * s, torch.zeros_like(xs)).reshape(x.shape)


def exact(case, seed):
    op, B, Hq, Hk, M, N = (case[x] for x in ("op", "B", "Hq", "Hk", "M", "N"))
    window, sinks, G = case["window"], case["sinks"], Hq // Hk
    dtype, D = _DTYPES[case["dtype"]], case["D"]
    if op == "rewrite":
        got = []
        lens = _lengths(case)
        for x in _new_rows(case, seed):
            y = _exact_values(x)
            for b in range(B):
                y[b, :, :max(0, M - lens[b])] = 0.0
            got.append(y)
        return tuple(got)
    if op == "cache":
        q = _normal((B, Hq, M, D), dtype, seed, 1)
        out = torch.zeros((B, Hq, M, D), dtype=torch.float64, device="cuda")
        for b in range(B):
            k, v = _history(case, seed, b)
            k, v = _exact_values(k[0]), _exact_values(v[0])
            n = k.shape[1]
            rows = min(M, n)
            for h in range(Hq):
                out[b, h, M - rows:] = _exact_head(q[b, h, M - rows:].double(), k[h // G], v[h // G], window, sinks)
        return out
    q = _normal((B, Hq, M, D), dtype, seed, 1).double()
    k, v = _normal((B, Hk, N, D), dtype, seed, 2).double(), _normal((B, Hk, N, D), dtype, seed, 3).double()
    out = torch.empty_like(q)
    if op == "window":
        for b in range(B):
            for h in range(Hq):
                out[b, h] = _exact_head(q[b, h], k[b, h // G], v[b, h // G], window, sinks)
        return out
    g = _normal((B, Hq, M, D), dtype, seed, 4).double()
    dq, dk, dv = torch.empty_like(q), torch.zeros_like(k), torch.zeros_like(v)
    for b in range(B):
        for h in range(Hq):
            x = [t.detach().clone().requires_grad_(True) for t in (q[b, h], k[b, h // G], v[b, h // G])]
            with torch.enable_grad():
                o = _exact_head(*x, window, sinks)
                grads = torch.autograd.grad(o, x, g[b, h])
            out[b, h], dq[b, h] = o.detach(), grads[0]
            dk[b, h // G] += grads[1]
            dv[b, h // G] += grads[2]
    return out, dq, dk, dv
