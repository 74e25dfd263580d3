"""The operators of the cache that is held in four bits, as cases whose time can be taken and whose results can be checked.

* ``store``: `tokens` new tokens of each of `requests` requests, behind the tokens that those hold already: their keys and values
  (rows of `kv_heads` heads of `head_dim` elements, as the projection and the rotation leave them) are quantised into the pages, and
  the rows are read back as the values they are held as.
* ``read``: the rows that the requests hold are read back as values, in pages, as a prompt's portion reads what lies before it.
  With a window: the rows its first token sees, and the kept first ones.
* ``attention``: the last `tokens` tokens of every request attend to the request's rows.  Options as the designs have them: a window
  with kept first keys, a sink, capped scores, a bias by distance.

How rows are held: a group is 32 neighbouring elements of one token's head (heads are held as 64, 128 or 256 elements, the rest zeros).
With e its element of largest magnitude (the positive one of two), s = -e / 8 with e rounded to five significant bits, ties to even; an
element x is held as the code c = x / s rounded to the nearest whole number, ties to even, within -8 .. 7, and stands for c s.  Groups whose e is below
2^-96 are held as zeros, those with an element of 2^120 or more, or none that is a number, as NaN.  A page of one layer and kv head is
one run of bytes: the keys' codes, the values' codes, the keys' scales, the values' scales, token after token; eight codes (plus 8) are a
little-endian word: element 2 i at bit 4 i, element 2 i + 1 at bit 16 + 4 i; scales are bfloat16.
"""
from __future__ import annotations

import math

import numpy as np
import torch

own = False
DEVICE = "cuda:0"

# ---- the cases ---------------------------------------------------------------------------------------------------------


def _case(name, op, requests, context, tokens, heads, kv_heads, head_dim, page_size=64, dtype="bfloat16", window=0, keep_first=0, sink=False,
          softcap=0.0, bias=0, ragged=True):
    c = {"name": name, "op": op, "requests": requests, "context": context, "tokens": tokens, "heads": heads, "kv_heads": kv_heads,
         "head_dim": head_dim, "page_size": page_size, "dtype": dtype, "window": window, "keep_first": keep_first, "sink": sink, "softcap": softcap,
         "bias": bias, "ragged": ragged}
    return c if name else {k: v for k, v in c.items() if k != "name"}


def listed():
    return [
        # a decode step of eight conversations: one token each, latency counts (Llama-3-8B's heads)
        _case("store-8x1", "store", 8, 8128, 1, 32, 8, 128, ragged=False),
        # a prompt's portion as a step's token budget cuts it
        _case("store-2048", "store", 1, 2048, 2048, 32, 8, 128),
        # three prompts in true 32 bit: a head size and pages of odd sizes
        _case("store-3x517-float32", "store", 3, 700, 517, 6, 3, 100, page_size=24, dtype="float32"),
        # what lies before the portions of four long prompts
        _case("read-4x8192", "read", 4, 8192, 0, 32, 8, 128, ragged=False),
        # a window's rows and the kept first ones, ragged contexts
        _case("read-11-window", "read", 11, 3001, 0, 8, 2, 80, page_size=16, window=900, keep_first=20),
        # one conversation with a small model: latency (Llama-3.2-1B's heads)
        _case("decode-1x640", "attention", 1, 640, 1, 32, 8, 64),
        # the benchmark's own step: eight long conversations (Llama-3-8B's heads)
        _case("decode-8x8192", "attention", 8, 8192, 1, 32, 8, 128, ragged=False),
        # a busy server: 64 conversations of unequal length, a head for every kv head (Llama-2-13B's)
        _case("decode-64-ragged-heads40", "attention", 64, 3840, 1, 40, 40, 128),
        # one very long document
        _case("decode-1x131072", "attention", 1, 131072, 1, 32, 8, 128),
        # a windowed design: kept first keys, a sink, a bias by distance, ragged
        _case("decode-32-window-sink-bias", "attention", 32, 5000, 1, 16, 4, 128, window=1024, keep_first=4, sink=True, bias=1024),
        # four drafted tokens of a few requests in true 32 bit, capped scores
        _case("tokens-5x4-float32-cap", "attention", 5, 1500, 4, 8, 2, 64, dtype="float32", softcap=30.0),
        # a prompt's portion behind what it has run already
        _case("portion-512-of-4096", "attention", 1, 4096, 512, 32, 8, 128),
    ]


def draw(rng):
    log = lambda a, b: int(round(math.exp(rng.uniform(math.log(a), math.log(b)))))
    op = rng.choice(["store", "read", "attention", "attention"])
    dtype = "float32" if rng.random() < 0.3 else "bfloat16"
    kv_heads, group = rng.choice([1, 2, 3, 4, 8, 16]), rng.choice([1, 2, 3, 4, 5, 7, 8])
    head_dim, page = rng.choice([16, 48, 64, 64, 80, 96, 100, 128, 128, 192, 256]), rng.choice([8, 16, 24, 32, 64, 64, 128])
    requests, context = log(1, 64), log(1, 40000)
    window = log(8, 3000) if op != "store" and rng.random() < 0.3 else 0
    keep = rng.choice([0, 1, 4, 33]) if window else 0
    most = 16_000_000 // (kv_heads * head_dim)         # rows of all requests
    if op == "store":
        tokens = rng.choice([1, 1, log(2, 2048)])
        tokens = min(tokens, context, max(1, most // (4 * requests)))
        context = max(tokens, min(context, 4 * most // requests))
        return _case(None, op, requests, context, tokens, kv_heads * group, kv_heads, head_dim, page, dtype)
    context = max(1, min(context, 4 * most // requests if op == "attention" else most // requests))
    if op == "read":
        return _case(None, op, requests, context, 0, kv_heads * group, kv_heads, head_dim, page, dtype, window, keep)
    tokens = rng.choice([1, 1, 1, rng.randint(2, 6), log(8, 300)])
    if tokens > 6:                                     # a portion of a prompt
        requests, context = min(requests, 4), min(context, 2500 if dtype == "float32" or head_dim > 128 or head_dim % 16 else 6000)
    tokens = min(tokens, context)
    extra = rng.choice(["", "", "", "cap", "bias"])
    return _case(None, op, requests, context, tokens, kv_heads * group, kv_heads, head_dim, page, dtype, window, keep, rng.random() < 0.3,
                 30.0 if extra == "cap" else 0.0, log(2, 2000) if extra == "bias" else 0)


def _contexts(case):
    """The requests' lengths: the first has the case's, with `ragged` the others down to a third of it."""
    least = max(1, case["tokens"])
    return [max(least, int(case["context"] * (1.0 - 0.66 * case["ragged"] * ((0.618 * i) % 1.0)))) for i in range(case["requests"])]


def _held(head_dim):
    return 64 if head_dim <= 64 else 128 if head_dim <= 128 else 256


def _block_bytes(case):
    return case["page_size"] * (_held(case["head_dim"]) + _held(case["head_dim"]) // 8)


def _seen(case, end, tokens):
    """(first position that a request's last `tokens` tokens see, rows seen ahead of it)."""
    first = max(0, end - tokens - case["window"] + 1) if case["window"] else 0
    return first, min(case["keep_first"], first)


def work(case):
    es, K, D, hs = (4 if case["dtype"] == "float32" else 2), case["kv_heads"], case["head_dim"], _held(case["head_dim"])
    row, held = 2 * K * D * es, 2 * K * (hs // 2 + hs // 16)
    if case["op"] == "store":
        n = case["requests"] * case["tokens"]
        return {"bytes": n * (2 * row + 2 * held), "flops": 2 * n * 2 * K * D}
    tokens = max(1, case["tokens"])
    spans = [(end, *_seen(case, end, tokens)) for end in _contexts(case)]
    rows = sum(end - first + kept for end, first, kept in spans)
    if case["op"] == "read":
        return {"bytes": rows * (row + held), "flops": rows * 2 * K * D}
    pairs = 0
    for end, first, kept in spans:
        for p in range(end - tokens, end):
            w = min(p + 1, case["window"]) if case["window"] else p + 1
            pairs += w + min(kept, p + 1 - w)
    n = case["requests"] * tokens
    return {"bytes": rows * held + 2 * n * case["heads"] * D * es, "flops": 4 * pairs * case["heads"] * D}


# ---- inputs ------------------------------------------------------------------------------------------------------------


def _quantise(x):
    """(codes int32, scales float32) of x [..., D] float32, groups of 32 along the held head."""
    D, hs = x.shape[-1], _held(x.shape[-1])
    g = torch.nn.functional.pad(x, (0, hs - D)).reshape(*x.shape[:-1], hs // 32, 32)
    hi, lo = g.amax(-1), g.amin(-1)
    e = torch.where(hi >= -lo, hi, lo)
    bits = e.view(torch.int32)
    near = ((bits + 0x3FFFF + ((bits >> 19) & 1)) & -0x80000).view(torch.float32)
    size = torch.maximum(hi.abs(), lo.abs())
    fine = size < 2.0 ** 120
    s = torch.where(fine, torch.where(size < 2.0 ** -96, torch.zeros_like(e), -near / 8), torch.full_like(e, float("nan")))
    live = fine & (s != 0)
    c = torch.where(live[..., None], (g / torch.where(live, s, torch.ones_like(s))[..., None]).round().clamp(-8, 7), torch.zeros_like(g))
    return c.to(torch.int32).reshape(*x.shape[:-1], hs), s


def _packed(codes):
    """Words of eight codes, as bytes: [..., hs] -> uint8 [..., hs / 2]."""
    u = (codes + 8).reshape(*codes.shape[:-1], -1, 8)
    w = u[..., 0]
    for i in range(1, 8):
        w = w | (u[..., i] << (4 * (i // 2) + 16 * (i % 2)))
    return w.contiguous().view(torch.uint8)


def _put(cache, case, pages, at, k, v):
    """Rows k, v [N, K, D] float32 into page pages[i], row at[i] of the cache [pages, 1, K, bytes]."""
    P, K, hs = case["page_size"], case["kv_heads"], _held(case["head_dim"])
    ng = hs // 32
    heads = torch.arange(K, device=cache.device)[None, :, None]
    flat = cache.view(-1)
    base = (pages.long()[:, None] * K)[..., None] * cache.shape[-1] + heads * cache.shape[-1]
    for which, x in ((0, k), (1, v)):
        codes, s = _quantise(x)
        for data, start, size in ((_packed(codes), which * P * hs // 2, hs // 2),
                                  (s.to(torch.bfloat16).view(torch.uint8).reshape(*s.shape[:-1], 2 * ng), P * hs + which * P * ng * 2, 2 * ng)):
            where = base + start + at.long()[:, None, None] * size + torch.arange(size, device=cache.device)
            flat[where] = data


def prepare(case, seed):
    B, T, K, D, P = case["requests"], max(1, case["tokens"]), case["kv_heads"], case["head_dim"], case["page_size"]
    dt = torch.float32 if case["dtype"] == "float32" else torch.bfloat16
    g = torch.Generator(device=DEVICE).manual_seed(seed * 7919 + 11)
    ends = np.array(_contexts(case), dtype=np.int64)
    pages = -(-ends // P)
    most = int(pages.max()) + 1
    order = torch.randperm(int(pages.sum()) + 3, generator=g, device=DEVICE).to(torch.int32)
    table = torch.full((B, most), -1, dtype=torch.int32, device=DEVICE)
    start = np.concatenate([[0], np.cumsum(pages)])
    owner = torch.from_numpy(np.repeat(np.arange(B), pages)).to(DEVICE)
    slot = torch.from_numpy(np.concatenate([np.arange(n) for n in pages])).to(DEVICE)
    table[owner, slot] = order[:int(pages.sum())]
    cache = torch.zeros((int(pages.sum()) + 3, 1, K, _block_bytes(case)), dtype=torch.uint8, device=DEVICE)
    i32 = lambda a: torch.from_numpy(np.ascontiguousarray(a, dtype=np.int32)).to(DEVICE)
    # keys have a few channels that are much larger than the rest, and so a mean; values are plain
    loud = 1.0 + 5.0 * (torch.rand((K, D), generator=g, device=DEVICE) < 0.04)
    mean = torch.randn((K, D), generator=g, device=DEVICE) * (loud - 1.0)

    def rows(n):
        k = (torch.randn((n, K, D), generator=g, device=DEVICE) * loud.sqrt() + 0.3 * mean).to(dt)
        return k, torch.randn((n, K, D), generator=g, device=DEVICE).to(dt)

    # what the requests hold, a few thousand rows at a time
    if case["op"] != "store":
        held = np.concatenate([np.arange(n) for n in ends])
        of = torch.from_numpy(np.repeat(np.arange(B), ends)).to(DEVICE)
        held = torch.from_numpy(held).to(DEVICE)
        step = max(1, (1 << 26) // (K * D))
        for a in range(0, held.numel(), step):
            p, r = held[a:a + step], of[a:a + step]
            k, v = rows(p.numel())
            _put(cache, case, table[r, p // P], p % P, k.float(), v.float())
    n = B * T
    pos = (ends[:, None] - T + np.arange(T)[None, :]).reshape(-1)
    st = {"case": case, "cache": cache, "table": table, "ends": i32(ends), "pos0": i32(ends - T), "positions": i32(pos),
          "tok_seg": i32(np.repeat(np.arange(B), T)), "seg_start": i32(np.arange(B) * T), "seg_len": i32(np.full(B, T)),
          "len_host": np.full(B, T, dtype=np.int32), "pos0_host": (ends - T).astype(np.int32)}
    if case["op"] == "store":
        k, v = rows(n)
        # rows of the fused projection: queries, keys, values side by side
        qkv = torch.zeros((n, (case["heads"] + 2 * K) * D), dtype=dt, device=DEVICE)
        qkv[:, case["heads"] * D:] = torch.cat([k.reshape(n, -1), v.reshape(n, -1)], dim=1)
        st["k"], st["v"] = qkv[:, case["heads"] * D:(case["heads"] + K) * D], qkv[:, (case["heads"] + K) * D:]
    # the rows that are read back, the pages that hold them, and where each lies in the output
    if case["op"] == "store":
        first, kept = ends - T, np.zeros(B, dtype=np.int64)
    else:
        both = [_seen(case, int(e), 1) for e in ends]
        first, kept = np.array([a for a, _ in both]), np.array([b for _, b in both])
    lists = [np.concatenate([np.arange(min(-(-kp // P), f // P)), np.arange(f // P, (e - 1) // P + 1)]) for f, kp, e in zip(first, kept, ends)]
    st["first"], st["keep"] = i32(first), int(case["keep_first"]) if case["op"] == "read" else 0
    st["out_seg"] = torch.from_numpy(np.repeat(np.arange(B), [len(x) for x in lists])).to(DEVICE)
    st["out_page"] = torch.from_numpy(np.concatenate(lists)).to(DEVICE).long()
    st["out_pages"] = int(st["out_page"].numel())
    st["dtype"] = dt
    if case["op"] == "attention":
        H = case["heads"]
        q = torch.randn((n, H * D), generator=g, device=DEVICE) * (1.0 + torch.rand((n, H), generator=g, device=DEVICE)).repeat_interleave(D, dim=1)
        st["q"] = q.to(dt)
        st["scale"] = D ** -0.5
        st["sink"] = torch.randn(H, generator=g, device=DEVICE) if case["sink"] else None
        st["bias"] = None
        if case["bias"]:
            far = torch.arange(case["bias"], device=DEVICE, dtype=torch.float32)
            slope = 0.5 + torch.rand((H, 1), generator=g, device=DEVICE)
            st["bias"] = (-slope * torch.log1p(far) / st["scale"]).contiguous()
    return st


# ---- the plain forms ---------------------------------------------------------------------------------------------------


def _values(blocks, case):
    """Keys and values [..., 2, page, D] float32 that blocks [..., bytes] of the cache stand for."""
    P, hs, D = case["page_size"], _held(case["head_dim"]), case["head_dim"]
    lead, ng = blocks.shape[:-1], hs // 32
    words = blocks[..., :P * hs].contiguous().view(torch.int32).reshape(*lead, 2, P, hs // 8, 1)
    shifts = torch.tensor([0, 16, 4, 20, 8, 24, 12, 28], dtype=torch.int32, device=blocks.device)
    codes = ((words >> shifts) & 15) - 8
    s = blocks[..., P * hs:].contiguous().view(torch.bfloat16).float().reshape(*lead, 2, P, ng, 1)
    return (codes.reshape(*lead, 2, P, ng, 32) * s).reshape(*lead, 2, P, hs)[..., :D]


def _plain_read(st):
    case = st["case"]
    P, B = case["page_size"], case["requests"]
    pages = st["table"][st["out_seg"], st["out_page"]].long()
    x = _values(st["cache"][pages, 0], case).transpose(1, 2)                  # [pages, 2, K, P, D]
    pos = st["out_page"][:, None] * P + torch.arange(P, device=x.device)
    first, end = st["first"].long()[st["out_seg"]][:, None], st["ends"].long()[st["out_seg"]][:, None]
    seen = ((pos >= first) | (pos < st["keep"])) & (pos < end)
    return torch.where(seen[:, None, None, :, None], x, torch.zeros_like(x)).to(st["dtype"])


def _plain_store(st):
    case = st["case"]
    K, D, P = case["kv_heads"], case["head_dim"], case["page_size"]
    n = st["k"].shape[0]
    at = st["positions"].long()
    _put(st["cache"], case, st["table"][st["tok_seg"].long(), at // P], at % P, st["k"].float().reshape(n, K, D), st["v"].float().reshape(n, K, D))
    return _plain_read(st)


def _plain_attention(st):
    case = st["case"]
    B, H, K, D, P = case["requests"], case["heads"], case["kv_heads"], case["head_dim"], case["page_size"]
    T, G = case["tokens"], H // K
    n_pages = st["table"].shape[1] - 1
    x = _values(st["cache"][st["table"][:, :n_pages].clamp(min=0).long(), 0], case)            # [B, pages, K, 2, P, D]
    x = x.permute(3, 0, 2, 1, 4, 5).reshape(2, B, K, n_pages * P, D)
    key = torch.arange(n_pages * P, device=x.device)
    pos = st["positions"].long().reshape(B, T)[:, :, None]
    seen = key <= pos
    if case["window"]:
        seen = seen & ((key > pos - case["window"]) | (key < case["keep_first"]))              # [B, T, keys]
    q = st["q"].float().reshape(B, T, K, G, D).permute(0, 2, 1, 3, 4).reshape(B, K, T * G, D)
    s = (q @ x[0].transpose(-1, -2)).reshape(B, K, T, G, -1) * st["scale"]
    if st["bias"] is not None:
        far = (pos - key).clamp(0, case["bias"] - 1)                                           # [B, T, keys]
        s = s + (st["bias"] * st["scale"])[:, far].reshape(K, G, B, T, -1).permute(2, 0, 3, 1, 4)
    if case["softcap"]:
        s = case["softcap"] * torch.tanh(s / case["softcap"])
    seen = seen[:, None, :, None, :]
    s = torch.where(seen, s, torch.full_like(s, -math.inf))
    m = s.amax(-1, keepdim=True)
    p = torch.exp(s - m)
    total = p.sum(-1, keepdim=True)
    if st["sink"] is not None:
        total = total + torch.exp(st["sink"].reshape(1, K, 1, G, 1) - m)
    v = torch.where((key[None] < st["ends"].long()[:, None])[:, None, :, None], x[1], torch.zeros_like(x[1]))
    o = (p / total).reshape(B, K, T * G, -1) @ v
    return o.reshape(B, K, T, G, D).permute(0, 2, 1, 3, 4).reshape(B * T, H * D).to(st["dtype"])


def run(st):
    case = st["case"]
    if not own:
        return {"store": _plain_store, "read": _plain_read, "attention": _plain_attention}[case["op"]](st)
    from xyntetik_runner_b200 import kernels
    K, D, P = case["kv_heads"], case["head_dim"], case["page_size"]
    if case["op"] == "attention":
        out = torch.empty_like(st["q"])
        kernels.attention_kv4(st["q"], out, st["cache"], 0, P, st["seg_start"], st["seg_len"], st["pos0"], st["table"], case["heads"], D, st["scale"],
                              (st["len_host"], st["pos0_host"]), window=case["window"], sink=st["sink"], softcap=case["softcap"],
                              keep_first=case["keep_first"], bias=st["bias"])
        return out
    if case["op"] == "store":
        kernels.kv4_store(st["k"], st["v"], st["positions"], st["tok_seg"], st["table"], st["cache"], 0, P)
    out = torch.empty((st["out_pages"], 2, K, P, D), dtype=st["dtype"], device=st["cache"].device)
    kernels.kv4_read(st["cache"], 0, P, st["table"], st["first"], st["ends"], out, keep_first=st["keep"])
    return out


# ---- in 64 bits --------------------------------------------------------------------------------------------------------


def _exact_rows(raw, which, P, hs, D):
    """Values [P, D] float64 of one page's block (bytes), from the definition: half-bytes one by one."""
    b = raw.to(torch.int64)
    codes = b[which * P * hs // 2:(which + 1) * P * hs // 2].reshape(P, hs // 8, 4)
    low, high = codes & 15, codes >> 4
    # byte 0: elements 0, 2; byte 1: 4, 6; byte 2: 1, 3; byte 3: 5, 7
    e = torch.stack([low[..., 0], low[..., 2], high[..., 0], high[..., 2], low[..., 1], low[..., 3], high[..., 1], high[..., 3]], dim=-1)
    sc = b[P * hs + which * P * hs // 16:P * hs + (which + 1) * P * hs // 16].reshape(P, hs // 32, 2)
    s = ((sc[..., 0] | (sc[..., 1] << 8)) << 16).to(torch.int32).view(torch.float32).double()
    return (e.reshape(P, hs).double() - 8.0)[:, :D] * s.repeat_interleave(32, dim=1)[:, :D]


def _exact_quantised(x):
    """The values that x [N, D] float64 is held as, by arithmetic on the numbers alone."""
    N, D = x.shape
    hs = _held(D)
    g = torch.cat([x, torch.zeros((N, hs - D), dtype=x.dtype, device=x.device)], dim=1).reshape(N, hs // 32, 32)
    top, bottom = g.max(-1).values, g.min(-1).values
    e = torch.where(top + bottom >= 0, top, bottom)
    m, ex = torch.frexp(e)
    s = -torch.ldexp(torch.round(m * 32.0), ex - 5) / 8.0
    none = torch.isnan(top) | (top >= 2.0 ** 120) | (bottom <= -2.0 ** 120)
    zero = e.abs() < 2.0 ** -96
    c = torch.round(g / torch.where(zero | none, torch.ones_like(s), s)[..., None]).clamp(-8.0, 7.0)
    v = torch.where(zero[..., None], torch.zeros_like(g), c * s[..., None])
    return torch.where(none[..., None], torch.full_like(g, math.nan), v).reshape(N, hs)[:, :D]


def exact(case, seed):
    st = prepare(case, seed)
    B, H, K, D, P, hs = case["requests"], case["heads"], case["kv_heads"], case["head_dim"], case["page_size"], _held(case["head_dim"])
    ends, table = st["ends"].tolist(), st["table"].cpu().numpy()
    if case["op"] == "store":
        out = torch.zeros((st["out_pages"], 2, K, P, D), dtype=torch.float64, device=DEVICE)
        T, n = case["tokens"], st["k"].shape[0]
        kv = [_exact_quantised(x.double().reshape(n * K, D)).reshape(n, K, D) for x in (st["k"], st["v"])]
        at = 0
        for b, end in enumerate(ends):
            f = end - T
            count = (end - 1) // P - f // P + 1
            for w in (0, 1):
                flat = torch.zeros((count * P, K, D), dtype=torch.float64, device=DEVICE)
                flat[f % P:f % P + T] = kv[w][b * T:(b + 1) * T]
                out[at:at + count, w] = flat.reshape(count, P, K, D).transpose(1, 2)
            at += count
        return out
    if case["op"] == "read":
        out = torch.zeros((st["out_pages"], 2, K, P, D), dtype=torch.float64, device=DEVICE)
        seg, page, first = st["out_seg"].tolist(), st["out_page"].tolist(), st["first"].tolist()
        if st["out_pages"] * K > 30000:
            return None
        for j in range(st["out_pages"]):
            lo, hi = page[j] * P, (page[j] + 1) * P
            for h in range(K):
                raw = st["cache"][int(table[seg[j], page[j]]), 0, h]
                for w in (0, 1):
                    out[j, w, h] = _exact_rows(raw, w, P, hs, D)
            for p in range(lo, hi):
                if p >= ends[seg[j]] or (p < first[seg[j]] and p >= st["keep"]):
                    out[j, :, :, p - lo] = 0.0
        return out
    T, G = case["tokens"], H // K
    out = torch.zeros((B, T, H, D), dtype=torch.float64, device=DEVICE)
    if sum(-(-e // P) for e in ends) * K > 30000:
        # (too many pages to walk one by one: the same arithmetic on a request's pages at once)
        def rows_of(b, h, w, count):
            raw = st["cache"][torch.from_numpy(table[b, :count].astype(np.int64)).to(DEVICE), 0, h]
            codes = raw[:, w * P * hs // 2:(w + 1) * P * hs // 2].reshape(-1)
            scales = raw[:, P * hs + w * P * hs // 16:P * hs + (w + 1) * P * hs // 16].reshape(-1)
            joined = torch.cat([codes, codes, scales, scales])
            return _exact_rows(joined, 0, P * count, hs, D)
    else:
        def rows_of(b, h, w, count):
            return torch.cat([_exact_rows(st["cache"][int(table[b, i]), 0, h], w, P, hs, D) for i in range(count)])
    q = st["q"].double().reshape(B, T, H, D)
    for b, end in enumerate(ends):
        count = -(-end // P)
        j = torch.arange(end, device=DEVICE)
        for h in range(K):
            k, v = (rows_of(b, h, w, count)[:end] for w in (0, 1))
            for t in range(0, T, 64):
                qq = q[b, t:t + 64, h * G:(h + 1) * G]                       # [t, G, D]
                pos = torch.arange(end - T + t, end - T + t + qq.shape[0], device=DEVICE)[:, None]
                ok = j[None] <= pos
                if case["window"]:
                    ok = ok & ((pos - j[None] < case["window"]) | (j[None] < case["keep_first"]))
                s = torch.einsum("tgd,jd->tgj", qq, k) * st["scale"]
                if st["bias"] is not None:
                    far = torch.minimum((pos - j[None]).clamp(min=0), torch.tensor(case["bias"] - 1, device=DEVICE))
                    s = s + st["bias"].double()[h * G:(h + 1) * G][:, far].transpose(0, 1) * st["scale"]
                if case["softcap"]:
                    s = torch.tanh(s / case["softcap"]) * case["softcap"]
                s = s.masked_fill(~ok[:, None], -math.inf)
                if st["sink"] is not None:
                    s = torch.cat([s, st["sink"].double()[None, h * G:(h + 1) * G, None].expand(s.shape[0], -1, -1)], dim=-1)
                a = torch.softmax(s, dim=-1)[..., :end]
                out[b, t:t + 64, h * G:(h + 1) * G] = torch.einsum("tgj,jd->tgd", a, v)
    return out.reshape(B * T, H * D)
