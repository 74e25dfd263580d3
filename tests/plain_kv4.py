"""A cache in four bits, plainly, in 64 bits on the CPU: how rows are held, their bytes, and attention over them."""
import math

import numpy as np
import torch


def held(D):
    return 64 if D <= 64 else 128 if D <= 128 else 256


def round5(e):
    m, x = math.frexp(e)
    return math.ldexp(float(np.round(m * 32.0)), x - 5)            # (numpy rounds ties to even)


def group(x):
    """(codes, scale) of a group of 32 numbers."""
    if not np.all(np.isfinite(x)) or np.max(np.abs(x)) >= 2.0 ** 120:
        return np.zeros(32, dtype=np.int64), math.nan
    hi, lo = float(np.max(x)), float(np.min(x))
    e = hi if hi >= -lo else lo
    if abs(e) < 2.0 ** -96:
        return np.zeros(32, dtype=np.int64), 0.0
    s = -round5(e) / 8.0
    return np.clip(np.round(x / s), -8, 7).astype(np.int64), s


def quantised(rows):
    """rows [N, D] (any float tensor) -> (codes [N, hs], scales [N, hs / 32], values [N, D] float64)."""
    x = rows.detach().cpu().to(torch.float64).numpy()
    N, D = x.shape
    hs = held(D)
    g = np.zeros((N, hs))
    g[:, :D] = x
    codes, scales = np.zeros((N, hs), dtype=np.int64), np.zeros((N, hs // 32))
    for n in range(N):
        for i in range(hs // 32):
            codes[n, 32 * i:32 * i + 32], scales[n, i] = group(g[n, 32 * i:32 * i + 32])
    values = codes * np.repeat(scales, 32, axis=1)
    return codes, scales, torch.from_numpy(values[:, :D])


def scale_bytes(s):
    w = torch.tensor([s], dtype=torch.float64).to(torch.bfloat16)
    assert math.isnan(s) or float(w) == s                           # a scale is a bfloat16
    return w.view(torch.uint8).numpy()


def put(block, page_size, tok, plane, codes, scales):
    """Write one token's head into the bytes of a page, layer and kv head (numpy uint8)."""
    hs = len(codes)
    for w in range(hs // 8):
        word = 0
        for i in range(4):
            word |= int(codes[8 * w + 2 * i] + 8) << (4 * i)
            word |= int(codes[8 * w + 2 * i + 1] + 8) << (16 + 4 * i)
        at = plane * page_size * hs // 2 + tok * hs // 2 + 4 * w
        block[at:at + 4] = np.frombuffer(int(word).to_bytes(4, "little"), dtype=np.uint8)
    for i, s in enumerate(scales):
        at = page_size * hs + plane * page_size * hs // 16 + (tok * (hs // 32) + i) * 2
        block[at:at + 2] = scale_bytes(float(s))


def attention(q, k, v, pos0, scale, window=0, keep=0, sink=None, softcap=0.0, bias=None):
    """q [L, H, D], k and v [T, K, D] float64 values of positions 0 .. T - 1; query i is at pos0 + i.  Returns (out [L, H, D], what the sums are made
    of: sum a |v|, and the largest sum of |q k| scale over the keys seen, per query and head)."""
    L, H, D = q.shape
    K, G = k.shape[1], H // k.shape[1]
    out, size, raw = torch.zeros(L, H, D, dtype=torch.float64), torch.zeros(L, H, D, dtype=torch.float64), torch.zeros(L, H, dtype=torch.float64)
    for i in range(L):
        p = pos0 + i
        keys = [j for j in range(p + 1) if not window or p - j < window or j < keep]
        for h in range(H):
            kk, vv = k[keys, h // G], v[keys, h // G]
            s = (kk @ q[i, h]) * scale
            raw[i, h] = (kk.abs() @ q[i, h].abs()).max() * scale
            if bias is not None:
                s = s + torch.tensor([bias[h, min(p - j, bias.shape[1] - 1)] for j in keys], dtype=torch.float64) * scale
                raw[i, h] += float(bias[h].abs().max()) * scale
            if softcap:
                s = softcap * torch.tanh(s / softcap)
            m = s.max() if sink is None else torch.maximum(s.max(), sink[h])
            e = torch.exp(s - m)
            total = e.sum() + (0.0 if sink is None else torch.exp(sink[h] - m))
            a = e / total
            out[i, h] = a @ vv
            size[i, h] = a @ vv.abs()
    return out, size, raw


def tolerance(out, size, raw, D, dtype):
    """How far a kernel may be off.  Scores: sums of `hs` exact products in float32 (a product and 8 roundings to spare), and an exponent's argument and
    exponential rounded a few times: each weight is off by 4 d relatively (twice in the weight, twice in the sum).  bfloat16: weights rounded once
    (2^-8), outputs once (2^-8)."""
    hs = held(D)
    d = raw * ((hs + 8) * 2.0 ** -23) + raw * 2.0 ** -21 + 2.0 ** -20
    half = 2.0 ** -8 if dtype == torch.bfloat16 else 2.0 ** -23
    return (4 * d[..., None] + half) * size + half * out.abs() + 1e-30


def quantised_rows(x):
    """The values that rows x [..., D] are held as, all at once (float64, on x's device)."""
    D = x.shape[-1]
    g = torch.nn.functional.pad(x.double(), (0, held(D) - D)).reshape(*x.shape[:-1], -1, 32)
    hi, lo = g.amax(-1), g.amin(-1)
    e = torch.where(hi >= -lo, hi, lo)
    m, ex = torch.frexp(e)
    s = -torch.ldexp(torch.round(m * 32.0), ex - 5) / 8.0
    s = torch.where(e.abs() < 2.0 ** -96, torch.zeros_like(s), s)
    c = torch.round(g / torch.where(s == 0, torch.ones_like(s), s)[..., None]).clamp(-8, 7) * (s != 0)[..., None]
    return (c * s[..., None]).reshape(*x.shape[:-1], -1)[..., :D]
