"""The cache in four bits on the device: store, read and attention against the plain form in 64 bits (plain_kv4.py)."""
import math

import numpy as np
import pytest
import torch

import plain_kv4

pytestmark = pytest.mark.gpu
DEV = "cuda:0"
F32, BF16 = torch.float32, torch.bfloat16


def i32(a):
    return torch.tensor(np.asarray(a), dtype=torch.int32, device=DEV)


def tables(lens, P, g, spare=2):
    """Block tables of requests with these lengths, pages in a random order, and how many pages there are."""
    need = [-(-n // P) for n in lens]
    order = torch.randperm(sum(need) + spare, generator=g).tolist()
    bt = np.full((len(lens), max(max(need), 1) + 1), -1, dtype=np.int32)
    for r, n in enumerate(need):
        bt[r, :n] = [order.pop() for _ in range(n)]
    return bt, sum(need) + spare


def same(a, b):
    a, b = a.double().cpu(), b.double().cpu()
    return torch.equal(torch.isnan(a), torch.isnan(b)) and torch.equal(torch.nan_to_num(a), torch.nan_to_num(b))


STORE = [  # lens held ahead, tokens, K, D, Vd, page, dtype, extra columns of a row
    ([0], 1, 1, 64, 64, 8, BF16, 0), ([5, 0, 63], 9, 2, 128, 128, 16, BF16, 64), ([7], 40, 3, 100, 100, 24, F32, 3), ([30, 1], 5, 1, 16, 16, 64, BF16, 1),
    ([0, 17], 33, 2, 256, 256, 8, F32, 0), ([2], 7, 2, 80, 48, 32, BF16, 8), ([2], 7, 2, 33, 65, 32, F32, 0), ([11], 3, 40, 192, 192, 40, BF16, 0),
    ([0], 20, 1, 1, 1, 16, F32, 5)]


@pytest.mark.parametrize("held,T,K,D,Vd,P,dtype,extra", STORE)
def test_store_and_read(held, T, K, D, Vd, P, dtype, extra):
    """Bytes as the plain form writes them, nothing else touched; values read back are what the bytes stand for, exactly."""
    from xyntetik_runner_b200 import kernels
    g = torch.Generator().manual_seed(D * 100 + P + T)
    lens = [h + T for h in held]
    bt, n_pages = tables(lens, P, g)
    hs, B = plain_kv4.held(max(D, Vd)), len(held)
    cache = torch.randint(0, 256, (n_pages, 2, K, kernels.kv4_block_bytes(max(D, Vd), P)), generator=g, dtype=torch.uint8)
    n = B * T
    row = torch.randn(n, K * (D + Vd) + extra, generator=g) * torch.exp(torch.randn(n, 1, generator=g) * 3)
    row[0, :min(D, 32)] = 0.0                                        # a group of zeros
    row[-1, K * D:K * D + min(Vd, 32)] *= 1e-35                      # below what is held
    row = row.to(dtype)
    pos = np.concatenate([h + np.arange(T) for h in held])
    seg = np.repeat(np.arange(B), T)
    want = cache.numpy().copy()
    values = []
    for plane, (at, E) in enumerate(((0, D), (K * D, Vd))):
        full = torch.zeros(n * K, max(D, Vd), dtype=torch.float64)
        full[:, :E] = row[:, at:at + K * E].double().reshape(n * K, E)
        codes, scales, v = plain_kv4.quantised(full)
        values.append(v.reshape(n, K, -1))
        for t in range(n):
            for h in range(K):
                plain_kv4.put(want[bt[seg[t], pos[t] // P], 1, h], P, pos[t] % P, plane, codes[t * K + h], scales[t * K + h])
    dev, rows = cache.to(DEV), row.to(DEV)
    kernels.kv4_store(rows[:, :K * D], rows[:, K * D:K * (D + Vd)], i32(pos), i32(seg), i32(bt), dev, 1, P)
    assert torch.equal(dev.cpu(), torch.from_numpy(want))
    for out_dtype in (BF16, F32):
        first, end = i32(held), i32(lens)
        pages = sum((e - 1) // P - f // P + 1 for f, e in zip(held, lens))
        out = torch.full((pages + 1, 2, K, P, max(D, Vd)), 7.0, dtype=out_dtype, device=DEV)
        where = i32(np.full_like(bt, -9))
        kernels.kv4_read(dev, 1, P, i32(bt), first, end, out, tables=where)
        exp = torch.zeros(pages + 1, 2, K, P, max(D, Vd), dtype=torch.float64)
        exp[-1] = 7.0                                                # a page behind the last is left as it was
        j = 0
        exp_where = np.full_like(bt, -9)
        for r in range(B):
            for pi in range(held[r] // P, (lens[r] - 1) // P + 1):
                for p in range(max(pi * P, held[r]), min((pi + 1) * P, lens[r])):
                    for plane in (0, 1):
                        exp[j, plane, :, p - pi * P] = values[plane][r * T + p - held[r]]
                exp_where[r, pi] = j
                j += 1
        assert torch.equal(out.double().cpu(), exp) and torch.equal(where.cpu(), torch.from_numpy(exp_where))


def test_read_with_kept_rows():
    """Kept first rows ahead of a window's, requests that have none, rows that both name, pages that were given back."""
    from xyntetik_runner_b200 import kernels
    g = torch.Generator().manual_seed(8)
    P, K, D, lens, first, keep = 8, 2, 48, [100, 20, 9], [61, 15, 9], 11
    bt, n_pages = tables(lens, P, g)
    k, v = (torch.randn(sum(lens), K * D, generator=g).to(BF16) for _ in (0, 1))
    pos, seg = np.concatenate([np.arange(n) for n in lens]), np.repeat(np.arange(3), lens)
    cache = kernels.kv4_cache(n_pages, 1, K, D, P, DEV)
    kernels.kv4_store(k.to(DEV), v.to(DEV), i32(pos), i32(seg), i32(bt), cache, 0, P)
    bt[0, 2:7] = -1
    held = torch.stack([plain_kv4.quantised(x.reshape(-1, D))[2].reshape(-1, K, D) for x in (k, v)])
    want, pages = [], {0: [0, 1, 7, 8, 9, 10, 11, 12], 1: [0, 1, 2], 2: []}
    for r in range(3):
        for pi in pages[r]:
            page = torch.zeros(2, K, P, D, dtype=torch.float64)
            for t in range(P):
                p = pi * P + t
                if p < lens[r] and (p < keep or p >= first[r]) and bt[r, pi] >= 0:
                    page[:, :, t] = held[:, int(np.flatnonzero((seg == r) & (pos == p))[0])]
            want.append(page)
    out = torch.full((len(want) + 1, 2, K, P, D), 3.0, dtype=BF16, device=DEV)
    kernels.kv4_read(cache, 0, P, i32(bt), i32(first), i32(lens), out, keep_first=keep)
    assert torch.equal(out[:-1].double().cpu(), torch.stack(want)) and torch.all(out[-1] == 3.0)


@pytest.mark.parametrize("bad", [math.nan, math.inf, -math.inf, 2.0 ** 120, -2.0 ** 121, 2.0 ** 119, -2.0 ** -96, 2.0 ** -97, 0.0])
@pytest.mark.parametrize("dtype", [BF16, F32])
def test_borders_of_what_is_held(bad, dtype):
    """One element of a group out of the common: the group as the plain form has it, its neighbours as ever."""
    from xyntetik_runner_b200 import kernels
    g = torch.Generator().manual_seed(5)
    k = torch.randn(2, 128, generator=g)
    k[0, 32:64] *= 2.0 ** -100 if abs(bad) < 1e-20 else 1.0
    k[0, 40] = bad
    k, v = k.to(dtype), torch.randn(2, 128, generator=g).to(dtype)
    cache = kernels.kv4_cache(1, 1, 1, 128, 8, DEV)
    bt = i32([[0]])
    kernels.kv4_store(k.to(DEV), v.to(DEV), i32([0, 1]), i32([0, 0]), bt, cache, 0, 8)
    out = torch.empty(1, 2, 1, 8, 128, dtype=F32, device=DEV)
    kernels.kv4_read(cache, 0, 8, bt, i32([0]), i32([2]), out)
    assert same(out[0, 0, 0, :2], plain_kv4.quantised(k)[2]) and same(out[0, 1, 0, :2], plain_kv4.quantised(v)[2])


def test_halves_between_two_codes_go_to_even():
    """x / s of exactly n + 1/2, for every scale of five bits."""
    from xyntetik_runner_b200 import kernels
    rows = []
    for m in range(16, 32):
        s = m / 16.0
        half = [(c + 0.5) * s for c in range(-8, 7)] + [c * s for c in range(-7, 8)]
        rows.append([8.0 * s] + half + [0.0])
    k = torch.tensor(rows, dtype=torch.float32)
    k = torch.cat([k, -k], dim=0)
    n = k.shape[0]
    for dtype in (F32, BF16):
        x = k.to(dtype)
        cache = kernels.kv4_cache(4, 1, 1, 32, 8, DEV)
        bt = i32([[2, 0, 3, 1]])
        kernels.kv4_store(x.to(DEV), x.to(DEV), i32(np.arange(n)), i32(np.zeros(n)), bt, cache, 0, 8)
        out = torch.empty(4, 2, 1, 8, 32, dtype=F32, device=DEV)
        kernels.kv4_read(cache, 0, 8, bt, i32([0]), i32([n]), out)
        want = plain_kv4.quantised(x)[2]
        for plane in (0, 1):
            assert torch.equal(out[:, plane, 0].reshape(n, 32).double().cpu(), want)


def test_pages_that_are_not_held():
    """Tokens whose page is not held, or is not one of the cache's, are not written; rows on such pages are read as zeros; other requests are as ever."""
    from xyntetik_runner_b200 import kernels
    g = torch.Generator().manual_seed(6)
    P, K, D = 8, 2, 64
    bt = np.array([[3, -1, 1, 9], [0, 2, -5, 1 << 30]], dtype=np.int32)          # a cache of five pages
    pos, seg = np.array([3, 9, 17, 25, 40, -1, 1, 12, 18, 26, 5]), np.array([0, 0, 0, 0, 0, 0, 1, 1, 1, 1, 2])
    n = len(pos)
    k = torch.randn(n, K * D, generator=g).to(BF16)
    cache = kernels.kv4_cache(5, 1, K, D, P, DEV)
    kernels.kv4_store(k.to(DEV), k.to(DEV), i32(pos), i32(seg), i32(bt), cache, 0, P)
    want = np.zeros((5, 1, K, cache.shape[3]), dtype=np.uint8)
    codes, scales, values = plain_kv4.quantised(k.reshape(n * K, D))
    kept = [0, 2, 6, 7]
    for t in kept:
        for plane in (0, 1):
            for h in range(K):
                plain_kv4.put(want[bt[seg[t], pos[t] // P], 0, h], P, pos[t] % P, plane, codes[t * K + h], scales[t * K + h])
    assert torch.equal(cache.cpu(), torch.from_numpy(want))
    out = torch.full((8, 2, K, P, D), 5.0, dtype=BF16, device=DEV)
    kernels.kv4_read(cache, 0, P, i32(bt), i32([0, 0]), i32([100, 32]), out)
    exp = torch.zeros(8, 2, K, P, D, dtype=torch.float64)
    for t in kept:
        exp[4 * seg[t] + pos[t] // P, :, :, pos[t] % P] = values.reshape(n, K, D)[t]
    got = out.double().cpu()
    for t in kept:
        assert torch.equal(got[4 * seg[t] + pos[t] // P, :, :, pos[t] % P], exp[4 * seg[t] + pos[t] // P, :, :, pos[t] % P])
    for page in (1, 3, 6, 7):
        assert not got[page].any()


ATT = [  # contexts, tokens, H, K, D, page, dtype, window, keep, sink, cap, bias
    ([1], 1, 1, 1, 64, 8, BF16, 0, 0, 0, 0, 0), ([1, 2, 33], 1, 4, 2, 128, 64, BF16, 0, 0, 0, 0, 0), ([64, 65, 129, 300], 1, 8, 2, 64, 64, BF16, 0, 0, 0, 0, 0),
    ([700], 1, 8, 1, 128, 16, BF16, 0, 0, 1, 0, 0), ([333, 40], 1, 4, 4, 256, 24, BF16, 0, 0, 0, 0, 0), ([100, 31], 1, 5, 1, 100, 40, BF16, 0, 0, 0, 0, 0),
    ([90], 3, 6, 2, 80, 32, BF16, 0, 0, 0, 0, 0), ([200, 17], 4, 16, 4, 128, 64, BF16, 0, 0, 1, 0, 0), ([150, 6], 6, 14, 2, 64, 8, BF16, 0, 0, 0, 20.0, 0),
    ([500, 260], 1, 8, 2, 128, 64, BF16, 100, 0, 0, 0, 0), ([500, 60], 1, 8, 2, 128, 16, BF16, 33, 5, 1, 0, 40), ([400], 5, 4, 1, 64, 16, BF16, 64, 70, 0, 0, 200),
    ([300], 1, 71, 1, 64, 64, BF16, 0, 0, 0, 0, 0), ([200], 3, 130, 2, 64, 64, BF16, 0, 0, 0, 0, 0), ([40], 40, 24, 1, 64, 16, F32, 0, 0, 0, 0, 0), ([120], 2, 20, 1, 192, 64, BF16, 50, 3, 1, 0, 0), ([77], 1, 3, 3, 16, 8, BF16, 0, 0, 0, 0, 0),
    ([1, 90], 1, 4, 2, 64, 64, F32, 0, 0, 0, 0, 0), ([333], 1, 8, 2, 128, 64, F32, 0, 0, 1, 30.0, 0), ([130, 20], 7, 6, 3, 100, 24, F32, 40, 9, 0, 0, 30),
    ([60], 60, 4, 2, 128, 16, F32, 0, 0, 0, 0, 0), ([80], 3, 2, 1, 256, 64, F32, 0, 0, 0, 0, 0),
    # portions that are read back for the prompt kernels, beside short ones (enough row blocks for that; then fewer)
    ([90, 30], [70, 5], 128, 16, 128, 64, BF16, 0, 0, 0, 0, 0), ([150], 33, 264, 66, 64, 16, BF16, 40, 5, 1, 0, 0), ([100], 80, 117, 39, 48, 24, BF16, 30, 10, 0, 0, 0),
    ([200], 64, 82, 41, 64, 64, BF16, 0, 0, 0, 15.0, 0), ([90, 12, 110], [70, 1, 50], 64, 32, 128, 16, BF16, 60, 0, 1, 0, 70),
    ([90], 70, 8, 2, 128, 64, BF16, 0, 0, 0, 0, 0), ([150], 33, 4, 2, 64, 16, BF16, 40, 5, 1, 0, 0), ([100], 80, 3, 1, 48, 24, BF16, 30, 10, 0, 0, 0),
    ([70], 40, 3, 1, 100, 24, BF16, 0, 0, 0, 0, 0), ([120], 100, 2, 2, 256, 64, BF16, 0, 0, 0, 0, 0)]


def attention_case(contexts, T, H, K, D, P, dtype, window, keep, sink, cap, bias, seed=1, layers=2, layer=1):
    """(arguments of attention_kv4 but for q and out, q on the CPU, the held values of every request, plain options)"""
    from xyntetik_runner_b200 import kernels
    g = torch.Generator().manual_seed(seed * 1000 + D + P + sum(contexts))
    Ts = [T] * len(contexts) if isinstance(T, int) else T
    bt, n_pages = tables(contexts, P, g)
    cache = torch.randint(0, 256, (n_pages, layers, K, kernels.kv4_block_bytes(D, P)), generator=g, dtype=torch.uint8).to(DEV)   # garbage, NaN scales among it
    kv = [(torch.randn(c, K * D, generator=g) * 1.5).to(dtype) for c in contexts for _ in (0, 1)]
    pos = np.concatenate([np.arange(c) for c in contexts])
    seg = np.repeat(np.arange(len(contexts)), contexts)
    kernels.kv4_store(torch.cat(kv[0::2]).to(DEV), torch.cat(kv[1::2]).to(DEV), i32(pos), i32(seg), i32(bt), cache, layer, P)
    held = [plain_kv4.quantised(x.reshape(-1, D))[2].reshape(-1, K, D) for x in kv]
    n = sum(Ts)
    q = (torch.randn(n, H * D, generator=g) * 1.3).to(dtype)
    sinks = torch.randn(H, generator=g) if sink else None
    table = -torch.rand(H, bias, generator=g) * 30 if bias else None
    starts = np.concatenate([[0], np.cumsum(Ts)[:-1]])
    pos0 = np.array(contexts) - np.array(Ts)
    if window:
        # pages that no token of the portion sees any more are given back
        for r, p0 in enumerate(pos0):
            for pi in range(bt.shape[1]):
                last = (pi + 1) * P - 1
                if last < p0 - window + 1 and pi * P >= keep:
                    bt[r, pi] = -1
    args = dict(cache=cache, layer=layer, page_size=P, seg_start=i32(starts), seg_len=i32(Ts), seg_pos0=i32(pos0), block_tables=i32(bt), heads=H, head_dim=D,
                scale=D ** -0.5, lengths=(np.array(Ts, dtype=np.int32), pos0.astype(np.int32)), window=window, sink=None if sinks is None else sinks.to(DEV),
                softcap=cap, keep_first=keep, bias=None if table is None else table.to(DEV))
    plain = dict(scale=D ** -0.5, window=window, keep=keep, sink=None if sinks is None else sinks.double(), softcap=cap, bias=None if table is None else table.double())
    return args, q, held, plain, Ts, starts, pos0


def check(got, q, held, plain, Ts, starts, pos0, H, D, dtype):
    for r, T in enumerate(Ts):
        s = starts[r]
        if T == 0:
            continue
        o, size, raw = plain_kv4.attention(q[s:s + T].double().reshape(T, H, D), held[2 * r], held[2 * r + 1], int(pos0[r]), **plain)
        tol = plain_kv4.tolerance(o, size, raw, D, dtype)
        off = (got[s:s + T].double().cpu().reshape(T, H, D) - o).abs()
        assert torch.all(off <= tol), f"request {r}: {float((off / tol).max()):.3g} of the tolerance"


@pytest.mark.parametrize("contexts,T,H,K,D,P,dtype,window,keep,sink,cap,bias", ATT)
def test_attention(contexts, T, H, K, D, P, dtype, window, keep, sink, cap, bias):
    from xyntetik_runner_b200 import kernels
    args, q, held, plain, Ts, starts, pos0 = attention_case(contexts, T, H, K, D, P, dtype, window, keep, sink, cap, bias)
    wide = torch.zeros(q.shape[0], H * D + 24, dtype=dtype, device=DEV)          # q's rows lie in wider ones
    wide[:, :H * D] = q.to(DEV)
    if sum(T if isinstance(T, list) else [T]) * H > 5000 and dtype is BF16:      # (the cases that are there for the prompt kernels go through them)
        assert kernels.kv4_plan(args["lengths"], q.shape[0], K, H // K, D, P, kernels.BF16, window, keep, 64)[1] > 0
    for rows in (q.to(DEV), wide, wide[:, :H * D]):
        out = torch.full((q.shape[0] + 3, H * D), 9.0, dtype=dtype, device=DEV)
        kernels.attention_kv4(rows, out[:q.shape[0]], **args)
        kernels.tc_check_status(torch.device(DEV))
        check(out, q, held, plain, Ts, starts, pos0, H, D, dtype)
        assert torch.all(out[q.shape[0]:] == 9.0)


@pytest.mark.parametrize("contexts,T,H,K,D,P", [([415, 300], 1, 8, 4, 256, 8), ([20000, 9000], 2, 8, 4, 16, 24), ([4000], 5, 6, 2, 128, 64)])
def test_float32_is_as_exact_as_float32(contexts, T, H, K, D, P):
    """Off by no more than twice what the formula in float32 with sums that are rounded to nearest is: both round every product's sum and every weight
    once, the kernel's further roundings (of three pieces, of the spans' sums) are as many at most."""
    from xyntetik_runner_b200 import kernels
    args, q, held, plain, Ts, starts, pos0 = attention_case(contexts, T, H, K, D, P, F32, 0, 0, 0, 0, 0)
    out = torch.empty(q.shape[0], H * D, device=DEV)
    kernels.attention_kv4(q.to(DEV), out, **args)
    mine = theirs = 0.0
    for r, n in enumerate(Ts):
        s, k, v = starts[r], held[2 * r], held[2 * r + 1]
        x = q[s:s + n].reshape(n, H, D)
        o = plain_kv4.attention(x.double(), k, v, int(pos0[r]), **plain)[0]
        kk, vv = (y.float().repeat_interleave(H // K, 1) for y in (k, v))
        score = torch.einsum("nhd,khd->hnk", x, kk) * D ** -0.5
        score.masked_fill_(torch.arange(k.shape[0])[None, None, :] > int(pos0[r]) + torch.arange(n)[None, :, None], -math.inf)
        f = torch.einsum("hnk,khd->nhd", torch.softmax(score, -1), vv)
        mine += float((out[s:s + n].double().cpu().reshape(n, H, D) - o).square().sum())
        theirs += float((f.double() - o).square().sum())
    assert mine <= 4.0 * theirs, f"{math.sqrt(mine / theirs):.3g} times as far"


def run_case(case, **change):
    from xyntetik_runner_b200 import kernels
    args, q, held, plain, Ts, starts, pos0 = attention_case(*case)
    H, D, dtype = case[2], case[4], case[6]
    args.update(change)
    out = torch.full((q.shape[0], H * D), 9.0, dtype=dtype, device=DEV)
    kernels.attention_kv4(q.to(DEV), out, **args)
    kernels.tc_check_status(torch.device(DEV))
    return out, args, q, held, plain, Ts, starts, pos0


@pytest.mark.parametrize("case", [
    ([640], 1, 4, 1, 128, 64, BF16, 0, 0, 1, 0, 0), ([2500], 1, 4, 1, 128, 64, BF16, 0, 0, 1, 0, 0), ([9000, 300], 1, 2, 1, 64, 64, BF16, 0, 0, 0, 0, 0),
    ([20000], 1, 8, 1, 128, 64, BF16, 0, 0, 0, 0, 0), ([6000], 2, 2, 1, 256, 16, F32, 0, 0, 1, 0, 0), ([5000] * 2, 1, 16, 8, 64, 24, BF16, 3000, 40, 0, 0, 0),
    ([60] * 70, 1, 40, 40, 64, 16, BF16, 0, 0, 0, 0, 0)])
def test_requests_that_are_cut(case):
    """One block a request, spans that meet in a cluster, spans that a second kernel combines (test_kv4_cpu.py: which are which)."""
    out, args, q, held, plain, Ts, starts, pos0 = run_case(case)
    check(out, q, held, plain, Ts, starts, pos0, case[2], case[4], case[6])


@pytest.mark.parametrize("dtype", [BF16, F32])
@pytest.mark.parametrize("lowest", [-math.inf, torch.finfo(torch.float32).min])
@pytest.mark.parametrize("near", [0, 7])
def test_a_bias_that_hides_keys(dtype, lowest, near):
    """Distances of `near` and more have the lowest bias there is: such keys have no weight beside others; where all keys have it (near 0) and it is a number,
    scores are lost beside it and the row is the keys' average; the softmax of nothing but minus infinity is no number."""
    from xyntetik_runner_b200 import kernels
    H, K, D, P, n, T = 4, 2, 64, 16, 100, 3
    args, q, held, plain, Ts, starts, pos0 = attention_case([n], T, H, K, D, P, dtype, 0, 0, 0, 0, 20)
    table = plain["bias"].float()
    table[:, near:] = lowest
    args["bias"] = table.to(DEV)
    out = torch.full((T, H * D), 9.0, dtype=dtype, device=DEV)
    kernels.attention_kv4(q.to(DEV), out, **args)
    if near == 0:
        # equal weights; sums of 100 values in float32, the output's rounding
        tol = (2.0 ** -7 if dtype is BF16 else 2.0 ** -18) * float(held[1].abs().max())
        for i in range(T):
            want = held[1][:n - T + 1 + i].mean(0).repeat_interleave(H // K, 0)
            got = out[i].double().cpu().reshape(H, D)
            assert torch.isnan(got).all() if lowest == -math.inf else torch.all((got - want).abs() <= tol)
        return
    # (what is seen is a window of seven)
    check(out, q, held, {**plain, "window": near, "bias": table.clamp(min=-100.0).double()}, Ts, starts, pos0, H, D, dtype)


@pytest.mark.parametrize("dtype", [BF16, F32])
@pytest.mark.parametrize("bad", [math.nan, math.inf, -math.inf])
@pytest.mark.parametrize("cap,bias", [(0, 0), (20.0, 0), (0, 30)])
def test_queries_that_are_no_numbers(dtype, bad, cap, bias):
    """One element of one head's query: that head of that token is no number (some key is zero there), all others are as ever."""
    from xyntetik_runner_b200 import kernels
    H, K, D, P, T = 6, 2, 64, 16, 3
    args, q, held, plain, Ts, starts, pos0 = attention_case([90], T, H, K, D, P, dtype, 0, 0, 0, cap, bias)
    assert (held[0][:88, 1, 9] == 0).any()
    q[1, 4 * D + 9] = bad
    out = torch.full((T, H * D), 9.0, dtype=dtype, device=DEV)
    kernels.attention_kv4(q.to(DEV), out, **args)
    got = out.double().cpu().reshape(T, H, D)
    assert torch.isnan(got[1, 4]).all()
    q[1, 4 * D + 9] = 0.0
    o, size, raw = plain_kv4.attention(q.double().reshape(T, H, D), held[0], held[1], int(pos0[0]), **plain)
    near = (got - o).abs() <= plain_kv4.tolerance(o, size, raw, D, dtype)
    near[1, 4] = True
    assert near.all()


def test_empty_portions():
    """Portions of no tokens beside others, and a call without any token."""
    from xyntetik_runner_b200 import kernels
    case = ([50, 7, 90], [1, 0, 3], 4, 2, 64, 16, BF16, 0, 0, 0, 0, 0)
    out, args, q, held, plain, Ts, starts, pos0 = run_case(case)
    check(out, q, held, plain, Ts, starts, pos0, 4, 64, BF16)
    none = np.zeros(3, dtype=np.int32)
    args.update(seg_len=i32(none), lengths=(none, args["lengths"][1]))
    kernels.attention_kv4(q[:0].to(DEV), out[:0], **args)


def test_captured_and_replayed():
    """A captured call serves other positions, longer and shorter than those it was captured with; two graphs side by side in one stream."""
    from xyntetik_runner_b200 import kernels
    case = ([300, 40], 1, 8, 2, 128, 64, BF16, 0, 0, 0, 0, 0)
    args, q, held, plain, Ts, starts, pos0 = attention_case(*case)
    qd, graphs, outs = q.to(DEV), [], []
    pos = args["seg_pos0"]
    for ends in ([300, 40], [20, 10]):                               # captured as if the requests were this long
        at = np.array([e - 1 for e in ends], dtype=np.int32)
        pos.copy_(i32(at))
        out = torch.zeros(2, 8 * 128, dtype=BF16, device=DEV)
        call = lambda: kernels.attention_kv4(qd, out, **{**args, "lengths": (args["lengths"][0], at), "max_kv_len": 320})
        side = torch.cuda.Stream()
        side.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(side):
            call()
        torch.cuda.current_stream().wait_stream(side)
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            call()
        graphs.append(g)
        outs.append(out)
    for ends in ([300, 40], [20, 10], [129, 1], [65, 33]):
        at = np.array([e - 1 for e in ends])
        pos.copy_(i32(at))
        for g, out in zip(graphs, outs):
            out.zero_()
            g.replay()
        for out in outs:
            check(out, q, held, plain, Ts, starts, at, 8, 128, BF16)


@pytest.mark.parametrize("window,keep", [(0, 0), (70, 20)])
@pytest.mark.parametrize("said", [0, 450])
def test_prompt_portions_captured_and_replayed(said, window, keep):
    """Portions that are read back, captured near the start of their requests and replayed further on, where the rows they see take more pages."""
    from xyntetik_runner_b200 import kernels
    H, K, D, P = 64, 8, 64, 16
    args, q, held, plain, Ts, starts, pos0 = attention_case([450, 300], [100, 50], H, K, D, P, BF16, 0, 0, 0, 0, 0)
    args.update(window=window, keep_first=keep)
    plain.update(window=window, keep=keep)
    qd, pos, at = q.to(DEV), args["seg_pos0"], np.array([20, 0], dtype=np.int32)
    assert kernels.kv4_plan((args["lengths"][0], at), 150, K, H // K, D, P, kernels.BF16, window, keep, 64)[1] == 2
    out = torch.zeros(150, H * D, dtype=BF16, device=DEV)
    call = lambda: kernels.attention_kv4(qd, out, **{**args, "lengths": (args["lengths"][0], at), "max_kv_len": said})
    pos.copy_(i32(at))
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        call()
    torch.cuda.current_stream().wait_stream(side)
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        call()
    for where in ([20, 0], [350, 250], [0, 123], [337, 17]):
        pos.copy_(i32(where))
        out.zero_()
        g.replay()
        kernels.tc_check_status(torch.device(DEV))
        check(out, q, held, plain, Ts, starts, where, H, D, BF16)


def test_store_read_and_attend_on_another_stream():
    """The three together, as a step uses them, on a stream of their own and twice over."""
    from xyntetik_runner_b200 import kernels
    g = torch.Generator().manual_seed(9)
    P, K, H, D, lens = 16, 2, 4, 64, [33, 70]
    bt, n_pages = tables(lens, P, g)
    rows = [torch.randn(sum(lens), K * D, generator=g).to(BF16) for _ in (0, 1)]
    q = torch.randn(2, H * D, generator=g).to(BF16)
    pos, seg = np.concatenate([np.arange(n) for n in lens]), np.repeat(np.arange(2), lens)
    side = torch.cuda.Stream()
    dev = [x.to(DEV) for x in (*rows, q)]
    ints = [i32(x) for x in (pos, seg, bt, [0, 1], [1, 1], [n - 1 for n in lens], [0, 0], lens)]
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        for _ in range(2):
            cache = kernels.kv4_cache(n_pages, 1, K, D, P, DEV)
            kernels.kv4_store(dev[0], dev[1], ints[0], ints[1], ints[2], cache, 0, P)
            out, back = torch.empty_like(dev[2]), torch.empty(3 + 5, 2, K, P, D, dtype=BF16, device=DEV)
            kernels.attention_kv4(dev[2], out, cache, 0, P, ints[3], ints[4], ints[5], ints[2], H, D, D ** -0.5,
                                  (np.ones(2, dtype=np.int32), np.array(lens, dtype=np.int32) - 1))
            kernels.kv4_read(cache, 0, P, ints[2], ints[6], ints[7], back)
    torch.cuda.current_stream().wait_stream(side)
    held = []
    for r in range(2):
        for x in rows:
            held.append(plain_kv4.quantised(x[seg == r].reshape(-1, D))[2].reshape(-1, K, D))
    check(out, q, held, dict(scale=D ** -0.5), [1, 1], [0, 1], [n - 1 for n in lens], H, D, BF16)
    got = back.double().cpu()
    assert torch.equal(got[:3].permute(1, 0, 3, 2, 4).reshape(2, -1, K, D)[:, :33], torch.stack(held[:2]))
    assert torch.equal(got[3:].permute(1, 0, 3, 2, 4).reshape(2, -1, K, D)[:, :70], torch.stack(held[2:]))


def check_nan(got, want, tol):
    got = got.double().cpu()
    assert torch.equal(torch.isnan(got), torch.isnan(want))
    fine = ~torch.isnan(want)
    assert torch.all((got - want).abs()[fine] <= tol[fine])


@pytest.mark.parametrize("dtype", [BF16, F32])
@pytest.mark.parametrize("what,at", [("k", 20), ("v", 20), ("v", 37), ("k", 37), ("v", 38), ("v", 3), ("k", 3)])
def test_rows_that_are_no_numbers(what, at, dtype):
    """A NaN among a request's rows: in a portion of four tokens at 36 .. 39 with a window of 30, whoever does not see the row is as ever, a key's NaN
    reaches whoever sees it, a value's its group of 32 elements."""
    from xyntetik_runner_b200 import kernels
    g = torch.Generator().manual_seed(at)
    P, K, H, D, n, T = 8, 1, 2, 64, 40, 4
    k, v = (torch.randn(n, D, generator=g).to(dtype) for _ in (0, 1))
    (k if what == "k" else v)[at, 5] = math.nan
    bt, n_pages = tables([n], P, g)
    cache = kernels.kv4_cache(n_pages, 1, K, D, P, DEV)
    kernels.kv4_store(k.to(DEV), v.to(DEV), i32(np.arange(n)), i32(np.zeros(n)), i32(bt), cache, 0, P)
    q = torch.randn(T, H * D, generator=g).to(dtype)
    out = torch.empty(T, H * D, dtype=dtype, device=DEV)
    one = np.array([T], dtype=np.int32), np.array([n - T], dtype=np.int32)
    kernels.attention_kv4(q.to(DEV), out, cache, 0, P, i32([0]), i32([T]), i32([n - T]), i32(bt), H, D, 0.125, one, window=30)
    held = [plain_kv4.quantised(x)[2].reshape(n, 1, D) for x in (k, v)]
    want, size, raw = plain_kv4.attention(q.double().reshape(T, H, D), held[0], held[1], n - T, 0.125, window=30)
    tol = plain_kv4.tolerance(want, size, raw, D, dtype)
    check_nan(out.reshape(T, H, D), want, tol)
    assert torch.isnan(want).any() == (at > n - T - 30)


@pytest.mark.parametrize("dtype", [BF16, F32])
def test_values_of_many_sizes(dtype):
    """Values that grow and shrink by powers of ten along a request, zeros first; queries of tiny and huge size, zeros, infinities and NaN among them."""
    from xyntetik_runner_b200 import kernels
    g = torch.Generator().manual_seed(4)
    P, K, D, n = 16, 1, 128, 400
    v = torch.randn(n, D, generator=g) * torch.pow(10.0, torch.linspace(-9, 9, n))[:, None]
    v[:130] = 0.0
    k = torch.randn(n, D, generator=g)
    k, v = k.to(dtype), v.to(dtype)
    q = torch.randn(8, D, generator=g)
    q[1] *= 1e-30
    q[2] = 0.0
    q[3] *= 30.0
    q[4, :100] *= 1e-6
    q[5, 7] = math.nan
    q[6, 9] = math.inf
    q = q.to(dtype).reshape(1, 8 * D)
    bt, n_pages = tables([n], P, g)
    cache = kernels.kv4_cache(n_pages, 1, K, D, P, DEV)
    kernels.kv4_store(k.to(DEV), v.to(DEV), i32(np.arange(n)), i32(np.zeros(n)), i32(bt), cache, 0, P)
    out = torch.empty(1, 8 * D, dtype=dtype, device=DEV)
    kernels.attention_kv4(q.to(DEV), out, cache, 0, P, i32([0]), i32([1]), i32([n - 1]), i32(bt), 8, D, 0.09, (np.array([1], dtype=np.int32), np.array([n - 1], dtype=np.int32)))
    held = [plain_kv4.quantised(x)[2].reshape(n, 1, D) for x in (k, v)]
    qq = q.double().reshape(1, 8, D)
    want, size, raw = plain_kv4.attention(qq, held[0], held[1], n - 1, 0.09)
    tol = plain_kv4.tolerance(want, size, raw, D, dtype)
    got = out.double().cpu().reshape(1, 8, D)
    assert torch.isnan(got[0, 5:7]).all()                           # (a score of an infinity, or of no number)
    fine = [0, 1, 2, 3, 4, 7]
    assert torch.all((got - want).abs()[0, fine] <= tol[0, fine]), ((got - want).abs() / tol)[0, fine].max()


def test_pages_beyond_four_gigabytes():
    """A cache whose pages lie further apart than 32 bits of bytes."""
    from xyntetik_runner_b200 import kernels
    K, D, P, n = 8, 128, 64, 150
    per = K * kernels.kv4_block_bytes(D, P)
    pages = (1 << 32) // per + 40
    g = torch.Generator().manual_seed(2)
    cache = torch.empty((pages, 1, K, kernels.kv4_block_bytes(D, P)), dtype=torch.uint8, device=DEV)
    bt = i32([[pages - 1, 3, pages - 7, -1]])
    k, v = (torch.randn(n, K * D, generator=g).to(BF16) for _ in (0, 1))
    kernels.kv4_store(k.to(DEV), v.to(DEV), i32(np.arange(n)), i32(np.zeros(n)), bt, cache, 0, P)
    q = torch.randn(1, K * D, generator=g).to(BF16)
    out, back = torch.empty(1, K * D, dtype=BF16, device=DEV), torch.empty(3, 2, K, P, D, dtype=BF16, device=DEV)
    kernels.attention_kv4(q.to(DEV), out, cache, 0, P, i32([0]), i32([1]), i32([n - 1]), bt, K, D, 0.09, (np.array([1], dtype=np.int32), np.array([n - 1], dtype=np.int32)))
    kernels.kv4_read(cache, 0, P, bt, i32([0]), i32([n]), back)
    held = [plain_kv4.quantised_rows(x.reshape(n, K, D)) for x in (k, v)]
    check(out, q, held, dict(scale=0.09), [1], [0], [n - 1], K, D, BF16)
    assert torch.equal(back.double().cpu().permute(1, 0, 3, 2, 4).reshape(2, -1, K, D)[:, :n], torch.stack(held))


def test_refused_by_the_launchers():
    """What the wrappers let through and the library does not take: a cache off its border, a scale that is not positive is the wrappers'."""
    from xyntetik_runner_b200 import kernels
    raw = torch.zeros(2 * 1 * 1 * kernels.kv4_block_bytes(64, 16) + 16, dtype=torch.uint8, device=DEV)
    off = raw[4:4 + 2 * kernels.kv4_block_bytes(64, 16)].view(2, 1, 1, -1)
    k = torch.zeros(1, 64, dtype=BF16, device=DEV)
    with pytest.raises(kernels.KernelError, match="refuses these sizes"):
        kernels.kv4_store(k, k, i32([0]), i32([0]), i32([[0]]), off, 0, 16)
    with pytest.raises(kernels.KernelError, match="refuses these sizes"):
        kernels.kv4_read(off, 0, 16, i32([[0]]), i32([0]), i32([1]), torch.zeros(1, 2, 1, 16, 64, device=DEV))
    with pytest.raises(kernels.KernelError, match="refuses these sizes"):
        kernels.attention_kv4(k, torch.zeros_like(k), off, 0, 16, i32([0]), i32([1]), i32([0]), i32([[0]]), 1, 64, 0.1,
                              (np.array([1], dtype=np.int32), np.array([0], dtype=np.int32)))
    with pytest.raises(kernels.KernelError, match="current CUDA device"):
        kernels.kv4_store(k.cpu(), k.cpu(), i32([0]), i32([0]), i32([[0]]), off, 0, 16)
