"""The cache in four bits where calls follow one another, share scratch, or leave the common sizes; against the plain form in 64 bits (plain_kv4.py)."""
import math

import numpy as np
import pytest
import torch

import plain_kv4
from test_kv4_gpu import BF16, DEV, F32, attention_case, check, i32

pytestmark = pytest.mark.gpu


def shared():
    """Scratch as an engine keeps it: one buffer a name and type, made anew when it is too small."""
    held = {}

    def buf(name, shape, dtype):
        n = math.prod(shape)
        if (name, dtype) not in held or held[name, dtype].numel() < n:
            held[name, dtype] = torch.empty(n, dtype=dtype, device=DEV)
        return held[name, dtype][:n].view(*shape)
    return buf


def check_many(got, q, held, Ts, starts, pos0, H, D, dtype):
    """``check`` without options, all tokens of a request at once."""
    for r, T in enumerate(Ts):
        if T == 0:
            continue
        x = q[starts[r]:starts[r] + T].double().reshape(T, H, D)
        k, v = (y.repeat_interleave(H // y.shape[1], 1) for y in held[2 * r:2 * r + 2])
        hidden = torch.arange(k.shape[0])[None, None, :] > (int(pos0[r]) + torch.arange(T))[:, None, None]
        a = torch.softmax(torch.einsum("nhd,khd->nhk", x, k).mul_(D ** -0.5).masked_fill_(hidden, -math.inf), -1)
        o, size = torch.einsum("nhk,khd->nhd", a, v), torch.einsum("nhk,khd->nhd", a, v.abs())
        raw = torch.einsum("nhd,khd->nhk", x.abs(), k.abs()).mul_(D ** -0.5).masked_fill_(hidden, 0.0).amax(-1)
        off, tol = (got[starts[r]:starts[r] + T].double().cpu().reshape(T, H, D) - o).abs(), plain_kv4.tolerance(o, size, raw, D, dtype)
        assert torch.all(off <= tol), f"request {r}: {float((off / tol).max()):.3g} of the tolerance"


@pytest.mark.parametrize("H,K,D,P,kernel", [(64, 8, 128, 64, "attention_tc"), (66, 33, 48, 24, "attention_mma")])
def test_prompt_portions_one_call_after_the_other(H, K, D, P, kernel, monkeypatch):
    """Calls with other lengths every time through one scratch, all queued behind a long call: each finds the lengths of its own portions, not those that the
    call ahead of it left in the scratch."""
    from xyntetik_runner_b200 import kernels
    used = []
    real = getattr(kernels, kernel)
    monkeypatch.setattr(kernels, kernel, lambda *a, **k: (used.append(1), real(*a, **k)))
    contexts = [400, 300, 500]
    first = attention_case(contexts, [100, 1, 150], H, K, D, P, BF16, 0, 0, 0, 0, 0)
    buf, calls = shared(), []
    for Ts in ([100, 1, 150], [1, 130, 60], [150, 90, 0], [40, 110, 100], [1, 1, 248], [248, 1, 1]):
        # the same requests and rows, other portions of them
        pos0 = np.array(contexts) - np.array(Ts)
        starts = np.concatenate([[0], np.cumsum(Ts)[:-1]])
        args = {**first[0], "seg_start": i32(starts), "seg_len": i32(Ts), "seg_pos0": i32(pos0), "lengths": (np.array(Ts, dtype=np.int32), pos0.astype(np.int32))}
        q = torch.randn(sum(Ts), H * D, generator=torch.Generator().manual_seed(Ts[0])).to(BF16)
        calls.append((args, q, q.to(DEV), torch.full((sum(Ts) + 9, H * D), 9.0, dtype=BF16, device=DEV), Ts, starts, pos0))
    long = attention_case([6000] * 4, 4, 32, 8, 128, 64, BF16, 0, 0, 0, 0, 0, seed=2)
    far, long_q = torch.empty(16, 32 * 128, dtype=BF16, device=DEV), long[1].to(DEV)
    torch.cuda.synchronize()
    for args, q, qd, out, *_ in calls:
        kernels.attention_kv4(long_q, far, **long[0])
        kernels.attention_kv4(qd, out[:-9], **args, buf=buf)
    kernels.tc_check_status(torch.device(DEV))
    assert len(used) == len(calls)
    for args, q, qd, out, Ts, starts, pos0 in calls:
        check_many(out[:-9], q, first[2], Ts, starts, pos0, H, D, BF16)
        assert torch.all(out[-9:] == 9.0)


@pytest.mark.parametrize("case,cut", [
    (([640], 1, 1, 1, 64, 64, BF16, 0, 0, 0, 0, 0), "cluster"), (([640, 500, 77], 1, 3, 3, 64, 16, F32, 0, 0, 1, 0, 0), "cluster"),
    (([1000] * 5, 1, 24, 8, 128, 64, BF16, 300, 9, 1, 0, 60), "cluster"), (([1200, 900], 3, 8, 2, 256, 64, BF16, 0, 0, 0, 20.0, 0), "spans"),
    (([700, 90], 2, 6, 2, 100, 24, F32, 0, 0, 0, 30.0, 0), "cluster"), (([9000, 300], 1, 2, 1, 64, 64, BF16, 0, 0, 0, 0, 0), "spans")])
def test_spans_that_meet(case, cut):
    """Rows of half a warp's quadruples, and counts that part a warp, ahead of the cluster's barriers: right, and the same bits every time."""
    from xyntetik_runner_b200 import kernels
    args, q, held, plain, Ts, starts, pos0 = attention_case(*case)
    H, K, D, P, dtype = case[2:7]
    said = dict(zip(kernels._PLAN, kernels.kv4_plan(args["lengths"], q.shape[0], K, H // K, D, P, kernels.dtype_code(dtype), case[7], case[8], 1 << 30)))
    assert said["splits"] > 1 and bool(said["clustered"]) == (cut == "cluster")
    qd = q.to(DEV)
    outs = [torch.full((q.shape[0], H * D), 9.0, dtype=dtype, device=DEV) for _ in range(40)]
    for out in outs:
        kernels.attention_kv4(qd, out, **args)
    check(outs[0], q, held, plain, Ts, starts, pos0, H, D, dtype)
    assert all(torch.equal(out, outs[0]) for out in outs)


@pytest.mark.parametrize("case,kernel", [(([100], 80, 117, 39, 48, 24, BF16, 0, 0, 0, 0, 0), "attention_mma"), (([120, 90], 40, 117, 39, 80, 24, BF16, 50, 9, 0, 0, 0), "attention_mma"),
                                         (([200], 64, 82, 41, 64, 64, BF16, 0, 0, 0, 0, 0), "attention_tc"), (([100, 80], 3, 4, 2, 64, 24, F32, 0, 0, 0, 0, 0), None)])
def test_positions_beyond_the_tables(case, kernel, monkeypatch):
    """Block tables that name fewer rows than a request has: the others count as zeros, whichever way the portion goes."""
    from xyntetik_runner_b200 import kernels
    used = []
    if kernel:
        real = getattr(kernels, kernel)
        monkeypatch.setattr(kernels, kernel, lambda *a, **k: (used.append(1), real(*a, **k)))
    args, q, held, plain, Ts, starts, pos0 = attention_case(*case)
    H, D, P, dtype = case[2], case[4], case[5], case[6]
    pages = min(case[0]) // P - 1                                     # (the last request's neighbour in the array would be the next row's first pages)
    args["block_tables"] = args["block_tables"][:, :pages].contiguous()
    for x in held:
        x[pages * P:] = 0.0
    out = torch.full((q.shape[0], H * D), 9.0, dtype=dtype, device=DEV)
    kernels.attention_kv4(q.to(DEV), out, **args)
    kernels.tc_check_status(torch.device(DEV))
    assert bool(used) == bool(kernel)
    check(out, q, held, plain, Ts, starts, pos0, H, D, dtype)


@pytest.mark.parametrize("case", [([200, 90], 1, 4, 2, 64, 16, BF16, 40, 0, 0, 0, 0), ([200], 3, 4, 2, 64, 16, F32, 40, 0, 0, 0, 0),
                                  ([150], 70, 64, 16, 64, 16, BF16, 40, 0, 0, 0, 0), ([150], 70, 66, 33, 48, 24, BF16, 40, 0, 0, 0, 0)])
@pytest.mark.parametrize("window,keep", [(40, 2 ** 31 - 1), (2 ** 31 - 1, 0), (2 ** 31 - 1, 2 ** 31 - 1)])
def test_the_longest_windows_and_kept_rows(case, window, keep):
    """Every row is seen."""
    from xyntetik_runner_b200 import kernels
    args, q, held, plain, Ts, starts, pos0 = attention_case(*case[:7], 0, 0, 0, 0, 0)
    out = torch.full((q.shape[0], case[2] * case[4]), 9.0, dtype=case[6], device=DEV)
    kernels.attention_kv4(q.to(DEV), out, **{**args, "window": window, "keep_first": keep})
    check(out, q, held, plain, Ts, starts, pos0, case[2], case[4], case[6])


def test_reading_from_before_the_first_row():
    """A first row below zero reads from row 0 on; as many kept rows as there are numbers are all rows."""
    from xyntetik_runner_b200 import kernels
    g = torch.Generator().manual_seed(7)
    P, K, D, n = 16, 2, 64, 60
    k, v = (torch.randn(n, K * D, generator=g).to(BF16) for _ in (0, 1))
    cache, bt = kernels.kv4_cache(4, 1, K, D, P, DEV), i32([[2, 0, 3, 1]])
    kernels.kv4_store(k.to(DEV), v.to(DEV), i32(np.arange(n)), i32(np.zeros(n)), bt, cache, 0, P)
    want = torch.stack([plain_kv4.quantised_rows(x.reshape(n, K, D)) for x in (k, v)])
    for first, keep in ((0, 0), (-1, 0), (-2 ** 31, 0), (59, 2 ** 31 - 1), (-2 ** 31, 2 ** 31 - 1)):
        out = torch.full((4, 2, K, P, D), 3.0, dtype=BF16, device=DEV)
        kernels.kv4_read(cache, 0, P, bt, i32([first]), i32([n]), out, keep_first=keep)
        got = out.double().cpu().permute(1, 0, 3, 2, 4).reshape(2, 4 * P, K, D)
        assert torch.equal(got[:, :n], want) and not got[:, n:].any(), (first, keep)


@pytest.mark.parametrize("dtype", [BF16, F32])
@pytest.mark.parametrize("scale", [0.1, 0.7, 1.0, 3.0])
@pytest.mark.parametrize("value", [-1.0, 1.0])
def test_a_bias_of_the_largest_size_on_every_key(dtype, scale, value):
    """The lowest and the highest number as the bias of all keys: scores are lost beside it, whatever the scale, and the row is the keys' average."""
    from xyntetik_runner_b200 import kernels
    H, K, D, P, n, T = 4, 2, 64, 16, 700, 3
    args, q, held, plain, Ts, starts, pos0 = attention_case([n], T, H, K, D, P, dtype, 0, 0, 0, 0, 20)
    args.update(bias=torch.full((H, 20), value * torch.finfo(torch.float32).max, device=DEV), scale=scale)
    out = torch.full((T, H * D), 9.0, dtype=dtype, device=DEV)
    kernels.attention_kv4(q.to(DEV), out, **args)
    # weights that are equal and exact; sums of 700 values in float32 and the output's rounding
    tol = (2.0 ** -8 if dtype is BF16 else 2.0 ** -24 * 700) * float(held[1].abs().max())
    for i in range(T):
        want = held[1][:n - T + 1 + i].mean(0).repeat_interleave(H // K, 0)
        assert torch.all((out[i].double().cpu().reshape(H, D) - want).abs() <= tol)


def sized_case(v, dtype, heads=1, T=1, requests=1):
    """Requests with the same rows, values v [n, D], keys and queries normal: (outputs, queries, held rows of one)."""
    from xyntetik_runner_b200 import kernels
    g = torch.Generator().manual_seed(3)
    n, D = v.shape
    P = 16
    pages = -(-n // P)
    cache = kernels.kv4_cache(pages, 1, 1, D, P, DEV)
    k, v = torch.randn(n, D, generator=g).to(dtype), v.to(dtype)
    bt = i32([np.arange(pages)] * requests)
    kernels.kv4_store(k.to(DEV), v.to(DEV), i32(np.arange(n)), i32(np.zeros(n)), bt, cache, 0, P)
    q = torch.randn(T * requests, heads * D, generator=g).to(dtype)
    out = torch.full((T * requests, heads * D), 9.0, dtype=dtype, device=DEV)
    at = np.full(requests, T, dtype=np.int32), np.full(requests, n - T, dtype=np.int32)
    said = kernels.kv4_plan(at, T * requests, 1, heads, D, P, kernels.dtype_code(dtype), 0, 0, 1 << 30)
    assert requests == 1 or dict(zip(kernels._PLAN, said))["splits"] == 1        # (many requests: one block walks all keys of one)
    kernels.attention_kv4(q.to(DEV), out, cache, 0, P, i32(T * np.arange(requests)), i32(at[0]), i32(at[1]), bt, heads, D, D ** -0.5, at)
    return out, q, [plain_kv4.quantised(x)[2].reshape(n, 1, D) for x in (k, v)]


@pytest.mark.parametrize("dtype", [BF16, F32])
@pytest.mark.parametrize("D", [64, 100, 128, 256])
@pytest.mark.parametrize("T", [1, 9])
def test_groups_of_other_sizes_within_a_head(dtype, D, T):
    """A head's groups of 32 elements lie powers of two apart, 2^-40 to 2^30: every element is as exact as it would be alone."""
    g = torch.Generator().manual_seed(D)
    sizes = torch.tensor([0.0, -21.0, 30.0, -40.0, 8.0, -13.0, -30.0, 14.0])
    v = torch.randn(300, D, generator=g) * torch.exp2(sizes.repeat_interleave(32)[:D])
    out, q, held = sized_case(v, dtype, heads=2, T=T)
    check(out, q, held, dict(scale=D ** -0.5), [T], [0], [300 - T], 2, D, dtype)


@pytest.mark.parametrize("dtype", [BF16, F32])
@pytest.mark.parametrize("first,then", [(-90.0, 100.0), (100.0, -90.0), (-95.0, 30.0), (0.0, -20.0), (3.0, -14.0)])
def test_values_that_begin_small_or_large(dtype, first, then):
    """The first 320 tokens' values are of one size, the others' of another: within what is held, however far apart."""
    g = torch.Generator().manual_seed(1)
    v = torch.randn(640, 64, generator=g)
    v[:320] *= 2.0 ** first
    v[320:] *= 2.0 ** then
    for requests in (1, 1000):
        out, q, held = sized_case(v, dtype, heads=3, requests=requests)
        for r in (0, requests - 1):
            check(out[r:r + 1], q[r:r + 1], held, dict(scale=0.125), [1], [0], [639], 3, 64, dtype)


@pytest.mark.parametrize("dtype", [BF16, F32])
def test_a_loud_token_that_nobody_looks_at(dtype):
    """One token's values are 2^20 times the others', and a bias hides it: the row is what the others make, as exact as ever."""
    from xyntetik_runner_b200 import kernels
    H, K, D, P, n = 2, 1, 64, 16, 300
    g = torch.Generator().manual_seed(2)
    k, v = torch.randn(n, D, generator=g).to(dtype), torch.randn(n, D, generator=g)
    v[n - 4] *= 2.0 ** 20
    v = v.to(dtype)
    cache = kernels.kv4_cache(19, 1, 1, D, P, DEV)
    bt = i32([np.arange(19)])
    kernels.kv4_store(k.to(DEV), v.to(DEV), i32(np.arange(n)), i32(np.zeros(n)), bt, cache, 0, P)
    q = torch.randn(1, H * D, generator=g).to(dtype)
    table = torch.zeros(H, 6)
    table[:, 3] = torch.finfo(torch.float32).min
    out = torch.empty(1, H * D, dtype=dtype, device=DEV)
    at = np.array([1], dtype=np.int32), np.array([n - 1], dtype=np.int32)
    kernels.attention_kv4(q.to(DEV), out, cache, 0, P, i32([0]), i32([1]), i32([n - 1]), bt, H, D, 0.125, at, bias=table.to(DEV))
    held = [plain_kv4.quantised(x)[2].reshape(n, 1, D) for x in (k, v)]
    held[1][n - 4] = 0.0
    table[:, 3] = -1e4                                               # (no weight either way)
    o, size, _ = plain_kv4.attention(q.double().reshape(1, H, D), *held, n - 1, 0.125, bias=table.double())
    raw = plain_kv4.attention(q.double().reshape(1, H, D), *held, n - 1, 0.125)[2]
    assert torch.all((out.double().cpu().reshape(1, H, D) - o).abs() <= plain_kv4.tolerance(o, size, raw, D, dtype))


@pytest.mark.parametrize("dtype", [BF16, F32])
def test_a_query_of_zeros_and_the_smallest_scales(dtype):
    """Scores of zero: equal weights, for every position and every positive scale."""
    from xyntetik_runner_b200 import kernels
    for scale in (1.0, 1e-3, 1e-12, 1e-30, 1e-38):
        args, q, held, plain, Ts, starts, pos0 = attention_case([200, 70], 3, 4, 2, 64, 16, dtype, 0, 0, 0, 0, 0)
        q[:, :] = 0.0
        q[1] = 1e-20
        args["scale"] = plain["scale"] = scale
        out = torch.full((q.shape[0], 4 * 64), 9.0, dtype=dtype, device=DEV)
        kernels.attention_kv4(q.to(DEV), out, **args)
        check(out, q, held, plain, Ts, starts, pos0, 4, 64, dtype)


@pytest.mark.parametrize("H,K,D,P", [(64, 8, 128, 64), (66, 33, 48, 24)])
@pytest.mark.parametrize("captured", [False, True])
def test_rows_read_back_a_few_requests_at_a_time(H, K, D, P, captured, monkeypatch):
    """A step whose rows are more than are read back at once: the same bits as in one go, within the bytes that are said or one request's."""
    from xyntetik_runner_b200 import kernels
    contexts, Ts = [400, 90, 300, 5, 700, 200, 120], [100, 1, 60, 5, 90, 0, 120]
    args, q, held, plain, Ts, starts, pos0 = attention_case(contexts, Ts, H, K, D, P, BF16, 0, 0, 0, 0, 0)
    if captured:
        args.update({name: args[name].view(1, -1) for name in ("seg_start", "seg_len", "seg_pos0")})       # (so many values, whatever their shape)
    qd, outs, asked = q.to(DEV), [], []
    for pages in (10 ** 6, 9, 1):
        monkeypatch.setattr(kernels, "KV4_VALUES_BYTES", pages * 4 * K * P * D)
        out, buf, sizes = torch.full((q.shape[0] + 5, H * D), 9.0, dtype=BF16, device=DEV), shared(), {}
        call = lambda: kernels.attention_kv4(qd, out[:-5], **args, buf=lambda name, shape, dtype: (sizes.__setitem__(name, shape), buf(name, shape, dtype))[1])
        call()
        if captured:
            g = torch.cuda.CUDAGraph()
            torch.cuda.synchronize()
            with torch.cuda.graph(g):
                call()
            out[:-5] = 9.0
            g.replay()
        kernels.tc_check_status(torch.device(DEV))
        outs.append(out)
        asked.append(sizes["kv4_values"][0])
    check_many(outs[0][:-5], q, held, Ts, starts, pos0, H, D, BF16)
    assert all(torch.equal(out, outs[0]) for out in outs) and torch.all(outs[0][-5:] == 9.0)
    longest = args["block_tables"].shape[1]
    assert asked[0] >= sum(-(-c // P) for c, T in zip(contexts, Ts) if T * H // K > 64) and asked[1] <= max(9, longest) and asked[2] <= longest


@pytest.mark.parametrize("contexts,Ts,H,K,D,P,dtype", [
    ([9000, 300, 5000, 60], [1, 40, 5, 0], 8, 2, 64, 64, BF16), ([9000, 300, 5000, 60], [1, 40, 5, 0], 8, 2, 64, 64, F32),
    ([6000, 300, 300, 700], [1, 210, 8, 7], 32, 4, 128, 64, BF16), ([4000, 9000, 300, 2000], [3, 1, 30, 7], 6, 3, 100, 24, BF16)])
def test_partial_sums_of_portions_of_many_lengths(contexts, Ts, H, K, D, P, dtype):
    """Spans of portions with one row block and with many, empty ones and ones that go another way among them, in the scratch that the plan says and no further."""
    from xyntetik_runner_b200 import kernels
    args, q, held, plain, Ts, starts, pos0 = attention_case(contexts, Ts, H, K, D, P, dtype, 0, 0, 0, 0, 0)
    aligned = dtype is BF16 and D % 16 == 0
    said = dict(zip(kernels._PLAN, kernels.kv4_plan(args["lengths"], q.shape[0], K, H // K, D, P, kernels.dtype_code(dtype), 0, 0, 64 if aligned else 1 << 30)))
    assert said["floats"] > 0 and said["row_blocks"] > 1 and (said["long"] > 0) == (H == 32)
    whole = {}

    def buf(name, shape, dt):
        t = torch.empty(math.prod(shape) + 64, dtype=dt, device=DEV)
        if name == "kv4_spans":
            t.fill_(math.nan)
            whole[name] = t
        return t[:math.prod(shape)].view(*shape)
    for b in (None, buf):
        out = torch.full((q.shape[0], H * D), 9.0, dtype=dtype, device=DEV)
        kernels.attention_kv4(q.to(DEV), out, **args, buf=b)
        kernels.tc_check_status(torch.device(DEV))
        check_many(out, q, held, Ts, starts, pos0, H, D, dtype)
    assert torch.isnan(whole["kv4_spans"][said["floats"]:]).all()


@pytest.mark.parametrize("dtype", [BF16, F32])
def test_pages_of_no_tokens_are_refused(dtype):
    """A page size of 0 is a mistake, not another way to store: the rotation writes rows only where it is told to, and then the same keys and values."""
    from xyntetik_runner_b200 import kernels
    g = torch.Generator().manual_seed(3)
    n, H, K, D, P = 5, 4, 2, 64, 8
    qkv = torch.randn(n, (H + 2 * K) * D, generator=g).to(dtype).to(DEV)
    pos, seg, bt = i32(np.arange(n)), i32(np.zeros(n)), i32([[0]])
    freq = (10000.0 ** (-torch.arange(32) / 32.0))
    pages, rows = torch.zeros(1, 2, K, P, D, dtype=dtype, device=DEV), torch.zeros(n, 2 * K * D, dtype=dtype, device=DEV)
    turn = lambda cache, stride, v_at, page, **k: kernels.rope_store(qkv.clone(), pos, seg, bt, freq.to(DEV), cache.data_ptr(), stride, v_at, H, K, D, D, 1, page, **k)
    norm = lambda cache, stride, v_at, page, **k: kernels.qk_norm_rope_store(
        qkv, torch.zeros(n, H * D, dtype=dtype, device=DEV), pos, seg, bt, freq.double().to(DEV), None, None, cache.data_ptr(), stride, v_at, H, K, D, D, D, D, 1, page, False, 1e-5, **k)
    for fn in (turn, norm):
        for page in (0, -1):
            with pytest.raises(kernels.KernelError, match="refuses these sizes"):
                fn(pages, 2 * K * P * D, K * P * D, page)
        assert not pages.any()
        fn(pages, 2 * K * P * D, K * P * D, P)
        fn(rows, 2 * K * D, K * D, P, to_rows=True)
        assert torch.equal(pages[0, :, :, :n].permute(2, 0, 1, 3).reshape(n, -1), rows) and rows.any()
        pages.zero_(), rows.zero_()


@pytest.mark.parametrize("H,K,D,P,dtype,contexts,T,window,keep", [
    (8, 2, 128, 64, BF16, [2500, 300, 700], 1, 0, 0), (8, 8, 64, 16, BF16, [2500, 300, 700], 1, 0, 0), (8, 2, 64, 64, F32, [2500, 300, 700], 1, 0, 0),
    (2, 1, 64, 64, BF16, [9000, 40], 1, 0, 0), (8, 2, 128, 16, BF16, [3000, 1100], 1, 900, 70), (8, 2, 100, 24, BF16, [1200, 500], 3, 0, 0), (4, 2, 256, 64, F32, [900] * 3, 2, 0, 0)])
def test_rows_of_earlier_steps_read_ahead_of_the_kernel_before(H, K, D, P, dtype, contexts, T, window, keep):
    """Steps as an engine queues them: a copy of the positions, a store of the step's own rows, the attention, which may read earlier rows at once.  The same bits as
    a call that waits, whose last step is compared with the plain form."""
    from xyntetik_runner_b200 import kernels
    steps, R = 12, len(contexts)
    ends = [c + steps * T for c in contexts]
    args, _, held, plain, *_ = attention_case(ends, T, H, K, D, P, dtype, 0, 0, 0, 0, 0)
    args.update(window=window, keep_first=keep)
    plain.update(window=window, keep=keep)
    g = torch.Generator().manual_seed(8)
    new = [torch.randn(steps, R * T, K * D, generator=g).to(dtype) for _ in (0, 1)]
    q = torch.randn(steps, R * T, H * D, generator=g).to(dtype)
    starts = np.repeat(contexts, T) + np.tile(np.arange(T), R)
    flat = [torch.from_numpy((starts + s * T).astype(np.int32)).pin_memory() for s in range(steps)]
    first = [torch.from_numpy((np.array(contexts) + s * T).astype(np.int32)).pin_memory() for s in range(steps)]
    seg = i32(np.repeat(np.arange(R), T))
    one = np.full(R, T, dtype=np.int32)
    new_d, q_d, clean, cuts = [x.to(DEV) for x in new], q.to(DEV), args["cache"].clone(), set()
    outs = {}
    for early in (False, True):
        args["cache"].copy_(clean)
        # (what lies where the steps' rows go: anything)
        out = torch.full((steps, R * T, H * D), 9.0, dtype=dtype, device=DEV)
        pos, pos0 = i32(starts), i32(contexts)
        torch.cuda.synchronize()
        for s in range(steps):
            pos.copy_(flat[s], non_blocking=True)
            pos0.copy_(first[s], non_blocking=True)
            kernels.kv4_store(new_d[0][s], new_d[1][s], pos, seg, args["block_tables"], args["cache"], args["layer"], P)
            lengths = one, first[s].numpy()
            said = dict(zip(kernels._PLAN, kernels.kv4_plan(lengths, R * T, K, H // K, D, P, kernels.dtype_code(dtype), window, keep, 1 << 30, max(ends))))
            cuts.add((said["splits"] > 1, bool(said["clustered"])))
            kernels.attention_kv4(q_d[s], out[s], **{**args, "seg_pos0": pos0, "lengths": lengths}, max_kv_len=max(ends), early=early)
        torch.cuda.synchronize()
        outs[early] = out
    assert cuts <= {(True, True), (True, False)} and torch.equal(outs[True], outs[False])
    full = []
    for r, (c, e) in enumerate(zip(contexts, ends)):
        for plane in (0, 1):
            x = held[2 * r + plane].clone()
            x[c:] = plain_kv4.quantised_rows(new[plane][:, r * T:(r + 1) * T].reshape(steps * T, K, D))
            full.append(x)
    check(outs[True][-1], q[-1], full, plain, [T] * R, np.arange(R) * T, np.array(ends) - T, H, D, dtype)


def test_two_calls_at_once():
    """On two streams, each with portions that are read back, spans with scratch and single tokens: the bits that each gives alone."""
    from xyntetik_runner_b200 import kernels
    cases = [([6000, 300, 300, 700], [1, 210, 8, 7], 32, 4, 128, 64, BF16, 0, 0, 0, 0, 0), ([5000, 400, 80], [2, 130, 1], 66, 33, 48, 24, BF16, 0, 0, 1, 0, 0)]
    made = [attention_case(*c, seed=i) for i, c in enumerate(cases)]
    qs = [m[1].to(DEV) for m in made]
    alone = [torch.empty(q.shape[0], c[2] * c[4], dtype=BF16, device=DEV) for q, c in zip(qs, cases)]
    for m, q, out in zip(made, qs, alone):
        kernels.attention_kv4(q, out, **m[0])
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in cases]
    outs = [[torch.empty_like(alone[i]) for _ in range(20)] for i in (0, 1)]
    torch.cuda.synchronize()
    for n in range(20):
        for i in (0, 1):
            with torch.cuda.stream(streams[i]):
                kernels.attention_kv4(qs[i], outs[i][n], **made[i][0])
    torch.cuda.synchronize()
    kernels.tc_check_status(torch.device(DEV))
    assert all(torch.equal(out, alone[i]) for i in (0, 1) for out in outs[i])
    check_many(alone[0], made[0][1], made[0][2], cases[0][1], made[0][5], made[0][6], 32, 128, BF16)
