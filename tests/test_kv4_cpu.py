"""The cache in four bits: its numbers and its refusals, without a GPU."""
import math

import numpy as np
import pytest
import torch

import plain_kv4
from xyntetik_runner_b200 import kernels


def test_values_are_bfloat16_numbers():
    """c s has at most eight significant bits for every code and every scale: three (or a power of two) times five."""
    for m in range(16, 32):
        for c in range(-8, 8):
            x = c * -(m / 32.0) / 8.0
            assert float(torch.tensor(x, dtype=torch.float64).to(torch.bfloat16)) == x
        assert float(torch.tensor(24.0 * m, dtype=torch.float64).to(torch.bfloat16)) == 24.0 * m


def test_a_group_is_near_what_it_holds():
    """Half a step everywhere but at the smaller side's end, where seven steps reach: a step is the largest magnitude / 8, give or take 1 / 32."""
    g = np.random.default_rng(3)
    for _ in range(300):
        x = g.standard_normal(32) * math.exp(g.uniform(-20, 20))
        codes, s = plain_kv4.group(x)
        off = np.abs(codes * s - x)
        inside = x / s <= 7.5
        assert np.all(off[inside] <= abs(s) * 0.5 * (1 + 1e-12)) and np.all(off <= abs(s) * 1.26)
        assert abs(abs(s) * 8 / np.max(np.abs(x)) - 1) <= 1 / 32


def test_sizes():
    assert [kernels.kv4_held(d) for d in (1, 16, 64, 65, 128, 129, 256)] == [64, 64, 64, 128, 128, 256, 256]
    assert kernels.kv4_block_bytes(128, 64) == 64 * 144 and kernels.kv4_block_bytes(40, 8) == 8 * 72
    for hd in (0, 257, -1):
        with pytest.raises(kernels.KernelError, match="heads of 1 to 256"):
            kernels.kv4_held(hd)
    for page in (0, 4, 12, 20, -8, 1 << 17):
        with pytest.raises(kernels.KernelError, match="multiple of 8"):
            kernels.kv4_block_bytes(64, page)
    c = kernels.kv4_cache(3, 2, 4, 100, 16, "cpu")
    assert c.shape == (3, 2, 4, 16 * 144) and c.dtype == torch.uint8 and not c.any()


def _parts(K=2, D=64, P=16, n=4, S=2):
    i = torch.zeros(n, dtype=torch.int32)
    return dict(k=torch.zeros(n, K * D), v=torch.zeros(n, K * D), positions=i, tok_seg=i, block_tables=torch.zeros(S, 3, dtype=torch.int32),
                cache=kernels.kv4_cache(3, 1, K, D, P, "cpu"), layer=0, page_size=P)


@pytest.mark.parametrize("change, message", [
    (dict(k=torch.zeros(4, 127)), "kv heads"), (dict(v=torch.zeros(3, 128)), "kv heads"), (dict(v=torch.zeros(4, 128, dtype=torch.bfloat16)), "one type"),
    (dict(k=torch.zeros(128, 4).t()), "side by side"), (dict(positions=torch.zeros(4, dtype=torch.int64)), "int32"),
    (dict(tok_seg=torch.zeros(3, dtype=torch.int32)), "int32"), (dict(block_tables=torch.zeros(6, dtype=torch.int32)), "block tables"),
    (dict(cache=torch.zeros(3, 1, 2, 8)), "current CUDA device|uint8"), ({}, "current CUDA device")])
def test_store_refuses(change, message):
    with pytest.raises(kernels.KernelError, match=message):
        kernels.kv4_store(**{**_parts(), **change})


@pytest.mark.parametrize("change, message", [
    (dict(out=torch.zeros(2, 2, 2, 8, 64)), "out is"), (dict(out=torch.zeros(2, 2, 3, 16, 64)), "out is"), (dict(keep_first=-1), "keep_first"),
    (dict(first=torch.zeros(1, dtype=torch.int32)), "first"), (dict(tables=torch.zeros(2, 2, dtype=torch.int32)), "tables"), ({}, "current CUDA device")])
def test_read_refuses(change, message):
    p = _parts()
    i = torch.zeros(2, dtype=torch.int32)
    args = dict(cache=p["cache"], layer=0, page_size=16, block_tables=p["block_tables"], first=i, end=i, out=torch.zeros(2, 2, 2, 16, 64))
    with pytest.raises(kernels.KernelError, match=message):
        kernels.kv4_read(**{**args, **change})


@pytest.mark.parametrize("change, message", [
    (dict(heads=3), "query heads"), (dict(out=torch.zeros(4, 255)), "rows of the same tokens"), (dict(q=torch.zeros(4, 255)), "rows of the same tokens"),
    (dict(q=torch.zeros(4, 256, dtype=torch.bfloat16)), "rows of the same tokens"), (dict(scale=0.0), "scale"), (dict(scale=math.nan), "scale"),
    (dict(window=-1), "window"), (dict(softcap=-1.0), "window"), (dict(softcap=1.0, bias=torch.zeros(4, 3)), "without a cap|CUDA"),
    (dict(sink=torch.zeros(3)), "sink"), (dict(seg_pos0=torch.zeros(2)), "seg_pos0"), ({}, "current CUDA device")])
def test_attention_refuses(change, message):
    p, i = _parts(), torch.zeros(2, dtype=torch.int32)
    two = np.array([2, 2], dtype=np.int32)
    args = dict(q=torch.zeros(4, 256), out=torch.zeros(4, 256), cache=p["cache"], layer=0, page_size=16, seg_start=i, seg_len=i, seg_pos0=i,
                block_tables=p["block_tables"], heads=4, head_dim=64, scale=0.1, lengths=(two, two))
    with pytest.raises(kernels.KernelError, match=message):
        kernels.attention_kv4(**{**args, **change})


def test_what_portions_ask_for():
    """Pages that are read back, row tiles and scratch, from lengths on the host (the library's part that needs no device)."""
    a = lambda *x: np.array(x, dtype=np.int32)
    # (2,000 pairs: more row blocks than go by the codes, whatever the portions)
    plan = lambda l, p, window=0, keep=0, most=0, n=100: kernels.kv4_plan((l, p), n, 2000, 4, 64, 16, kernels.BF16, window, keep, most).tolist()[:9]
    assert plan(a(1, 60), a(0, 15)) == [0, 2, 0, 1 + 5, 60, 1 + 2, 1 + 4, 75, 0]
    assert plan(a(0, 60), a(7, 15))[:4] == [0, 1, 0, 5]
    assert plan(a(30), a(100), 10, 20)[3] == 2 + 4          # rows 91 .. 129 lie in pages 5 to 8, the kept in 0 and 1
    assert plan(a(30), a(40), 20, 33)[3] == 1 + 4           # kept rows that the window's pages hold are not there twice
    # anywhere up to `mx` rows: all pages of them, or the window's at its worst place and the kept
    far = lambda l, p, window, keep, mx: kernels.kv4_plan((l, p), 100, 2000, 4, 64, 16, kernels.BF16, window, keep, 0, mx).tolist()
    assert far(a(30), a(100), 0, 0, 500)[3] == 32 and far(a(30), a(100), 0, 0, 500)[7] == 500 and far(a(30), a(100), 0, 0, 90)[3] == 9
    for window, keep in ((10, 20), (1, 0), (33, 5), (400, 3)):
        held = far(a(30), a(0), window, keep, 300)[3]
        need = [plan(a(30), a(p), window, keep)[3] for p in range(271)]
        assert max(need) <= held <= max(need) + 1
    assert plan(a(1, 60), a(0, 15), most=64)[:2] == [1, 1] and plan(a(1, 60), a(0, 15), most=64)[8] == 64
    few = kernels.kv4_plan((a(1, 60), a(0, 15)), 100, 2, 4, 64, 16, kernels.BF16, 0, 0, 64).tolist()
    assert few[:2] == [2, 0] and few[8] == 1 << 30          # 30 row blocks: by the codes
    at = lambda kv, *l, d=128: kernels.kv4_plan((a(*l), a(*[900] * len(l))), 400, kv, 4, d, 16, kernels.BF16, 0, 0, 64).tolist()[:2]
    assert at(16, 64) == [1, 0] and at(17, 64) == [0, 1]    # full row tiles: 256 row blocks, 272
    assert at(20, 64, d=64) == [1, 0] and at(21, 64, d=64) == [0, 1]
    assert at(16, 64, 1) == [2, 0] and at(17, 64, 1) == [1, 1]
    assert at(64, 24) == [1, 0] and at(65, 24) == [0, 1]    # a part full one: 384, 390
    assert at(96, 24, d=64) == [1, 0] and at(97, 24, d=48) == [0, 1]
    assert at(8, 64, 64) == [2, 0] and at(12, 64, 64) == [0, 2]
    assert at(16, 64, 24) == [2, 0] and at(18, 64, 24) == [0, 2]
    for l, p, n in ((a(-1), a(0), 9), (a(1), a(-1), 9), (a(5, 5), a(0, 0), 9), (a(8), a(2 ** 31 - 8), 9)):
        with pytest.raises(kernels.KernelError, match="does not hold"):
            plan(l, p, n=n)
    for l, p in ((a(1), a(1, 2)), (a(1).astype(np.int64), a(1)), (a(1).astype(">i4"), a(1)), (a(1), a(1).astype(np.float32))):
        with pytest.raises(kernels.KernelError, match="one value a portion"):
            plan(l, p)
    with pytest.raises((BufferError, ValueError), match="contiguous"):
        plan(np.zeros(8, dtype=np.int32)[::2], np.zeros(8, dtype=np.int32)[::2])


@pytest.mark.parametrize("lens,K,G,D,cut", [
    ([60] * 70, 40, 1, 64, "whole"), ([64], 1, 4, 128, "whole"), ([640], 1, 4, 128, "cluster"), ([640], 8, 4, 64, "cluster"), ([8192] * 8, 8, 4, 128, "cluster"),
    ([20000], 1, 8, 128, "spans"), ([131072], 8, 4, 128, "spans")])
def test_how_requests_are_cut(lens, K, G, D, cut):
    """Whole, in spans that a cluster combines, in spans with scratch and a second kernel; every tile belongs to a span, with requests as long as is announced too."""
    n = np.array(lens, dtype=np.int32)
    for most in (0, 3 * max(lens)):
        said = dict(zip(kernels._PLAN, kernels.kv4_plan((np.ones_like(n), n - 1), len(lens), K, G, D, 64, kernels.BF16, 0, 0, 1 << 30, most)))
        assert said["short"] == len(lens) and said["long"] == 0 and said["row_blocks"] == 1
        if most == 0:
            assert ("whole" if said["splits"] == 1 else "cluster" if said["clustered"] else "spans") == cut
        assert (said["floats"] > 0) == (said["splits"] > 1 and not said["clustered"]) and (not said["clustered"] or said["splits"] <= 8)
        assert said["splits"] * said["span_tiles"] * 64 >= max(lens)


def test_a_plan_through_either_way_of_calling(monkeypatch):
    """Buffers reach the library from the direct calls and through ctypes alike."""
    l, p = np.array([1, 70, 0], dtype=np.int32), np.array([900, 30, 5], dtype=np.int32)
    args = ((l, p), 80, 900, 4, 64, 16, kernels.BF16, 100, 3, 64)
    direct = kernels.kv4_plan(*args)
    monkeypatch.setattr(kernels, "_c", kernels._CtypesCalls(kernels.lib()))
    assert kernels.kv4_plan(*args) == direct and direct[0] == 1 and direct[1] == 1
    with pytest.raises((BufferError, ValueError), match="contiguous"):
        kernels.kv4_plan((np.zeros(8, dtype=np.int32)[::2], np.zeros(8, dtype=np.int32)[::2]), *args[1:])


def test_engine_refuses_before_it_looks_for_a_device():
    from xyntetik_runner_b200.engine.engine import Engine, EngineParams
    with pytest.raises(ValueError, match="same or int4"):
        Engine("nowhere", EngineParams(kv="q8_0"))
    with pytest.raises(ValueError, match="multiple of 8"):
        Engine("nowhere", EngineParams(kv="int4", page_size=20))


def test_bytes_of_a_token():
    from xyntetik_runner_b200.engine.model import kv_head_bytes
    from xyntetik_runner_b200.parts.base import KVNeed
    assert kv_head_bytes(KVNeed(8, 128, four_bits=True), 2, True) == 144 and kv_head_bytes(KVNeed(8, 128, four_bits=True), 2, False) == 512
    assert kv_head_bytes(KVNeed(1, 576, planes=1), 2, True) == 1152 and kv_head_bytes(KVNeed(1, 40, four_bits=True), 4, True) == 72


def test_option():
    from xyntetik_runner_b200 import cli
    assert cli.build_parser().parse_args(["-m", "x"]).kv == "same" and cli.build_parser().parse_args(["-m", "x", "--kv", "int4"]).kv == "int4"


def test_plans_of_the_longest_windows_and_kept_rows():
    """Up to the largest 32-bit number: as if there were no window."""
    l, p = np.array([1, 3, 70], dtype=np.int32), np.array([5000, 40, 900], dtype=np.int32)
    for most in (64, 1 << 30):
        plain = kernels.kv4_plan((l, p), 100, 900, 4, 64, 16, kernels.BF16, 0, 0, most)
        for window, keep in ((40, 2 ** 31 - 1), (2 ** 31 - 1, 0), (2 ** 31 - 1, 2 ** 31 - 1)):
            assert kernels.kv4_plan((l, p), 100, 900, 4, 64, 16, kernels.BF16, window, keep, most) == plain
            kernels.kv4_plan((l, p), 100, 900, 4, 64, 16, kernels.BF16, window, keep, most, 2 ** 31 - 1)


@pytest.mark.parametrize("name", ["window", "keep_first", "max_kv_len"])
def test_numbers_that_have_more_than_31_bits(name):
    p, i = _parts(), torch.zeros(2, dtype=torch.int32)
    two = np.array([2, 2], dtype=np.int32)
    for much in (2 ** 31, 2 ** 32 + 5):
        with pytest.raises(kernels.KernelError, match="31 bits"):
            kernels.attention_kv4(torch.zeros(4, 256), torch.zeros(4, 256), p["cache"], 0, 16, i, i, i, p["block_tables"], 4, 64, 0.1, (two, two), **{name: much})
    if name == "keep_first":
        with pytest.raises(kernels.KernelError, match="keep_first"):
            kernels.kv4_read(p["cache"], 0, 16, p["block_tables"], i, i, torch.zeros(2, 2, 2, 16, 64), keep_first=2 ** 31)


def test_portions_that_are_read_back_together():
    """Neighbours up to so many pages, one at least, none without a page; the sums are those of one plan over each."""
    l, p = np.array([60, 1, 90, 0, 60, 200, 60], dtype=np.int32), np.array([100, 900, 10, 4, 0, 800, 4], dtype=np.int32)
    plan = lambda a, b: kernels.kv4_plan((l[a:b], p[a:b]), 1000, 900, 4, 64, 16, kernels.BF16, 0, 0, 64, 0, rule=False)
    each = [plan(i, i + 1)[3] for i in range(7)]
    assert each == [10, 0, 7, 0, 4, 63, 4]
    for at_once in (1, 10, 11, 17, 21, 84, 88, 1000):
        groups = kernels._kv4_groups(plan, 7, at_once)
        assert sum(g[2] for g in groups) == sum(each) and [g[0] for g in groups] == sorted(g[0] for g in groups)
        for a, b, pages, longest, t128, t64, end in groups:
            long = [i for i in range(a, b) if each[i]]
            assert pages == sum(each[a:b]) and (pages <= at_once or len(long) == 1)
            assert longest == max(l[i] for i in long) and end == max(l[i] + p[i] for i in long)
            assert t128 == sum(-(-4 * l[i] // 128) for i in long) and t64 == sum(-(-4 * l[i] // 64) for i in long)
    assert len(kernels._kv4_groups(plan, 7, 1000)) == 1 and len(kernels._kv4_groups(plan, 7, 1)) == 5
    # a rule that is asked may send portions to the codes; one that stands does not
    few = (np.array([60], dtype=np.int32), np.array([15], dtype=np.int32))
    asked, stands = (kernels.kv4_plan(few, 100, 2, 4, 64, 16, kernels.BF16, 0, 0, 64, 0, rule=r) for r in (True, False))
    assert asked[:2].tolist() == [1, 0] and stands[:2].tolist() == [0, 1] and stands[8] == 64


def test_the_context_that_fits(monkeypatch):
    """-c 0 with four bits: the pool and the buffer of rows read back, as the attention asks for it, fit; one more page of every request does not."""
    from xyntetik_runner_b200 import architectures  # noqa: F401
    from xyntetik_runner_b200.config import registry
    from xyntetik_runner_b200.engine.runner import Runner
    d = {"architectures": ["LlamaForCausalLM"], "hidden_size": 256, "num_hidden_layers": 3, "num_attention_heads": 8, "num_key_value_heads": 2, "head_dim": 64,
         "intermediate_size": 320, "vocab_size": 300, "rms_norm_eps": 1e-5, "rope_theta": 10000.0, "max_position_embeddings": 1 << 30,
         "tie_word_embeddings": False, "torch_dtype": "bfloat16"}
    arch = registry.resolve(registry.architecture_name(d))
    for dtype, heads_dim in (("bfloat16", 64), ("bfloat16", 100), ("float32", 64)):
        cfg = arch.config_from_dict({**d, "head_dim": heads_dim})
        weights = 2 * sum(math.prod(s.shape) for s in arch.build_plan(cfg).tensor_specs().values())
        reads = dtype == "bfloat16" and heads_dim % 16 == 0
        for free in (1 << 26, 1 << 30, 7 << 30, 150 << 30):
            monkeypatch.setattr(torch.cuda, "mem_get_info", lambda *a, f=free: (f, 1 << 38))
            for parallel in (1, 3, 64):
                for P in (16, 64):
                    room = int(0.9 * free) - 2 * weights
                    token = 3 * 2 * kernels.kv4_block_bytes(heads_dim, 8) // 8
                    values = 2 * 2 * heads_dim * 2 if reads else 0

                    def held(n):
                        rows = max(kernels.KV4_VALUES_BYTES, values * n)              # one request's rows, or so many bytes of several
                        return n * token * parallel + min(rows, 2 * values * n * parallel)
                    n = Runner._fit_context(arch, cfg, 1 << 30, parallel, P, dtype, "cuda:0", "int4")
                    assert n % P == 0 and held(n) <= room and (held(n + P) > room or n == 1 << 30)
                    elem = 2 if dtype == "bfloat16" else 4
                    same = Runner._fit_context(arch, cfg, 1 << 30, parallel, P, dtype, "cuda:0")
                    assert same == room // (3 * 2 * 2 * heads_dim * elem * parallel) // P * P
        monkeypatch.setattr(torch.cuda, "mem_get_info", lambda *a: (2 * weights, 1 << 38))
        with pytest.raises(ValueError, match="no context fits"):
            Runner._fit_context(arch, cfg, 1 << 30, 4, 16, dtype, "cuda:0", "int4")


def test_a_larger_buffer_does_not_wait_beside_the_old_one(monkeypatch):
    """An engine's buffer that grows: the old one and everything that holds it are gone when the new one is made; a failure leaves none behind."""
    import weakref
    from types import SimpleNamespace
    from xyntetik_runner_b200.engine.engine import Engine, StepContext
    eng = Engine.__new__(Engine)
    eng.params, eng.device = SimpleNamespace(max_step_tokens=0), torch.device("cpu")
    eng._bufs, eng._views, eng._graphs, eng._uneven_of_shape, eng._buf_generation = {}, {}, {}, {}, 0
    ctx = StepContext.__new__(StepContext)
    ctx._eng, ctx._views = eng, eng._views
    ctx.buf("a", (10,), torch.int32)
    old = weakref.ref(eng._bufs[("a", torch.int32)])
    eng._graphs["one"] = object()
    real, seen = torch.empty, []
    monkeypatch.setattr(torch, "empty", lambda *a, **k: (seen.append(old() is None and not eng._graphs), real(*a, **k))[1])
    assert ctx.buf("a", (11,), torch.int32).shape == (11,) and seen == [True] and eng._buf_generation == 2

    def fails(*a, **k):
        raise torch.cuda.OutOfMemoryError("no room")
    monkeypatch.setattr(torch, "empty", fails)
    with pytest.raises(torch.cuda.OutOfMemoryError):
        ctx.buf("a", (12,), torch.int32)
    monkeypatch.setattr(torch, "empty", real)
    assert ctx.buf("a", (12,), torch.int32).shape == (12,) and eng._buf_generation == 4


@pytest.mark.parametrize("lens,ends,K,G,D,code", [([1985] + [1] * 63, [1985] + [8001] * 63, 8, 4, 128, 0), ([40] + [1] * 63, [40] + [8001] * 62 + [131001], 8, 4, 128, 1),
                                                  ([1900, 1], [1900, 100001], 8, 4, 192, 1), ([1900] + [1] * 31, [1900] + [8001] * 31, 2, 4, 256, 1)])
def test_scratch_of_steps_that_mix_portions_and_single_tokens(lens, ends, K, G, D, code):
    """Scratch goes by the row blocks that there are, within 256 MB; every tile still belongs to a span."""
    l, e = np.array(lens, dtype=np.int32), np.array(ends, dtype=np.int32)
    said = dict(zip(kernels._PLAN, kernels.kv4_plan((l, e - l), int(l.sum()), K, G, D, 64, code, 0, 0, 1 << 30)))
    rows = 8 if code == 0 or not said["wide"] else 16
    assert said["splits"] > 1 and not said["clustered"] and said["blocks"] == sum(-(-n * G // rows) for n in lens)
    assert said["floats"] == said["blocks"] * K * said["splits"] * rows * (plain_kv4.held(D) + 2) <= 1 << 26
    assert said["splits"] * said["span_tiles"] * (64 if D <= 128 else 32) >= max(ends)


@pytest.mark.parametrize("T,H,code,blocks", [(1, 8, 0, 148), (1, 16, 0, 148), (4, 32, 1, 148), (1, 32, 1, 296)])
def test_spans_of_heads_of_256_elements_run_at_once(T, H, code, blocks):
    """Equal requests that fit in one round are cut into one: an SM holds one block of sixteen rows or of float32, two of eight bfloat16 rows (148 SMs)."""
    l, p = np.full(8, T, dtype=np.int32), np.full(8, 8192 - T, dtype=np.int32)
    said = dict(zip(kernels._PLAN, kernels.kv4_plan((l, p), 8 * T, 8, H // 8, 256, 64, code, 0, 0, 1 << 30)))
    assert said["splits"] > 1 and 8 * 8 * said["splits"] <= blocks


@pytest.mark.parametrize("requests,keys,reach,window,splits,cut", [
    (64, 1000, 1024, 0, 1, "whole"), (64, 200, 1024, 0, 1, "whole"), (64, 8192, 8192, 0, 4, "spans"), (1, 8192, 8192, 0, 32, "spans"), (1, 100, 1024, 0, 4, "cluster"),
    (1, 300, 1024, 0, 4, "cluster"), (8, 7300, 8192, 0, 6, "cluster"), (32, 5000, 5120, 1024, 1, "whole"), (1, 5000, 5120, 1024, 5, "cluster")])
def test_captured_steps_are_cut_for_the_lengths_that_they_may_meet(requests, keys, reach, window, splits, cut):
    """8 kv heads of 128 elements, single tokens: what is planned does not hang on the lengths at capture, and is what the longest lengths ask for."""
    one = np.ones(requests, dtype=np.int32)
    plan = lambda n, reach: dict(zip(kernels._PLAN, kernels.kv4_plan((one, np.full(requests, n - 1, dtype=np.int32)), requests, 8, 4, 128, 64, kernels.BF16, window, 0, 64, reach)))
    said = plan(keys, reach)
    assert said["splits"] == splits and ("whole" if splits == 1 else "cluster" if said["clustered"] else "spans") == cut
    assert (said["floats"] > 0) == (cut == "spans")
    assert all(plan(n, reach) == said for n in (max(1, reach - 1000), reach - 500, reach))
    if not window:
        assert plan(reach, 0) == said


def test_rows_on_pages_that_were_let_go_are_zeros():
    """An engine without four bits: nothing of the page that stands in for a missing one, numbers or not; the cache stays as it is."""
    from types import SimpleNamespace
    from xyntetik_runner_b200.engine.engine import Engine
    eng = Engine.__new__(Engine)
    P, K, D = 4, 2, 3
    eng.device, eng.act_dtype, eng.params = torch.device("cpu"), torch.float32, SimpleNamespace(page_size=P)
    eng.model = SimpleNamespace(layers=[SimpleNamespace(group=0, layer_in_group=1)], groups=[SimpleNamespace(planes=2, kv_heads=K, head_dim=D)])
    kv = torch.arange(3 * 2 * 2 * K * P * D, dtype=torch.float32).view(3, 2, 2, K, P, D)
    kv[0, 1, 0], kv[0, 1, 1] = math.nan, math.inf
    eng.kv, eng.four_bits = [kv], [False]
    eng.cache = SimpleNamespace(length=lambda r: 10, block_table=lambda g, r: np.array([-1, 2, 1, -1], dtype=np.int32))
    before = kv.clone()
    k, v = eng.cached_rows("a", 0)
    for rows, plane in ((k, 0), (v, 1)):
        assert rows.shape == (10, K, D) and not rows[:4].any()
        assert torch.equal(rows[4:8], kv[2, 1, plane].permute(1, 0, 2)) and torch.equal(rows[8:], kv[1, 1, plane, :, :2].permute(1, 0, 2))
    assert torch.equal(torch.nan_to_num(kv), torch.nan_to_num(before))


def test_entries_that_can_and_that_cannot(monkeypatch):
    """Mixers that cannot have their rows in four bits beside others that can: without four bits they share groups and caches as ever; with them a
    cache is in four bits where everyone who writes or reads it can."""
    from types import SimpleNamespace
    from xyntetik_runner_b200.engine import model
    from xyntetik_runner_b200.parts.base import KVNeed
    mixer = lambda four, **k: SimpleNamespace(mixer=SimpleNamespace(kv_need=lambda: KVNeed(2, 64, four_bits=four, **k), state_need=lambda: None))
    state = SimpleNamespace(mixer=SimpleNamespace(kv_need=lambda: None, state_need=lambda: None))
    blocks = [mixer(True), mixer(False), mixer(True, window=9), mixer(True), state]
    entry = model.ScheduleEntry
    schedule = [entry(0), entry(1), entry(0), entry(1, cache_from=2), entry(2), entry(3), entry(4), entry(0, cache_from=1), entry(3, cache_from=5)]
    plan = model.ModelPlan(None, blocks, schedule, None, None, 64, 10, 100)
    plan.validate()
    assert plan.four_bits() == [True, False, False, False, True, True, False, True, True]
    monkeypatch.setattr(model.ModelPlan, "parts", lambda self: [])
    monkeypatch.setattr(model, "load_tensors", lambda *a: {})
    rt = SimpleNamespace(device="cpu")
    same, four = model.LoadedModel(plan, None, rt), model.LoadedModel(plan, None, rt, four_bits=True)
    # entries 0, 1, 2, 5 need the same; entry 4 has a window
    assert [(g.n_layers, g.spec.window) for g in same.groups] == [(4, None), (1, 9)]
    assert [(lay.group, lay.layer_in_group) for lay in same.layers] == [(0, 0), (0, 1), (0, 2), (0, 2), (1, 0), (0, 3), (-1, -1), (0, 1), (0, 3)]
    assert [(g.n_layers, g.spec.window, g.four_bits) for g in four.groups] == [(2, None, True), (2, None, False), (1, 9, True)]
    assert [lay.group for lay in four.layers] == [0, 1, 1, 1, 2, 0, -1, 1, 0]
    assert same.kv_bytes_per_token(2) == 5 * 2 * 256 and four.kv_bytes_per_token(2, True) == 3 * 2 * 72 + 2 * 2 * 256


def test_the_plain_implementation_has_no_cache_to_keep_in_four_bits(tmp_path, capsys):
    import tiny
    from xyntetik_runner_b200.cli import main
    folder = tiny.make_folder(str(tmp_path / "a"), "A")
    assert main(["-m", folder, "-p", "ids:7,8", "-n", "2", "--ref", "--kv", "int4"]) == 2
    said = capsys.readouterr()
    assert "--kv int4" in said.err and said.out == ""
    assert main(["-m", folder, "-p", "ids:7,8", "-n", "2", "--ref", "--kv", "same", "--ignore-eos"]) == 0


def test_lengths_that_are_no_arrays():
    """Lists, tensors, one array alone: refused as what they are, not by what they lack."""
    a = np.array([1, 2], dtype=np.int32)
    for l, p in (([1, 2], [0, 0]), (torch.tensor([1, 2], dtype=torch.int32), torch.zeros(2, dtype=torch.int32)), (a, [0, 0]), (None, None)):
        with pytest.raises(kernels.KernelError, match="two int32 numpy arrays"):
            kernels.kv4_plan((l, p), 9, 2, 4, 64, 16, kernels.BF16, 0, 0, 64)
