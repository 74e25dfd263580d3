"""An engine whose cache is in four bits against an engine that keeps rows in the activations' type and whose pages are quantised by the plain form
between store and attention; steps in graphs and without, cut in every way; generation through the entry points."""
import json
import math
import os
import subprocess
import sys

import numpy as np
import pytest
import torch

import plain_kv4

pytestmark = pytest.mark.gpu
ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))

DENSE = {"kind": "dense", "ff": 64}
MOE = {"kind": "moe", "router": {"experts": 2, "top": 2}, "expert": {"ff": 64}, "shared": {"ff": 64}}


def llama(head_dim=64, heads=8, kv_heads=2, layers=2, window=None):
    d = {"architectures": ["LlamaForCausalLM"], "hidden_size": 256, "num_hidden_layers": layers, "num_attention_heads": heads,
         "num_key_value_heads": kv_heads, "head_dim": head_dim, "intermediate_size": 320, "vocab_size": 300, "rms_norm_eps": 1e-5, "rope_theta": 10000.0,
         "max_position_embeddings": 4096, "tie_word_embeddings": False, "torch_dtype": "bfloat16"}
    return d


def besolix():
    """Attention with a norm a head, values of another size, a window; the latent layer keeps its rows as they are."""
    at = dict(heads=4, kv_heads=2, dim=64, vdim=48, scale=0.15, rot={"base": 10000.0, "dims": 32}, mask={"size": 70})
    la = dict(heads=2, dim=32, rot_dim=16, vdim=32, kv_rank=64, q_rank=48, scale=0.15, rot={"base": 10000.0, "dims": 16}, mask={"size": 90})
    return {"architecture": "Besolix", "vocab": 300, "width": 128, "norm": {"eps": 1e-5},
            "layers": [{"type": "attention", "mlp": DENSE, "mixer": at}, {"type": "latent_attention", "mlp": DENSE, "mixer": la},
                       {"type": "attention", "mlp": DENSE, "mixer": dict(at, dim=128, vdim=128, rot={"base": 10000.0, "dims": 128})}]}


def tiny(module, name):
    import importlib
    return importlib.import_module("tiny_" + module).CONFIGS[name]


def semesun():
    """Windows with kept first keys, a bias by distance, values that layers share."""
    import tiny_semesun as t
    return t.clean(t.model(160, 128, 1e-5, [t.layer(t.attention(4, 2, 64, 64, 0.12, 70, 5, 48, 32, True), DENSE),
                                            t.layer(t.attention(2, 1, 128, 128, 0.09, 130, 140, 200, 32, True), DENSE),
                                            t.layer(t.attention(16, 2, 64, 48, 0.15, 33, 1, 20, 32), None),
                                            t.layer(t.attention(3, 3, 24, 20, 0.2, None, 0, 90, 32), DENSE)]))


MODELS = {"llama64": llama, "llama128": lambda: llama(128, 6, 2), "llama100": lambda: llama(100, 3, 1), "mqa": lambda: llama(64, 18, 1), "wide": lambda: llama(64, 128, 32),
          "besolix": besolix, "pitolix": lambda: tiny("pitolix", "mix"), "buzarax": lambda: tiny("buzarax", "mix"), "semesun": semesun,
          "lilalorn": lambda: tiny("lilalorn", "mix")}


def engine(model, dtype, kv, page_size=16, graphs=True, requests=4, max_tokens=2048):
    from xyntetik_runner_b200 import architectures  # noqa: F401
    from xyntetik_runner_b200.config import registry
    from xyntetik_runner_b200.engine.engine import EngineParams, random_engine
    c = MODELS[model]()
    arch = registry.resolve(registry.architecture_name(c))
    return random_engine(arch.config_from_dict(c), 7, EngineParams(dtype=dtype, max_tokens=max_tokens, page_size=page_size, max_requests=requests,
                                                                   max_request_tokens=512, max_step_tokens=512, cuda_graphs=graphs, kv=kv), std=0.08)


STEPS = [  # request -> tokens of each step
    {"a": 1, "b": 37}, {"a": 5, "b": 1, "c": 90}, {"a": 1, "b": 1, "c": 1}, {"a": 1, "b": 1, "c": 1}, {"a": 1, "b": 1, "c": 1}, {"b": 3, "c": 64}, {"a": 1, "c": 1}]


def run(eng, steps=STEPS, vocab=250):
    from xyntetik_runner_b200.engine.engine import StepEntry
    rng = np.random.RandomState(3)
    out = []
    for st in steps:
        entries = [StepEntry(r, [int(t) for t in rng.randint(0, vocab, n)], list(range(n))) for r, n in st.items()]
        out.append(eng.step(entries).clone())
    eng.check_status()
    return out


def quantise_pages(eng, monkeypatch):
    """Before every attention of this engine, all rows in its pages become the values that four bits hold (which leaves values that are held already as
    they are)."""
    from xyntetik_runner_b200 import kernels

    def behind(fn):
        def call(*a, **k):
            for t, g in zip(eng.kv, eng.model.groups):
                if g.four_bits:
                    t.copy_(plain_kv4.quantised_rows(t).to(t.dtype))
            return fn(*a, **k)
        return call
    for name in ("attention_simt", "attention_mma", "attention_tc"):
        monkeypatch.setattr(kernels, name, behind(getattr(kernels, name)))


def record_choices(monkeypatch, given=None):
    """A list that receives the logits by which each token of each routed layer chooses its experts, call by call (a choice of few tokens is left to the same
    kernels).  `given`: such a list of another run, by whose logits the choices are then made."""
    from xyntetik_runner_b200 import kernels
    from xyntetik_runner_b200.parts import moe
    monkeypatch.setattr(moe, "FEW_TOKENS", 0)
    said = []

    def ahead(fn):
        def call(z, *a, **k):
            said.append(z.clone())
            if given is not None:
                z.copy_(given[len(said) - 1])
            return fn(z, *a, **k)
        return call
    for name in ("route_topk", "route_groups"):
        monkeypatch.setattr(kernels, name, ahead(getattr(kernels, name)))
    return said


def rows_of(eng, request):
    return [torch.stack(eng.cached_rows(request, lay.entry)) for lay in eng.model.layers if lay.group >= 0 and eng.model.groups[lay.group].four_bits and lay.writes_cache]


@pytest.mark.parametrize("dtype", ["float32", "bfloat16"])
@pytest.mark.parametrize("model", list(MODELS))
def test_engine_against_quantised_pages(model, dtype, monkeypatch):
    """Rows: the first layer's are those of the plain form, bit for bit; the others' differ where a rounding ahead of them took a value to the other side of a
    border between two codes (float32: none to a few in 100,000).  Logits: as near as the arithmetic is where no row differs.  A choice of experts may hang on
    a rounding: both engines choose by the first one's logits, and the second's are compared with them."""
    from xyntetik_runner_b200.parts import attention
    eng = engine(model, dtype, "int4", graphs=model not in ("buzarax", "lilalorn"))
    vocab = min(250, eng.plan.vocab_size)
    before = attention.counters["kv4"]
    with monkeypatch.context() as m:
        mine = record_choices(m)
        got = run(eng, vocab=vocab)
    assert attention.counters["kv4"] > before and any(eng.four_bits)
    rows = {r: rows_of(eng, r) for r in "abc"}
    ref = engine(model, dtype, "same", graphs=False)
    with monkeypatch.context() as m:
        theirs = record_choices(m, mine)
        quantise_pages(ref, m)
        want = run(ref, vocab=vocab)
    assert len(mine) == len(theirs) and (mine or model not in ("buzarax", "lilalorn"))
    differ = total = 0
    for r in "abc":
        for i, (x, y) in enumerate(zip(rows[r], rows_of(ref, r))):
            assert x.shape == y.shape and x.abs().max() > 0
            if i == 0 and model.startswith(("llama", "mqa", "wide")):
                assert torch.equal(x, y)                             # (the first layer's input is the embedding)
            differ += int((x != y).sum())
            total += x.numel()
            assert float((x - y).abs().max()) <= 0.6 * float(y.abs().max())
    assert differ <= (1e-4 if dtype == "float32" else 0.1) * total, f"{differ} of {total}"
    for a, b in [*zip(got, want), *zip(mine, theirs)]:
        scale, off = float(b.abs().max()), float((a - b).abs().max())
        if dtype == "float32":
            assert off <= (1e-4 if differ == 0 else 0.02) * scale, f"{off / scale:.3g}"
        else:
            # bfloat16 activations differ by their rounding, and a value near a border between two codes may fall on its other side: one step, an eighth of
            # its group's largest magnitude, 0.31 of the values' size where that is 2.5 of it (32 normal values: 2.2 on average).  A share f of such values is
            # an error of 0.31 sqrt(f) in keys and in values of every layer, independent of one another; beside it 2^-6 for the roundings
            # of the products, norms and weights along two to four layers.
            rel = float((a - b).norm() / b.norm())
            most = 2.0 ** -6 + 0.31 * math.sqrt(differ / total * 2 * len(rows["a"]))
            assert off <= 0.1 * scale and rel <= most, f"{rel:.3g} of {most:.3g}, {differ} of {total}"


def test_first_layers_rows_are_the_plain_forms():
    """What four bits hold of the rows that an engine without them keeps."""
    for dtype in ("float32", "bfloat16"):
        four, same = engine("llama64", dtype, "int4"), engine("llama64", dtype, "same")
        run(four), run(same)
        for r in "abc":
            for x, y in zip(four.cached_rows(r, 0), same.cached_rows(r, 0)):
                n = y.shape[0] * y.shape[1]
                assert torch.equal(x.double().cpu().reshape(n, -1), plain_kv4.quantised(y.reshape(n, -1))[2])


@pytest.mark.parametrize("model", ["llama64", "semesun"])
def test_graphs_and_plain_steps_give_the_same_bits(model):
    steps = [{"a": 40, "b": 7}] + [{"a": 1, "b": 1}] * 6
    a, b = engine(model, "bfloat16", "int4", graphs=True), engine(model, "bfloat16", "int4", graphs=False)
    x, y = run(a, steps), run(b, steps)
    if a._graph_ok:
        assert a.graph_replays > 0
    assert all(torch.equal(p, q) for p, q in zip(x, y))


@pytest.mark.parametrize("model", ["llama64", "wide"])
def test_cutting_a_request_changes_little(model):
    """A prompt in one portion (with many heads read back for the prompt kernel), in portions that attend to the codes, token by token: the same logits within
    the activations' rounding; the first layer's rows in the cache are the plain form's of an engine that keeps them as they are, cut alike."""
    for dtype, tol in (("float32", 1e-4), ("bfloat16", 0.05)):
        ref = None
        for cut in ([96], [40, 56], [16] * 6, [5] * 19 + [1], [1] * 96):
            eng, same = engine(model, dtype, "int4"), engine(model, dtype, "same")
            x = torch.cat(run(eng, [{"a": n} for n in cut]))
            run(same, [{"a": n} for n in cut])
            for got, rows in zip(eng.cached_rows("a", 0), same.cached_rows("a", 0)):
                n = rows.shape[0] * rows.shape[1]
                assert torch.equal(got.double().cpu().reshape(n, -1), plain_kv4.quantised(rows.reshape(n, -1))[2])
            ref = x if ref is None else ref
            assert float((x - ref).abs().max()) <= tol * float(ref.abs().max())


def test_a_window_gives_pages_back_and_reads_zeros():
    eng = engine("besolix", "bfloat16", "int4")
    run(eng, [{"a": 120}] + [{"a": 1}] * 60)
    free = [p.n_free for p in eng.cache.pools]
    assert max(free) > 0
    k, v = eng.cached_rows("a", 0)
    assert k.shape[0] == 180 and not k[:64].any() and k[-70:].abs().amax(dim=(1, 2)).min() > 0
    eng.end("a")
    eng.cache.audit()
    eng._open("new")
    assert all(x.shape == (0, 2, 64) for x in eng.cached_rows("new", 0))
    with pytest.raises(ValueError, match="one row a token"):
        eng.cached_rows("new", 1)


@pytest.mark.parametrize("dtype", ["bfloat16", "float32"])
def test_generate_and_score(dtype):
    """Through the runner: many requests in a small pool give every request the tokens that it gets alone; a score."""
    from xyntetik_runner_b200 import Runner
    from xyntetik_runner_b200.config import registry
    c = llama()
    cfg = registry.resolve(registry.architecture_name(c)).config_from_dict(c)
    rng = np.random.RandomState(2)
    prompts = [[int(t) for t in rng.randint(0, 300, n)] for n in (3, 70, 150, 12)]
    r = Runner(config=cfg, random_seed=3, dtype=dtype, ctx=256, batch=96, parallel=4, kv="int4", page_size=32)
    together = r.generate(prompts, n=12, ignore_eos=True)
    assert all(len(x.tokens) == 12 for x in together)
    if dtype == "float32":
        for p, x in zip(prompts, together):
            assert r.generate(p, n=12, ignore_eos=True).tokens == x.tokens
    lp = r.score(prompts[1])
    assert len(lp) == 69 and all(np.isfinite(lp))
    same = Runner(config=cfg, random_seed=3, dtype=dtype, ctx=256, batch=96, parallel=4, page_size=32)
    assert np.corrcoef(lp, same.score(prompts[1]))[0, 1] > 0.9       # four bits are near what they hold
    assert r.engine.kv_bytes_per_token() * 3.5 < same.engine.kv_bytes_per_token()
    assert r.engine.kv_bytes_per_token() == 2 * 2 * 72


def test_command_line(tmp_path):
    path = tmp_path / "m"
    path.mkdir()
    (path / "config.json").write_text(json.dumps(llama()))
    cmd = [sys.executable, "-m", "xyntetik_runner_b200", "-m", str(path), "--random", "5", "-p", "ids:1,5,9", "-n", "5", "--ignore-eos", "-c", "128", "--kv", "int4"]
    a = subprocess.run(cmd, cwd=ROOT, capture_output=True, text=True, timeout=300)
    assert a.returncode == 0, a.stderr
    assert a.stdout.startswith("ids:") and len(a.stdout.split("\n")[0].split(",")) == 5


def long_engine(dtype, kv, layers, graphs, model="llama", max_tokens=6144):
    from xyntetik_runner_b200 import architectures  # noqa: F401
    from xyntetik_runner_b200.config import registry
    from xyntetik_runner_b200.engine.engine import EngineParams, random_engine
    c = llama(128, 6, 2, layers=layers) if model == "llama" else MODELS[model]()
    arch = registry.resolve(registry.architecture_name(c))
    return random_engine(arch.config_from_dict(c), 7, EngineParams(dtype=dtype, max_tokens=max_tokens, page_size=64, max_requests=4, max_request_tokens=4096,
                                                                   max_step_tokens=1024, cuda_graphs=graphs, kv=kv), std=0.08)


def long_run(eng, vocab=250):
    """Three requests of 300 to 3,000 tokens and a fourth that takes the second's pages; single tokens, a few, and none but one request's, in between."""
    from xyntetik_runner_b200.engine.engine import StepEntry
    rng = np.random.RandomState(5)
    out = []

    def step(**tokens):
        entries = [StepEntry(r, [int(t) for t in rng.randint(0, vocab, n)], list(range(max(0, n - 3), n))) for r, n in tokens.items()]
        out.append(eng.step(entries).clone())
    step(a=1000), step(a=900, b=100), step(a=1000, b=24), step(b=900), step(c=300)
    for _ in range(6):
        step(a=1, b=1, c=1)
    step(a=4, b=1, c=2)
    pages = set(eng.cache.block_table(0, "b").tolist()) - {-1}
    eng.end("b")
    step(d=1000), step(a=1, d=30)
    assert set(eng.cache.block_table(0, "d").tolist()) & pages        # (pages of the one that ended)
    for _ in range(6):
        step(a=1, c=1, d=1)
    for r in "ac":
        step(**{r: 1}), step(**{r: 1}), step(**{r: 1})
    eng.check_status()
    return out


@pytest.mark.parametrize("dtype", ["float32", "bfloat16"])
@pytest.mark.parametrize("layers,graphs", [(1, True), (1, False), (2, True)])
def test_long_requests_against_quantised_pages(dtype, layers, graphs, monkeypatch):
    """Requests whose keys are cut into spans that meet in a cluster or through a second kernel, read ahead of the kernel before.  One layer: its rows are the plain
    form's bit for bit, so that logits are as near as the arithmetic (float32: 1e-4 of the largest, which a span that is lost or read too soon is not)."""
    from xyntetik_runner_b200 import kernels
    cuts, real = set(), kernels.kv4_plan

    def plan(*a, **k):
        said = real(*a, **k)
        if said[0]:
            cuts.add((said[12] > 1, bool(said[13])))
        return said
    eng = long_engine(dtype, "int4", layers, graphs)
    with monkeypatch.context() as m:
        m.setattr(kernels, "kv4_plan", plan)
        got = long_run(eng)
    assert {(True, True), (True, False)} <= cuts and (eng.graph_replays > 0) == graphs
    ref = long_engine(dtype, "same", layers, False)
    with monkeypatch.context() as m:
        quantise_pages(ref, m)
        want = long_run(ref)
    differ = total = 0
    for r in "acd":
        for i, (x, y) in enumerate(zip(rows_of(eng, r), rows_of(ref, r))):
            assert x.shape == y.shape and (i > 0 or torch.equal(x, y))
            differ, total = differ + int((x != y).sum()), total + x.numel()
    assert differ <= (0 if layers == 1 else 1e-4 * total if dtype == "float32" else 0.1 * total)
    for a, b in zip(got, want):
        scale, off = float(b.abs().max()), float((a - b).abs().max())
        if dtype == "float32":
            assert off <= (1e-4 if differ == 0 else 0.02) * scale, f"{off / scale:.3g}"
        else:
            # (see test_engine_against_quantised_pages)
            rel = float((a - b).norm() / b.norm())
            assert rel <= 2.0 ** -6 + 0.31 * math.sqrt(differ / total * 2 * layers), f"{rel:.3g}, {differ} of {total}"
    if graphs:
        plain = long_run(long_engine(dtype, "int4", layers, False))
        for a, b in zip(got, plain):
            # (the same kernels, cut for other lengths at times: sums in another order)
            assert float((a - b).abs().max()) <= (1e-4 if dtype == "float32" else 0.05) * float(b.abs().max())


@pytest.mark.parametrize("dtype", ["float32", "bfloat16"])
def test_batches_that_are_filled_up(dtype, monkeypatch):
    """Eleven requests of 1 to 300 tokens: decode steps are filled up to sixteen rows, captured and replayed; what the filling rows leave is nobody's."""
    from xyntetik_runner_b200.engine.engine import StepEntry

    def go(eng):
        rng, out = np.random.RandomState(9), []
        lens = [1, 300, 17, 64, 65, 128, 9, 250, 33, 2, 100]
        for r, n in enumerate(lens):
            out.append(eng.step([StepEntry(r, [int(t) for t in rng.randint(0, 250, n)], [n - 1])]).clone())
        for _ in range(6):
            out.append(eng.step([StepEntry(r, [int(rng.randint(0, 250))], [0]) for r in range(len(lens))]).clone())
        eng.check_status()
        return out
    four, plain, ref = (engine("llama64", dtype, kv, graphs=graphs, requests=12, max_tokens=4096) for kv, graphs in (("int4", True), ("int4", False), ("same", False)))
    got, unfilled = go(four), go(plain)
    assert four.graph_replays > 0 and four._fill_ok and plain.graph_replays == 0
    with monkeypatch.context() as m:
        quantise_pages(ref, m)
        want = go(ref)
    for a, b, c in zip(got, unfilled, want):
        assert a.shape == c.shape
        scale = float(c.abs().max())
        # (a value on the other side of a border between two codes: see test_engine_against_quantised_pages)
        assert float((a - b).abs().max()) <= (0.02 if dtype == "float32" else 0.1) * scale
        assert float((a - c).abs().max()) <= (0.02 if dtype == "float32" else 0.1) * scale
    assert four.cached_rows(1, 0)[0].shape[0] == 306 and torch.equal(four.cached_rows(1, 0)[0], ref.cached_rows(1, 0)[0])
