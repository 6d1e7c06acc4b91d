"""The engine over a cache of 8 bits: its options, its pages, its steps with the plain forms of the kernels on the CPU, and on the GPU with
the kernels against those."""
import pytest
import torch

import helpers
import kernel_twins
import plain_qwen3
from e4m3_cases import PlainOps
from mini_engine_amd import LLM, SamplingParams
from mini_engine_amd.cache.manager import CacheManager
from mini_engine_amd.cache.pool import page_bytes
from mini_engine_amd.config.engine_config import EngineConfig
from mini_engine_amd.config.model_config import ConfigError
from mini_engine_amd.engine.runner import ModelRunner
from mini_engine_amd.kernels import ops
from mini_engine_amd.parts.attention import Attention
from mini_engine_amd.parts.base import PAGE, PageTensor
from mini_engine_amd.weights.loader import load_model


class Plain(PlainOps, kernel_twins.PlainBackend):
    pass


@pytest.fixture
def plain():
    ops.set_backend(Plain())
    PlainOps.calls = 0
    yield
    ops.set_backend(None)


def _runner(folder, device, kind, pages=40, page=16, graphs=False, most=512):
    model = load_model(folder, device, torch.bfloat16, most)
    model.hold_keys_and_values_in(kind)
    manager = CacheManager(pages, page, ModelRunner.windows_of(model), enable_prefix_caching=False)
    options = dict(use_graphs=True, mixed_graphs_after=0, mixed_graphs_max_tokens=4096) if graphs else {}
    return ModelRunner(model, manager, torch.bfloat16, device, most, poison_cache=True, **options), manager


def _feed(runner, manager, ids, cuts):
    """Requests in portions: cuts[r] are the sizes of request r's portions, one a step; float32 logits of all tokens, by request."""
    d = helpers.Driver(runner, manager)
    at = {r: 0 for r in ids}
    for i in range(max(len(c) for c in cuts.values())):
        step = {r: ids[r][at[r]:at[r] + cuts[r][i]] for r in ids if i < len(cuts[r])}
        for r in step:
            at[r] += len(step[r])
        d.step(step)
    return {r: d.result(r) for r in ids}


def _requests(vocab):
    lens = {"a": 70, "b": 9, "c": 33}
    ids = {r: helpers.random_ids(n, vocab, 50 + i) for i, (r, n) in enumerate(lens.items())}
    return ids, {"a": [40, 1, 1, 20, 1, 7], "b": [1, 3, 1, 1, 3], "c": [16, 16, 1]}


# ------------------------------------------------------------------ options and pages

def test_options(folders):
    config = EngineConfig(folders("A"), kv_cache_dtype="e4m3")
    assert config.kv_cache_dtype == "e4m3" and EngineConfig(folders("A")).kv_cache_dtype == "auto"
    for wrong in (dict(kv_cache_dtype="int8"), dict(kv_cache_dtype="e4m3", dtype="float32"), dict(kv_cache_dtype="e4m3", kvcache_block_size=8),
                  dict(kv_cache_dtype="e4m3", kvcache_block_size=48)):
        with pytest.raises(ConfigError):
            EngineConfig(folders("A"), **wrong)


def test_pages_in_half_the_bytes(folders):
    model = load_model(folders("A"), "cpu", torch.bfloat16, 64)
    full = sum(page_bytes(model.cache_plan(), 32, torch.bfloat16))
    model.hold_keys_and_values_in("e4m3")
    need = model.cache_plan().group_needs[0]
    assert [(t.name, t.sized(32), t.dtype) for t in need.tensors] == [
        ("k", (2, 32, 16), "e4m3"), ("v", (2, 16, 32), "e4m3"), ("k_scales", (2, 2), "uint8"), ("v_scales", (2, 2), "uint8")]
    # layers x (keys, values) x (heads x page x head size bytes, and a byte for every block and head)
    assert sum(page_bytes(model.cache_plan(), 32, torch.bfloat16)) == 2 * 2 * (2 * 32 * 16 + 2 * 2) == full // 2 + 2 * 2 * 2 * 2
    model.hold_keys_and_values_in("compute")
    assert sum(page_bytes(model.cache_plan(), 32, torch.bfloat16)) == full
    with pytest.raises(ValueError, match="multiple"):
        PageTensor("s", (2, PAGE), "uint8", 16).sized(24)


@pytest.mark.parametrize("options,what", [(dict(qkv_bias=True), "biases"), (dict(window=8, keep_first=2), "kept behind"), (dict(score_cap=5.0), "cap"),
                                          (dict(slopes=[0.1, 0.2]), "slopes")])
def test_attention_without_such_a_form_is_refused(options, what):
    mixer = Attention(32, 2, 2, 16, 0.25, **options)
    with pytest.raises(ValueError, match=what):
        mixer.hold_in("e4m3")
    assert mixer.pages_hold == "compute"
    with pytest.raises(ValueError, match="head sizes"):
        Attention(32, 2, 2, 24, 0.25).hold_in("e4m3")
    with pytest.raises(ValueError, match="pages hold"):
        Attention(32, 2, 2, 16, 0.25).hold_in("int8")


def test_models_without_such_a_form_are_refused(tmp_path):
    """Negosun's attention norms whole projections; the entry point says which option asked for what."""
    import negosun_cases
    name = next(iter(negosun_cases.CONFIGS))
    folder = negosun_cases.make_folder(name, str(tmp_path))
    with pytest.raises(ConfigError, match="kv_cache_dtype 'e4m3': layer 0"):
        LLM(folder, dtype="bfloat16", device="cpu", kv_cache_dtype="e4m3", num_kvcache_blocks=8, max_num_seqs=2, max_num_batched_tokens=16, max_model_len=16)


# ------------------------------------------------------------------ steps

def _rms(x):
    return float(x.double().pow(2).mean().sqrt())


@pytest.mark.parametrize("name", ["A", "C"])
def test_steps_on_the_cpu(folders, plain, name):
    """Every cut of the requests, a window among the layers: near the bfloat16 cache's logits by what 4 digits cost."""
    ids, cuts = _requests(helpers.CONFIGS[name]["vocab_size"])
    got = _feed(*_runner(folders(name), "cpu", "e4m3"), ids, cuts)
    assert PlainOps.calls == 6 * helpers.CONFIGS[name]["num_hidden_layers"]
    full = _feed(*_runner(folders(name), "cpu", "compute"), ids, cuts)
    for r in ids:
        plainly = helpers.plain_logits(folders(name), ids[r])
        assert torch.isfinite(got[r]).all()
        # a rounding to 4 digits is off by 2^-4 at most and 0.6 of half of that on average; keys and values of every layer bring one each,
        # their errors add up over the layers as squares at worst with a gain of 1: sqrt(2 * 4 layers) * 2^-4 * 0.6 = 0.11
        assert _rms(got[r] - plainly) <= 0.11 * _rms(plainly) + _rms(full[r] - plainly)
    # another way of cutting them: the blocks fill in other steps
    other = _feed(*_runner(folders(name), "cpu", "e4m3"), ids, {r: [len(ids[r])] for r in ids})
    for r in ids:
        assert _rms(other[r] - got[r]) <= 2 * 0.11 * _rms(got[r])


def test_generation_on_the_cpu(folders, plain):
    """Through the entry point: prefix caching, preemption by a small pool, run to the end with the tokens of requests that run alone."""
    prompts = [helpers.random_ids(n, 256, 7 + n) for n in (5, 37, 33)]
    options = dict(dtype="bfloat16", device="cpu", kv_cache_dtype="e4m3", max_num_seqs=4, max_num_batched_tokens=32, max_model_len=64, poison_cache=True)
    llm = LLM(folders("A"), num_kvcache_blocks=9, **options)
    assert llm.runner.pool.tensors[0]["k"].dtype == torch.float8_e4m3fn
    outs = llm.generate(prompts, SamplingParams(temperature=0, max_tokens=6), use_tqdm=False)
    again = llm.generate(prompts, SamplingParams(temperature=0, max_tokens=6), use_tqdm=False)
    assert [len(o["token_ids"]) for o in outs] == [6, 6, 6] and all(len(o["token_ids"]) == 6 for o in again)


def _evicted_and_refed(folder, vocab, lens, tokens, pages, **options):
    """A pool that is too small for all requests: some are evicted and fed again, into blocks that others held before; a second run finds the first
    one's full pages. Every token is the plain model's best, or lies within what 8 bits cost of it, and is the one that the request gets
    alone in a cache of its own, up to a first place where the plain model's logits of the two lie as near to each other."""
    prompts = [helpers.random_ids(n, vocab, 7 + n) for n in lens]
    params = SamplingParams(temperature=0, max_tokens=tokens)
    run = lambda llm, p: [o["token_ids"] for o in llm.generate(p, params, use_tqdm=False)]  # noqa: E731
    tight = LLM(folder, num_kvcache_blocks=pages, kv_cache_dtype="e4m3", dtype="bfloat16", poison_cache=True, **options)
    first = run(tight, prompts)
    assert tight.scheduler.num_preemptions > 0, "nobody was evicted"
    before = tight.scheduler.num_prefix_hits
    again = run(tight, prompts)
    assert tight.scheduler.num_prefix_hits > before, "no page was found again"
    cfg, w = plain_qwen3.read_model_folder(folder, torch.float64)
    for i, p in enumerate(prompts):
        own = LLM(folder, num_kvcache_blocks=64, kv_cache_dtype="e4m3", dtype="bfloat16", poison_cache=True, enable_prefix_caching=False, **options)
        alone = run(own, [p])[0]
        assert own.scheduler.num_preemptions == 0 and len(alone) == tokens
        for out in (first[i], again[i]):
            assert len(out) == tokens
            z = plain_qwen3.logits(cfg, w, p + out)
            same = True
            for j, tok in enumerate(out):
                row = z[len(p) + j - 1]
                near = 2 * 0.11 * 3 * _rms(row)           # two logits, each off by 0.11 of the logits' size on average (above), three times that at most
                assert float(row.max() - row[tok]) <= near, (i, j)
                if same and tok != alone[j]:
                    assert abs(float(row[alone[j]] - row[tok])) <= near, (i, j)
                    same = False


def test_evicted_requests_on_the_cpu(folders, plain):
    _evicted_and_refed(folders("A"), 256, (5, 37, 33), 20, 6, device="cpu", max_num_seqs=4, max_num_batched_tokens=32, max_model_len=64)


# Configurations of the other designs: None where all their attention has the 8-bit form, else why they are refused.
DESIGNS = {("sigosun_cases", n): None for n in ("mix", "odd", "att", "far", "real")} | {
    ("goluzen_cases", "one"): None, ("tavevik_cases", "two"): None, ("goluzen_cases", "real"): "kept behind a window", ("goluzen_cases", "routed"): "cap",
    ("tavevik_cases", "real"): "kept behind a window", ("tavevik_cases", "odd"): "kept behind a window", ("venezen_cases", "real"): "slopes",
    ("venezen_cases", "windows"): "slopes", ("negosun_cases", "real"): "whole projections", ("vefulix_cases", "real"): "nothing to hold",
    ("sigosun_cases", "ssm"): "nothing to hold"}


@pytest.mark.parametrize("module,name", list(DESIGNS), ids=lambda x: x)
def test_designs_that_have_the_form(tmp_path, module, name):
    import importlib
    model = load_model(importlib.import_module(module).make_folder(name, str(tmp_path / "model")), "cpu", torch.bfloat16, 64)
    lacks = DESIGNS[module, name]
    if lacks:
        with pytest.raises(ValueError, match=lacks):
            model.hold_keys_and_values_in("e4m3")
        return
    model.hold_keys_and_values_in("e4m3")
    kept = [t.dtype for need in model.cache_plan().group_needs for t in need.tensors]
    assert "e4m3" in kept and kept.count("e4m3") == kept.count("uint8")


@pytest.mark.parametrize("name", ["pair", "real"])
def test_a_refused_model_is_left_as_it_was(tmp_path, name):
    """Tavevik's first attention layer has the form, its second one has not."""
    import tavevik_cases
    model = load_model(tavevik_cases.make_folder(name, str(tmp_path / "model")), "cpu", torch.bfloat16, 64)
    before = model.cache_plan().group_needs
    with pytest.raises(ValueError, match="layer 1: .*no keys kept behind a window"):
        model.hold_keys_and_values_in("e4m3")
    assert model.cache_plan().group_needs == before


# ------------------------------------------------------------------ on the GPU

@pytest.mark.gpu
@pytest.mark.parametrize("graphs", [False, True], ids=["eager", "graphs"])
@pytest.mark.parametrize("name", ["A", "C", "R"])
def test_steps_on_the_gpu(folders, name, graphs):
    """The kernels' steps against the plain forms' on the same GPU tensors. The two differ by bfloat16's roundings in front of the cache, which
    make some stored numbers fall to the other side of a border: 2^-8 of a number in a step of 2^-3 of it, one in 16 at most, a step each:
    sqrt(1 / 16) * 2^-3 = 0.03 of a number's size on average, half of what storing it costs; both bounds of the CPU's test follow."""
    ids, cuts = _requests(helpers.CONFIGS[name]["vocab_size"])
    got = _feed(*_runner(folders(name), "cuda", "e4m3", graphs=graphs), ids, cuts)
    ops.set_backend(Plain())
    try:
        expect = _feed(*_runner(folders(name), "cuda", "e4m3"), ids, cuts)
        full = _feed(*_runner(folders(name), "cuda", "compute"), ids, cuts)
    finally:
        ops.set_backend(None)
    for r in ids:
        cost = _rms(expect[r] - full[r])
        assert torch.isfinite(got[r]).all()
        assert _rms(got[r] - expect[r]) <= cost + helpers.TOL_BF16 * _rms(full[r])
        plainly = helpers.plain_logits(folders(name), ids[r])
        assert _rms(got[r] - plainly) <= 0.11 * _rms(plainly) + helpers.TOL_BF16 * float(plainly.abs().max())


@pytest.mark.gpu
def test_generation_on_the_gpu(folders):
    """Captured decode steps, run ahead, prompts in portions; a pool sized from memory holds twice the pages. The libraries are the kernels' own."""
    prompts = [helpers.random_ids(n, 2048, 7 + n) for n in (5, 300, 33, 90)]
    options = dict(dtype="bfloat16", max_num_seqs=4, max_num_batched_tokens=128, max_model_len=512)
    llm = LLM(folders("R"), kv_cache_dtype="e4m3", num_kvcache_blocks=128, poison_cache=True, **options)
    outs = llm.generate(prompts, SamplingParams(temperature=0, max_tokens=20), use_tqdm=False)
    cfg, w = plain_qwen3.read_model_folder(folders("R"), torch.float64)
    for p, o in zip(prompts, outs):
        z = plain_qwen3.logits(cfg, w, p + o["token_ids"])
        assert len(o["token_ids"]) == 20
        for i, tok in enumerate(o["token_ids"]):
            row = z[len(p) + i - 1]
            # another token than the plain model's best only where the two lie within what 8 bits cost (twice the bound above: both may move)
            assert float(row.max() - row[tok]) <= 2 * 0.11 * 3 * _rms(row)
    assert any("libme_attn8_d128.so" in path for path in ops.loaded_libraries())


@pytest.mark.gpu
def test_other_designs_on_the_gpu(tmp_path):
    """Layers of other designs beside recurrences, windows, sinks, block masks, output gates and shared caches: those whose attention has the form run
    with it, in steps of every kind, and their logits stay near the bfloat16 cache's."""
    import goluzen_cases
    import sigosun_cases
    ran = 0
    for cases in (sigosun_cases, goluzen_cases):
        for name in list(cases.CONFIGS)[:2]:
            folder = cases.make_folder(name, str(tmp_path / f"{cases.__name__}_{name}"))
            found = {}
            try:
                for kind in ("e4m3", "compute"):
                    model = load_model(folder, "cuda", torch.bfloat16, 256)
                    model.hold_keys_and_values_in(kind)
                    manager = CacheManager(40, 16, ModelRunner.windows_of(model), num_state_slots=4, enable_prefix_caching=False)
                    runner = ModelRunner(model, manager, torch.bfloat16, "cuda", 256, poison_cache=True)
                    ids, cuts = _requests(model.embedding.vocab_size)
                    found[kind] = _feed(runner, manager, ids, cuts)
            except ValueError as e:
                assert "8-bit cache" in str(e) or "nothing to hold" in str(e)
                continue
            ran += 1
            for r in ids:
                assert torch.isfinite(found["e4m3"][r]).all()
                assert _rms(found["e4m3"][r] - found["compute"][r]) <= 0.3 * _rms(found["compute"][r])
    assert ran >= 1


@pytest.mark.gpu
def test_evicted_requests_on_the_gpu(folders):
    """Captured steps, run ahead, beside portions: the blocks that a step writes ahead of a request's end are others' soon after."""
    _evicted_and_refed(folders("R"), 2048, (5, 130, 33, 90), 40, 16, max_num_seqs=4, max_num_batched_tokens=64, max_model_len=256)


@pytest.mark.gpu
@pytest.mark.parametrize("module,name", [k for k, lacks in DESIGNS.items() if not lacks], ids=lambda x: x)
def test_designs_steps_on_the_gpu(tmp_path, module, name):
    """The kernels' steps against the plain forms' on the CPU. Two runs whose stored numbers were rounded with nothing to do with each
    other would differ by sqrt(2) of what storing costs; bfloat16's roundings in front of the cache cannot take them further apart."""
    import importlib
    folder = importlib.import_module(module).make_folder(name, str(tmp_path / "model"))

    def logits(kind, device):
        model = load_model(folder, device, torch.bfloat16, 256)
        model.hold_keys_and_values_in(kind)
        manager = CacheManager(40, 16, ModelRunner.windows_of(model), num_state_slots=4, enable_prefix_caching=False)
        ids, cuts = _requests(model.embedding.vocab_size)
        return _feed(ModelRunner(model, manager, torch.bfloat16, device, 256, poison_cache=True), manager, ids, cuts)
    got = logits("e4m3", "cuda")
    ops.set_backend(Plain())
    try:
        expect, full = logits("e4m3", "cpu"), logits("compute", "cpu")
    finally:
        ops.set_backend(None)
    for r in got:
        assert torch.isfinite(got[r]).all()
        assert _rms(got[r] - expect[r]) <= 2 ** 0.5 * _rms(expect[r] - full[r]) + helpers.TOL_BF16 * _rms(full[r])
