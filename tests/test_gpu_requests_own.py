"""GPU: requests of one batch that bring their own adapter, their own rules and ask for log-probabilities, through the engine's
entry points.  An adapter's requests are compared with the plain implementation run on the merged weights W + s B A."""

from __future__ import annotations

import json
import math
import subprocess

import pytest
import torch

import plain_qwen2 as plain
from conftest import ROOT, TINY, make_folder, random_tokens
from test_requests_own_cpu import adapter_tensors, write_folder

pytestmark = pytest.mark.gpu


def float_weights(tensors):
    return {k: v.float() for k, v in tensors.items()}


def merged(raw, tensors, adapter, scale, dtype=torch.float32):
    """W + s B A for every projection that the adapter has, its matrices as the engine holds them."""
    out = float_weights(tensors)
    for name in {key.rsplit(".lora_", 1)[0] for key in adapter}:
        a, b = (adapter[f"{name}.lora_{side}.weight"].to(dtype).float() for side in "AB")
        out[name + ".weight"] = out[name + ".weight"] + scale * (b @ a)
    return out


def make_engine(folder, dtype="float32", **options):
    from cie_amd import Engine

    defaults = dict(page_size=8, kv_tokens=2048, max_running=8, prefill_chunk=16, token_budget=48, prefix_cache_pages=0, max_adapters=3,
                    max_adapter_rank=8)
    defaults.update(options)
    return Engine(folder, dtype=dtype, **defaults)


def strong(raw, rank, seed, only=None):
    """An adapter that changes what the model says (the drawn weights have 0.02)."""
    return {name: t * (0.3 if ".lora_B." in name else 0.6) for name, t in adapter_tensors(raw, rank, seed, only).items()}


@pytest.mark.parametrize("name", ["A", "B", "C"])
@pytest.mark.parametrize("captured", [True, False])
def test_every_request_sees_its_own_adapter(tiny_folders, name, captured):
    from cie_amd import GenerationConfig

    folder, raw, tensors = tiny_folders[name]
    adapters = {"x": (strong(raw, 8, 1), 0.7), "y": (strong(raw, 4, 2), 1.3), "z": (strong(raw, 3, 3, only=("q_proj", "down_proj")), 2.0)}
    engine = make_engine(folder, graph_decode=captured)
    for key, (matrices, scale) in adapters.items():
        engine.load_adapter(key, tensors=matrices, scale=scale)
    lengths = [5, 33, 1, 17, 40, 9, 21, 12]
    wanted = ["x", None, "y", "z", "x", None, "y", "x"]
    prompts = [random_tokens(n, raw["vocab_size"], 700 + i) for i, n in enumerate(lengths)]
    results = engine.generate(prompts, [GenerationConfig(max_output_tokens=10, adapter=w) for w in wanted])
    for prompt, who, result in zip(prompts, wanted, results):
        weights = float_weights(tensors) if who is None else merged(raw, tensors, *adapters[who])
        assert result.token_ids == plain.generate_greedy(raw, weights, prompt, 10), who
    base = engine.generate([prompts[0]], GenerationConfig(max_output_tokens=10))[0].token_ids
    assert base == plain.generate_greedy(raw, float_weights(tensors), prompts[0], 10)
    # (the adapters are no small change: by the oracle, they move the logits by a good part of their spread)
    for who, index in (("x", 0), ("y", 2), ("z", 3)):
        one, other = (plain.forward(raw, w, prompts[index]) for w in (float_weights(tensors), merged(raw, tensors, *adapters[who])))
        assert (one - other).abs().max() > 0.2 * one.std()
    if captured:
        assert engine.runner.graphs.adapted_buckets and engine.runner.graph_replays > 8


@pytest.mark.parametrize("name", ["A", "B", "C"])
def test_logits_in_bfloat16(tiny_folders, name):
    """Step by step against the merged weights in float32: prompts in portions, mixed steps, captured decode steps."""
    from cie_amd.engine.runner import StepEntry

    folder, raw, tensors = tiny_folders[name]
    engine = make_engine(folder, dtype="bfloat16")
    matrices = {k: adapter_tensors(raw, 8, 20 + k) for k in range(2)}
    small = [{key: t * (0.1 if ".lora_B." in key else 0.3) for key, t in m.items()} for m in matrices.values()]
    for k in range(2):
        engine.load_adapter(str(k), tensors=small[k], scale=0.8)
    runner = engine.runner
    whole = {who: random_tokens(40, raw["vocab_size"], 60 + i) for i, who in enumerate(("none", "first", "second"))}
    slot = {"none": -1, "first": 0, "second": 1}
    for who in whole:
        runner.cache.admit(who)
    got = {who: [] for who in whole}
    at = 0
    for count in (7, 16, 9, 1, 1, 1, 1, 1, 1, 1, 1):
        entries = [StepEntry(who, tokens[at: at + count], at, tuple(range(count)), slot[who]) for who, tokens in whole.items()]
        logits = runner.run(entries).float().cpu().reshape(3, count, -1)
        for who, rows in zip(whole, logits):
            got[who].append(rows)
        at += count
    assert at == 40 and runner.graphs.adapted_buckets
    for who, tokens in whole.items():
        weights = float_weights(tensors) if slot[who] < 0 else merged(raw, tensors, small[slot[who]], 0.8, torch.bfloat16)
        expected = plain.forward(raw, weights, tokens)
        torch.testing.assert_close(torch.cat(got[who]), expected, rtol=2e-2, atol=2e-2)


def test_a_prefix_is_shared_with_requests_of_the_same_adapter_only(tiny_folders):
    from cie_amd import GenerationConfig

    folder, raw, tensors = tiny_folders["B"]
    engine = make_engine(folder, prefix_cache_pages=64)
    adapters = {"x": (strong(raw, 8, 1), 0.7), "y": (strong(raw, 4, 2), 1.3)}
    for key, (matrices, scale) in adapters.items():
        engine.load_adapter(key, tensors=matrices, scale=scale)
    prompt = random_tokens(41, raw["vocab_size"], 31)
    for who in ("x", None, "y", "x", None, "y"):
        result = engine.generate([prompt], GenerationConfig(max_output_tokens=6, adapter=who))[0]
        weights = float_weights(tensors) if who is None else merged(raw, tensors, *adapters[who])
        assert result.token_ids == plain.generate_greedy(raw, weights, prompt, 6), who
    assert engine.snapshot_metrics()["kv_cache"]["prefix_cache_hits"] == 3
    # a name that is loaded again is another adapter
    engine.unload_adapter("x")
    engine.load_adapter("x", tensors=adapters["y"][0], scale=1.3)
    again = engine.generate([prompt], GenerationConfig(max_output_tokens=6, adapter="x"))[0]
    assert again.token_ids == result.token_ids and engine.snapshot_metrics()["kv_cache"]["prefix_cache_hits"] == 3


def test_adapters_under_cache_pressure(tiny_folders):
    """Requests that are preempted and computed again keep their adapter."""
    from cie_amd import GenerationConfig

    folder, raw, tensors = tiny_folders["B"]
    engine = make_engine(folder, kv_tokens=200, admit_within_pool=False, max_running=4)
    adapters = {"x": (strong(raw, 8, 1), 0.7), "y": (strong(raw, 4, 2), 1.3)}
    for key, (matrices, scale) in adapters.items():
        engine.load_adapter(key, tensors=matrices, scale=scale)
    wanted = ["x", "y", None, "x"]
    prompts = [random_tokens(40, raw["vocab_size"], 90 + i) for i in range(4)]
    results = engine.generate(prompts, [GenerationConfig(max_output_tokens=24, adapter=w) for w in wanted])
    assert engine.snapshot_metrics()["requests"]["preempted_total"] > 0
    for prompt, who, result in zip(prompts, wanted, results):
        weights = float_weights(tensors) if who is None else merged(raw, tensors, *adapters[who])
        assert result.token_ids == plain.generate_greedy(raw, weights, prompt, 24), who


def test_names_and_rooms(tiny_folders):
    from cie_amd import GenerationConfig

    folder, raw, _ = tiny_folders["A"]
    engine = make_engine(folder, max_adapters=1)
    prompt = random_tokens(9, raw["vocab_size"], 3)
    with pytest.raises(ValueError):
        engine.submit(prompt, GenerationConfig(max_output_tokens=2, adapter="x"))
    engine.load_adapter("x", tensors=strong(raw, 8, 1), scale=1.0)
    for bad in (dict(name="y", tensors=strong(raw, 8, 1), scale=1.0), dict(name="x", tensors=strong(raw, 8, 1), scale=1.0),
                dict(name="z"), dict(name="z", tensors=strong(raw, 8, 1))):
        with pytest.raises(ValueError):
            engine.load_adapter(**bad)
    request = engine.submit(prompt, GenerationConfig(max_output_tokens=3, adapter="x"))
    with pytest.raises(ValueError):
        engine.unload_adapter("x")
    engine.scheduler.run_until_done()
    assert len(request.output) == 3
    engine.unload_adapter("x")
    with pytest.raises(ValueError):
        engine.unload_adapter("x")
    without = make_engine(folder, max_adapters=0)
    for call in (lambda: without.load_adapter("x", tensors=strong(raw, 8, 1), scale=1.0), lambda: without.unload_adapter("x"),
                 lambda: without.submit(prompt, GenerationConfig(max_output_tokens=2, adapter="x"))):
        with pytest.raises(ValueError):
            call()
    from cie_amd.engine.runner import StepEntry

    without.runner.cache.admit("a")
    with pytest.raises(ValueError):
        without.runner.run([StepEntry("a", [1], 0, (0,), 0)])


def log_softmax_of(raw, weights, prompt, output):
    logits = plain.forward(raw, weights, prompt + output[:-1])[len(prompt) - 1:].double()
    return torch.log_softmax(logits, -1)


@pytest.mark.parametrize("async_decode", [True, False])
def test_log_probabilities_are_the_models_own(tiny_folders, async_decode):
    from cie_amd import GenerationConfig

    folder, raw, tensors = tiny_folders["B"]
    engine = make_engine(folder, async_decode=async_decode)
    prompts = [random_tokens(n, raw["vocab_size"], 800 + n) for n in (4, 30, 17, 9)]
    gens = [GenerationConfig(max_output_tokens=9, logprobs=True), GenerationConfig(max_output_tokens=9, temperature=0.7, seed=1, logprobs=True),
            GenerationConfig(max_output_tokens=9), GenerationConfig(max_output_tokens=9, temperature=1.4, seed=2, top_k=20, top_p=0.8, logprobs=True)]
    results = engine.generate(prompts, gens)
    assert results[2].logprobs is None
    for prompt, result in zip(prompts, results):
        if result.logprobs is None:
            continue
        table = log_softmax_of(raw, float_weights(tensors), prompt, result.token_ids)
        want = [table[i, t].item() for i, t in enumerate(result.token_ids)]
        assert len(result.logprobs) == 9 and all(abs(a - b) < 1e-3 for a, b in zip(result.logprobs, want))


def test_draws_under_rules_stay_in_the_rules_and_off_the_batch(tiny_folders):
    from cie_amd import GenerationConfig

    folder, raw, tensors = tiny_folders["B"]
    prompts = [random_tokens(n, raw["vocab_size"], 900 + n) for n in (7, 30, 17, 9, 12, 25)]
    rules = [dict(top_k=1), dict(top_k=4), dict(top_p=0.3), dict(min_p=0.5), dict(), dict(top_k=30, top_p=0.7, min_p=0.05)]
    gens = [GenerationConfig(max_output_tokens=12, temperature=0.9, seed=40 + i, **r) for i, r in enumerate(rules)]
    together = make_engine(folder).generate(prompts, gens)
    for prompt, one, result in zip(prompts, gens, together):
        alone = make_engine(folder, token_budget=7, prefill_chunk=5).generate([prompt], one)[0]
        assert alone.token_ids == result.token_ids, one
    greedy = make_engine(folder).generate(prompts[:1], GenerationConfig(max_output_tokens=12))[0]
    assert together[0].token_ids == greedy.token_ids
    for index, bound in ((1, lambda p, i: (p > p[i]).sum() < 4), (2, lambda p, i: p[p > p[i]].sum() < 0.3 + 1e-4),
                         (3, lambda p, i: p[i] >= 0.5 * p.max() - 1e-6)):
        table = log_softmax_of(raw, float_weights(tensors), prompts[index], together[index].token_ids)
        for row, token in zip(table, together[index].token_ids):
            assert bound(torch.softmax(row / 0.9, -1), token), (index, token)


def test_the_sampler_joins_rows_with_and_without_rules():
    from cie_amd.sampling import Sampler

    g = torch.Generator().manual_seed(1)
    logits = (torch.randn((6, 9001), generator=g) * 3).cuda()
    uniforms = torch.rand(6, generator=g).tolist()
    temperatures = [0.8, 0.0, 1.2, 0.7, 0.0, 1.0]
    rules = [(5, 1.0, 0.0), None, None, (0, 0.9, 0.1), (3, 0.5, 0.0), None]
    sampler = Sampler()
    got = sampler.sample(logits, temperatures, uniforms, rules)
    for r in range(6):
        assert sampler.sample(logits[r: r + 1], temperatures[r: r + 1], uniforms[r: r + 1], rules[r: r + 1]) == [got[r]]
    plain_draws = sampler.sample(logits, temperatures, uniforms)
    assert [got[r] for r in (1, 2, 4, 5)] == [plain_draws[r] for r in (1, 2, 4, 5)]
    out = torch.full((6,), -7, dtype=torch.int32).cuda()
    assert sampler.sample_on_device(logits, temperatures, uniforms, out=out, rules=rules) is out and out.tolist() == got


def test_generate_from_the_command_line(tiny_folders, tmp_path):
    folder, raw, tensors = tiny_folders["B"]
    matrices = strong(raw, 12, 5)
    adapter = write_folder(tmp_path / "adapter", matrices, {"peft_type": "LORA", "r": 12, "lora_alpha": 6, "bias": "none"})
    prompt = random_tokens(6, raw["vocab_size"], 2)
    command = [str(ROOT / "bin" / "cie")]
    done = subprocess.run(command + ["generate", "--token-ids", " ".join(map(str, prompt)), "--model", str(folder), "--dtype", "fp32",
                                     "--max-output-tokens", "6", "--no-stream", "--ignore-eos", "--temperature", "0.5", "--top-k", "1",
                                     "--top-p", "0.9", "--min-p", "0.1", "--logprobs", "--adapter", str(adapter)],
                          capture_output=True, text=True, timeout=110)
    assert done.returncode == 0, done.stderr[-2000:]
    lines = done.stdout.strip().splitlines()
    weights = merged(raw, tensors, matrices, 0.5)
    tokens = plain.generate_greedy(raw, weights, prompt, 6)
    assert [int(t) for t in lines[0].split()] == tokens
    table = log_softmax_of(raw, weights, prompt, tokens)
    scores = json.loads(lines[1])["logprobs"]
    assert len(scores) == 6 and all(math.isfinite(s) and abs(s - table[i, t].item()) < 1e-3 for i, (s, t) in enumerate(zip(scores, tokens)))


PROJECTIONS = ("q_proj", "k_proj", "v_proj", "o_proj", "gate_proj", "up_proj", "down_proj")


def check_each_projection(folder, raw, tensors, counts, **options):
    """A sequence for each projection, with an adapter beside that one alone, and one without any, all in one batch: portions, then
    captured decode steps.  The engine keeps the stream in float32 and otherwise rounds where the plain model in bfloat16 does, plus
    the adapter's own sum, so it may be off by twice what that is.  A lost or doubled adapter lies far outside."""
    from cie_amd.engine.runner import StepEntry

    length = sum(counts)
    engine = make_engine(folder, dtype="bfloat16", max_adapters=7, token_budget=8 * max(counts), **options)
    base, slots, whole = float_weights(tensors), {"none": -1}, {"none": random_tokens(length, raw["vocab_size"], 60)}
    adapters = {}
    for slot, only in enumerate(PROJECTIONS):
        factor = 0.3 if only in ("v_proj", "o_proj") else 0.6
        adapters[only] = {key: t * (factor if ".lora_B." in key else 1.0) for key, t in adapter_tensors(raw, 8, 20 + slot, only).items()}
        engine.load_adapter(only, tensors=adapters[only], scale=0.8)
        slots[only], whole[only] = slot, random_tokens(length, raw["vocab_size"], 61 + slot)
    runner, got, at = engine.runner, {who: [] for who in whole}, 0
    for who in whole:
        runner.cache.admit(who)
    for count in counts:
        entries = [StepEntry(who, tokens[at: at + count], at, tuple(range(count)), slots[who]) for who, tokens in whole.items()]
        logits = runner.run(entries).float().cpu().reshape(len(whole), count, -1)
        for who, rows in zip(whole, logits):
            got[who].append(rows)
        at += count
    assert runner.graphs.adapted_buckets
    for who, tokens in whole.items():
        its = [merged(raw, tensors, adapters[who], scale, torch.bfloat16) if slots[who] >= 0 else base for scale in (0.8, 0.0, 1.6)]
        right, without, twice = (plain.forward(raw, weights, tokens) for weights in its)
        bound = 2 * (plain.forward(raw, its[0], tokens, dtype=torch.bfloat16).float() - right).abs().max()
        if slots[who] >= 0:
            for wrong in (without, twice):
                assert ((wrong - right).abs() > bound).float().mean() > 0.25, who  # (by the oracle alone)
        assert (torch.cat(got[who]) - right).abs().max() <= bound, who


@pytest.mark.parametrize("name", ["A", "B", "C"])
def test_each_projections_adapter_in_bfloat16(tiny_folders, name):
    check_each_projection(*tiny_folders[name], (7, 16, 9, 1, 1, 1, 1, 1, 1, 1, 1))


def test_each_projections_adapter_beside_the_wide_models_products(tmp_path):
    """Widths at which the products take the routes of a model of real size: K cut in parts that are added in no order or summed by
    the next norm, tiles of many rows, rows that a product would have made the norm of itself."""
    raw = {**TINY["A"], "hidden_size": 512, "num_attention_heads": 8, "num_key_value_heads": 2, "intermediate_size": 4608}
    folder, tensors = make_folder(tmp_path, raw, seed=31, factor=1.0)
    check_each_projection(folder, raw, tensors, (70, 16, 5, 2, 1, 1, 1), kv_tokens=1024)


def test_a_step_with_log_probabilities_waits_once(tiny_folders):
    """Tokens and their log-probabilities travel together: a step that asks for them synchronises no more often than one that
    does not."""
    import warnings

    from cie_amd import GenerationConfig

    folder, raw, _ = tiny_folders["A"]
    engine = make_engine(folder, async_decode=False)
    waits = {}
    for logprobs in (False, True):
        engine.generate([random_tokens(5, raw["vocab_size"], 1)], GenerationConfig(max_output_tokens=4, logprobs=logprobs))
        with warnings.catch_warnings(record=True) as seen:
            warnings.simplefilter("always")
            torch.cuda.set_sync_debug_mode("warn")
            try:
                result = engine.generate([random_tokens(6, raw["vocab_size"], 2)], GenerationConfig(max_output_tokens=4, logprobs=logprobs))[0]
            finally:
                torch.cuda.set_sync_debug_mode("default")
        waits[logprobs] = sum("synchronizing" in str(warning.message) for warning in seen)
    assert len(result.logprobs) == 4 and waits[False] > 0 and waits[True] <= waits[False], waits
