"""CPU: what a request may ask for itself (rules, log-probabilities, an adapter), how adapters are read, checked and kept, and
that requests of different adapters share no cached prefix."""

from __future__ import annotations

import json

import pytest
import torch

from conftest import TINY


def gen(**options):
    from cie_amd.engine.request import GenerationConfig

    return GenerationConfig(max_output_tokens=4, **options)


def test_rules_of_a_request():
    assert gen(temperature=1.0).rules is None and gen(top_k=5, top_p=0.5).rules is None  # greedy: no rule counts
    assert gen(temperature=0.5, top_k=5).rules == (5, 1.0, 0.0)
    assert gen(temperature=0.5, top_p=0.9, min_p=0.1).rules == (0, 0.9, 0.1)
    for bad in (dict(top_k=-1), dict(top_k=2.5), dict(top_k=1 << 31), dict(top_p=0.0), dict(top_p=1.01), dict(top_p=float("nan")),
                dict(min_p=-0.1), dict(min_p=1.5), dict(min_p=float("nan"))):
        with pytest.raises(ValueError):
            gen(temperature=1.0, **bad)


def test_engine_options_of_adapters():
    from cie_amd.config import build_engine_config

    assert build_engine_config(max_adapters=3, max_adapter_rank=128).max_adapters == 3
    for bad in (dict(max_adapters=-1), dict(max_adapter_rank=0), dict(max_adapter_rank=129)):
        with pytest.raises(ValueError):
            build_engine_config(**bad)


def model_of(raw, dtype="float32"):
    from cie_amd.config import config_from_dict
    from cie_amd.engine.loading import build_model
    from cie_amd.weights import RandomSource

    return build_model(config_from_dict(raw)).load(RandomSource(1), dtype, "cpu")


def module_shapes(raw):
    """(in, out) of every projection, from the configuration alone."""
    hidden, inner = raw["hidden_size"], raw["intermediate_size"]
    dim = raw.get("head_dim") or hidden // raw["num_attention_heads"]
    q, kv = raw["num_attention_heads"] * dim, raw["num_key_value_heads"] * dim
    names = {"self_attn.q_proj": (hidden, q), "self_attn.k_proj": (hidden, kv), "self_attn.v_proj": (hidden, kv),
             "self_attn.o_proj": (q, hidden), "mlp.gate_proj": (hidden, inner), "mlp.up_proj": (hidden, inner),
             "mlp.down_proj": (inner, hidden)}
    return {f"model.layers.{i}.{name}": shape for i in range(raw["num_hidden_layers"]) for name, shape in names.items()}


def adapter_tensors(raw, rank, seed, only=None):
    g = torch.Generator().manual_seed(seed)
    out = {}
    for name, (inputs, outputs) in module_shapes(raw).items():
        if only is None or name.endswith(only):
            out[name + ".lora_A.weight"] = torch.randn((rank, inputs), generator=g) * inputs ** -0.5
            out[name + ".lora_B.weight"] = torch.randn((outputs, rank), generator=g) * rank ** -0.5
    return out


@pytest.mark.parametrize("name", ["A", "B", "C"])
def test_a_room_holds_every_projection_where_its_product_has_it(name):
    """Site by site: W + s B A of the loaded adapter, in the layout in which the part runs the projection."""
    from cie_amd.parts.adapters import AdapterRoom

    raw = TINY[name]
    model = model_of(raw)
    room = AdapterRoom(model, 3, 5)
    assert room.rank == 8 and set(room.modules) == set(module_shapes(raw)) and model.adapter_room is room
    room.load(0, adapter_tensors(raw, 5, 1), 1.0)
    room.load(2, adapter_tensors(raw, 3, 2), 0.5)
    tensors = adapter_tensors(raw, 3, 2)
    prefix = "model.layers.1."
    mixer, ff = model.blocks[1].mixer, model.blocks[1].feed_forward
    dim, wide = mixer.head_dim, mixer.kernel_head_dim
    pad = lambda t: torch.nn.functional.pad(t.reshape(-1, dim, t.shape[1]), (0, 0, 0, wide - dim)).reshape(-1, t.shape[1])  # noqa: E731
    product = lambda n: tensors[n + ".lora_B.weight"] @ tensors[n + ".lora_A.weight"]  # noqa: E731
    for site, parts in ((mixer.site_qkv, [pad(product(prefix + f"self_attn.{p}_proj")) for p in "qkv"]),
                        (mixer.site_o, [pad(product(prefix + "self_attn.o_proj").t()).t()]),
                        (ff.site_gate_up, [product(prefix + f"mlp.{p}_proj") for p in ("gate", "up")]),
                        (ff.site_down, [product(prefix + "mlp.down_proj")])):
        begin = 0
        for piece, (want, width) in enumerate(zip(parts, site.columns)):
            rows = slice(piece * site.rank, (piece + 1) * site.rank)
            got = site.up[2, begin: begin + width] @ site.down[2, rows]
            torch.testing.assert_close(got, want)
            begin += width
        assert not site.down[1].any() and not site.up[1].any()
    assert room.scale.tolist() == [1.0, 0.0, 0.5]
    # a lower rank and fewer projections in a used slot: nothing of the one before is left
    room.load(0, adapter_tensors(raw, 2, 3, only="mlp.down_proj"), 2.0)
    assert not mixer.site_qkv.down[0].any() and not ff.site_gate_up.up[0].any()
    assert ff.site_down.down[0, :2].any() and not ff.site_down.down[0, 2:].any() and not ff.site_down.up[0, :, 2:].any()


def test_what_does_not_fit_is_refused_before_anything_is_written():
    from cie_amd.parts.adapters import AdapterError, AdapterRoom

    raw = TINY["A"]
    model = model_of(raw)
    room = AdapterRoom(model, 1, 8)
    good = adapter_tensors(raw, 4, 5)
    room.load(0, good, 1.0)
    before = [(site.down.clone(), site.up.clone()) for site in room.sites]
    name = "model.layers.0.self_attn.q_proj"
    bad = [
        {}, {"model.layers.9.self_attn.q_proj.lora_A.weight": good[name + ".lora_A.weight"]}, {name + ".bias": good[name + ".lora_A.weight"]},
        {name + ".lora_A.weight": good[name + ".lora_A.weight"]}, {name + ".lora_B.weight": good[name + ".lora_B.weight"]},
        {**good, name + ".lora_A.weight": torch.zeros(4, 63)}, {**good, name + ".lora_B.weight": torch.zeros(64, 3)},
        {**good, name + ".lora_A.weight": torch.zeros(9, 64), name + ".lora_B.weight": torch.zeros(64, 9)},
        {**good, name + ".lora_A.weight": torch.zeros(4, 64, dtype=torch.int32)},
    ]
    for tensors in bad:
        with pytest.raises(AdapterError):
            room.load(0, tensors, 3.0)
    with pytest.raises(ValueError):
        room.load(1, good, 1.0)
    for site, (down, up) in zip(room.sites, before):
        assert torch.equal(site.down, down) and torch.equal(site.up, up)
    assert room.scale.tolist() == [1.0]
    with pytest.raises(ValueError):
        AdapterRoom(model, 0, 8)
    with pytest.raises(ValueError):
        AdapterRoom(model, 1, 129)


def test_layers_without_a_place_for_adapters_are_refused():
    from polosun_util import SMALL
    from cie_amd.parts.adapters import AdapterError, AdapterRoom

    raw = SMALL["A"]
    with pytest.raises(AdapterError):
        AdapterRoom(model_of(raw), 1, 8)


def write_folder(folder, tensors, config, prefix="base_model.model."):
    import safetensors.torch

    folder.mkdir(exist_ok=True)
    (folder / "adapter_config.json").write_text(json.dumps(config))
    safetensors.torch.save_file({prefix + k: v.contiguous() for k, v in tensors.items()}, str(folder / "adapter_model.safetensors"))
    return folder


def test_reading_a_folder(tmp_path):
    from cie_amd.engine.adapters import read_adapter
    from cie_amd.parts.adapters import AdapterError

    tensors = adapter_tensors(TINY["A"], 4, 7)
    config = {"peft_type": "LORA", "r": 4, "lora_alpha": 6, "bias": "none", "target_modules": ["q_proj"], "use_dora": False}
    got, scale = read_adapter(write_folder(tmp_path / "a", tensors, config))
    assert scale == 1.5 and set(got) == set(tensors) and all(torch.equal(got[k], tensors[k]) for k in got)
    named = {k.replace(".weight", ".default.weight"): v for k, v in tensors.items()}
    got, scale = read_adapter(write_folder(tmp_path / "b", named, {**config, "use_rslora": True}, prefix=""))
    assert scale == 3.0 and set(got) == set(tensors)
    for change in ({"bias": "all"}, {"use_dora": True}, {"r": 0}, {"r": None}, {"lora_alpha": None}, {"peft_type": "IA3"},
                   {"modules_to_save": ["lm_head"]}, {"rank_pattern": {"q_proj": 8}}, {"fan_in_fan_out": True}):
        with pytest.raises(AdapterError):
            read_adapter(write_folder(tmp_path / "c", tensors, {**config, **change}))


def test_a_folder_that_says_what_is_not_run(tmp_path):
    from cie_amd.engine.adapters import read_adapter
    from cie_amd.parts.adapters import AdapterError

    tensors = adapter_tensors(TINY["A"], 4, 7)
    config = {"peft_type": "LORA", "r": 4, "lora_alpha": 6}
    read_adapter(write_folder(tmp_path / "a", tensors, config))
    for change in ({"lora_bias": True}, {"layer_replication": [[0, 1], [0, 2]]}, {"alora_invocation_tokens": [5, 6]}, {"r": 8}):
        with pytest.raises(AdapterError):
            read_adapter(write_folder(tmp_path / "b", tensors, {**config, **change}))


def test_names_and_slots():
    from cie_amd.engine.adapters import Adapters
    from cie_amd.parts.adapters import AdapterError, AdapterRoom

    raw = TINY["A"]
    adapters = Adapters(AdapterRoom(model_of(raw), 2, 8))
    one = adapters.load("one", adapter_tensors(raw, 4, 1), 1.0)
    two = adapters.load("two", adapter_tensors(raw, 4, 2), 1.0)
    assert (one.slot, two.slot) == (0, 1) and one.serial != two.serial and adapters.find("one") == one
    with pytest.raises(ValueError):
        adapters.load("three", adapter_tensors(raw, 4, 3), 1.0)
    with pytest.raises(ValueError):
        adapters.load("one", adapter_tensors(raw, 4, 3), 1.0)

    class Live:
        adapter = one

    with pytest.raises(ValueError):
        adapters.unload("one", [Live()])
    adapters.unload("one", [])
    with pytest.raises(ValueError):
        adapters.find("one")
    with pytest.raises(AdapterError):
        adapters.load("bad", {}, 1.0)
    for scale in (float("nan"), float("inf")):
        with pytest.raises(ValueError):
            adapters.load("bad", adapter_tensors(raw, 4, 3), scale)
    again = adapters.load("one", adapter_tensors(raw, 4, 3), 1.0)
    assert again.slot == 0 and again.serial not in (one.serial, two.serial)


def test_a_cached_prefix_belongs_to_its_variant():
    from cie_amd.cache.manager import CacheManager, PagedKV

    m = CacheManager([PagedKV(1, 8)], 4, 64, 4, 64, prefill_chunk=16, prefix_cache_pages=16)
    tokens = list(range(13))
    for rid, variant in (("a", None), ("b", 7), ("c", 8)):
        assert m.admit(rid, tokens, variant) == 0  # (nothing of another variant)
        m.ensure_capacity_batch({rid: 13})
        m.commit_lengths({rid: 13})
        assert m.publish_prefix(rid, tokens, variant) == 12
        m.release(rid, tokens, variant)
    pages = {}
    for rid, variant in (("d", None), ("e", 7), ("f", 8)):
        assert m.admit(rid, tokens, variant) == 12
        pages[rid] = tuple(m.block_table(0, rid))
    assert len(set(pages.values())) == 3 and not set(pages["d"]) & set(pages["e"]) and not set(pages["e"]) & set(pages["f"])


def test_log_probabilities_reach_the_request():
    from cie_amd.config import build_engine_config
    from cie_amd.engine.request import GenerationConfig, ScoredToken
    from cie_amd.engine.scheduler import Scheduler
    from cie_amd.metrics import Metrics
    from test_scheduler import FakeRunner

    class Scoring(FakeRunner):
        def execute_batch(self, plan):
            return {rid: ScoredToken.of(token, -0.25 * token) for rid, token in super().execute_batch(plan).items()}

    scheduler = Scheduler(build_engine_config(), Scoring(), Metrics())
    asks = scheduler.submit([1, 2], GenerationConfig(max_output_tokens=3, logprobs=True))
    silent = scheduler.submit([1, 2], GenerationConfig(max_output_tokens=3))
    scheduler.run_until_done()
    assert asks.output == [100, 101, 102] and asks.logprobs == [-25.0, -25.25, -25.5]
    assert silent.output == [100, 101, 102] and silent.logprobs == []
    assert all(type(token) is int for token in asks.output)


def test_rows_too_long_for_the_kernels_indexes():
    from cie_amd.kernels import ops

    def terms(k, n):
        return ops._lora_terms(torch.Size((1, k)), (k, 1), torch.bfloat16, torch.Size((1, n)), (n, 1), torch.bfloat16, torch.Size((1, 8, k)),
                               torch.Size((1, n, 8)), None, None, 256)

    assert terms(1 << 28, 64)[0] == terms(64, 1 << 28)[0] == 1
    for k, n in (((1 << 28) + 8, 64), (64, (1 << 28) + 8)):
        with pytest.raises(ValueError):
            terms(k, n)


def test_column_blocks_stay_in_a_grids_second_dimension():
    """The form for few rows has its column blocks there: for the widest rows, any rank and pieces of any width."""
    from cie_amd.kernels import ops

    forms = set()
    for n in (1, 128, 2560, 37888, 8388480, 8388609, 9000000, 1 << 28):
        for rows in (1, 64, 618, 65535):
            for rank in (1, 8, 64, 72, 128):
                *_, block, up_slots = ops.plan_lora(rows, 64, n, 4 * rank, rank, 3, 128, 256)
                assert block % 128 == 0
                if up_slots:
                    widths = [n] if n < 4 else [1, 1, n // 2, n - n // 2 - 2]
                    assert sum(-(-width // block) for width in widths) <= 65535, (n, rows, rank)
                    forms.add(block)
    assert len(forms) > 2 and ops.plan_lora(64, 2048, 22016, 32, 16, 16, 128, 256)[4] == 128  # (as it is for a model's widths)


@pytest.mark.parametrize("config", [{"r": None, "lora_alpha": 8}, {"lora_alpha": 8}, {"r": "4", "lora_alpha": 8}, {"r": 4.5, "lora_alpha": 8},
                                    {"r": 4, "lora_alpha": 8, "use_dora": True}, []])
def test_the_command_line_refuses_what_the_folder_says(tmp_path, config):
    """Before an engine is made, and with the refusal that names the fault."""
    from cie_amd.cli import main
    from cie_amd.parts.adapters import AdapterError

    folder = write_folder(tmp_path / "a", adapter_tensors(TINY["A"], 4, 7), config)
    with pytest.raises(AdapterError):
        main(["generate", "--token-ids", "1 2", "--model", str(tmp_path), "--adapter", str(folder)])


def test_adapters_trained_beside_other_weights_are_refused(tmp_path):
    """Starts that move a part of the weights into the matrices leave adapters that are wrong beside the weights themselves."""
    from cie_amd.engine.adapters import read_adapter
    from cie_amd.parts.adapters import AdapterError

    tensors = adapter_tensors(TINY["A"], 4, 7)
    config = {"peft_type": "LORA", "r": 4, "lora_alpha": 6}
    for fine in (True, False, None, "gaussian", "eva", "orthogonal"):
        assert read_adapter(write_folder(tmp_path / "a", tensors, {**config, "init_lora_weights": fine}))[1] == 1.5
    for start in ("pissa", "pissa_niter_16", "olora", "corda", "loftq", "lora_ga"):
        with pytest.raises(AdapterError):
            read_adapter(write_folder(tmp_path / "b", tensors, {**config, "init_lora_weights": start}))
    for change in ({"use_qalora": True}, {"use_bdlora": {"nblocks": 2}}, {"arrow_config": {"top_k": 2}}):
        with pytest.raises(AdapterError):
            read_adapter(write_folder(tmp_path / "b", tensors, {**config, **change}))


def test_a_matrix_under_two_names_is_refused(tmp_path):
    from cie_amd.engine.adapters import read_adapter
    from cie_amd.parts.adapters import AdapterError

    tensors = adapter_tensors(TINY["A"], 4, 7)
    name = next(iter(tensors))
    for other in (name.replace(".weight", ".default.weight"), "base_model.model." + name):
        both = {**tensors, other: tensors[name] + 1}
        with pytest.raises(AdapterError):
            read_adapter(write_folder(tmp_path / "a", both, {"r": 4, "lora_alpha": 6}, prefix=""))


@pytest.mark.parametrize("room", [False, True])
def test_a_warm_up_runs_the_products_of_steps_with_adapters(monkeypatch, room):
    """Every product that such a step makes of its rows runs once, in the form in which it makes it, if there is room for adapters."""
    from cie_amd.parts import attention, feed_forward
    from cie_amd.parts.adapters import AdapterRoom

    model = model_of(TINY["A"])
    if room:
        AdapterRoom(model, 1, 8)
    ran = []

    def product(x, weight, bias=None, epilogue=None, **_):
        ran.append((weight.data_ptr(), epilogue))
        return x.new_zeros((x.shape[0], weight.shape[0] // (2 if epilogue == "silu" else 1)))

    monkeypatch.setattr(attention, "linear", product)
    monkeypatch.setattr(feed_forward, "linear", product)
    block = model.blocks[0]
    block.warm_up(64)
    mixer, ff = block.mixer, block.feed_forward
    always = {(w.data_ptr(), None) for w in (mixer.w_qkv, mixer.w_o, ff.w_down)} | {(ff.w_gate_up.data_ptr(), "silu")}
    assert set(ran) == always | ({(ff.w_gate_up.data_ptr(), None)} if room else set())


def test_a_scale_that_32_bits_do_not_hold_is_refused():
    from cie_amd.engine.adapters import Adapters
    from cie_amd.parts.adapters import AdapterRoom

    adapters = Adapters(AdapterRoom(model_of(TINY["A"]), 1, 8))
    for scale in (1e39, -1e39, float("nan"), float("-inf")):
        with pytest.raises(ValueError):
            adapters.load("one", adapter_tensors(TINY["A"], 4, 3), scale)
    assert not adapters.loaded
    adapters.load("one", adapter_tensors(TINY["A"], 4, 3), -3e38)
    assert torch.isfinite(adapters.room.scale).all()
