"""Parts and engines with weights and cache in 8 bits: the wiring against plain statements, then whole runs against each other."""
import json
import os
import subprocess
import sys

import pytest
import torch

import helpers
import plain_eight_bit as plain
import tau_rs_b200
import tiny_configs
from tau_rs_b200 import Engine, SequenceCache, StepEntry, load_engine, load_model
from tau_rs_b200.config import AttentionSpec, NormSpec, PositionSpec, SwiGLUSpec
from tau_rs_b200.csrc import kernels
from tau_rs_b200.engine.batch import StepLayout, fill_step, step_views
from tau_rs_b200.parts import build

pytestmark = pytest.mark.gpu


def filled(part):
    torch.manual_seed(3)
    for name, spec in part.tensor_specs().items():
        value = 1.0 + 0.1 * torch.randn(spec.shape) if len(spec.shape) == 1 and "norm" in name else torch.randn(spec.shape) * 0.2
        part.assign(name, value.to("cuda", torch.bfloat16 if spec.role == "matrix" else torch.float32))
    part.finalize_weights()
    return part


def step_of(cache, runs, group="g"):
    entries = [StepEntry(slot, [0] * new) for slot, _, new in runs]
    starts = [start for _, start, _ in runs]
    longest = max(start + new for _, start, new in runs)
    layout = StepLayout(sum(new for *_, new in runs), len(runs), 0, {group: -(-longest // 64)})
    for (slot, start, new) in runs:
        cache.reserve(slot, start + new)
    import numpy as np

    staged = np.zeros(layout.total, dtype=np.int32)
    fill_step(layout, staged, entries, starts, cache)
    return step_views(layout, torch.from_numpy(staged).cuda(), max(new for *_, new in runs), longest, all(new == 1 for *_, new in runs))


@pytest.mark.parametrize("heads, kv_heads, dim, window, optimized", [(6, 2, 48, None, True), (4, 4, 64, 40, True), (18, 2, 32, None, True), (4, 2, 32, None, False)])
def test_an_attention_layer_over_8_bit_pages(monkeypatch, heads, kv_heads, dim, window, optimized):
    """Prompts, portions that continue them and single tokens of three sequences, queries and keys prepared as the ordinary kernel prepares them, every context against the
    statement (the bound of the kernels' own test)."""
    kernels.prefer_optimized(optimized)
    try:
        spec = AttentionSpec(hidden=64, n_heads=heads, n_kv_heads=kv_heads, head_dim=dim, bias=True, softmax_scale=dim ** -0.5, qk_norm=NormSpec(width=dim, eps=1e-5),
                             position=PositionSpec(rotary_dim=dim, theta=1e4, max_positions=512), window=window)
        part = filled(build("mixer", spec, prefix="attn", dtype=torch.bfloat16, device="cuda"))
        monkeypatch.setattr(part.out, "forward", lambda context: context)
        cache = SequenceCache({"g": (part.cache_need(), 1)}, 64 * 20, 512, torch.bfloat16, "cuda", cache_format="fp8")
        slots = [cache.open() for _ in range(3)]
        view = cache.layer_view("g", 0)
        keys, values = plain.Pages(20, kv_heads, dim), plain.Pages(20, kv_heads, dim)
        lengths, readers = [0, 0, 0], 0
        for news in ([70, 3, 130], [1, 1, 1], [60, 9, 1], [1, 1, 1]):
            runs = [(slot, length, new) for slot, length, new in zip(slots, lengths, news)]
            step = step_of(cache, runs)
            hidden = torch.randn(sum(news), 64, device="cuda").to(torch.bfloat16)
            found = part.forward(hidden, step, view, True).double().cpu()
            # A run that reads what another stored, from the same queries (a product of fewer features may be cut along K another way and round another way).
            if torch.equal(part.qkv.forward(hidden)[:, : part.q_width], part.qkv.forward(hidden, rows=part.q_width)):
                assert torch.equal(found, part.forward(hidden, step, view, False).double().cpu())
                readers += 1
            # The same queries, keys and values from the ordinary prepare kernel, in pages of its own.
            projected = part.qkv.forward(hidden)
            queries = torch.empty(sum(news), heads * dim, device="cuda", dtype=torch.bfloat16)
            pages = [torch.zeros(20, kv_heads, 64, dim, device="cuda", dtype=torch.bfloat16) for _ in range(2)]
            kernels.attention_prepare(projected, queries, *pages, True, part.q_norm.weight, part.k_norm.weight, 1e-5, part.position.cos, part.position.sin, dim, step.positions,
                                      step.token_seq, step.page_rows["g"], heads, kv_heads, dim)
            first = 0
            for index, (slot, start, new) in enumerate(runs):
                table = cache.page_rows("g", [slot], -(-(start + new) // 64))[0]
                rows = [(int(table[p // 64]), p % 64) for p in range(start, start + new)]
                for held, source in ((keys, pages[0]), (values, pages[1])):
                    held.store_run(table, start, torch.stack([source[page, :, place] for page, place in rows]).cpu())
                wanted, spread, reach = plain.attention(queries[first : first + new].view(new, heads, dim).cpu(), keys.sequence(table, start + new), values.sequence(table, start + new),
                                                        start, dim ** -0.5, window or 0)
                lost = 2.0 ** -8 + 2.0 * (dim + 4) * 2.0 ** -23 * reach + 2.0 ** -18
                bound = lost * spread + 2.0 ** -8 * (wanted.abs() + lost * spread)
                assert bool(((found[first : first + new].view(new, heads, dim) - wanted).abs() <= bound).all()), (news, index)
                lengths[index] = start + new
                cache.advance(slot, start + new)
                first += new
        assert readers >= 2      # the steps of single tokens at least: few rows are never cut
    finally:
        kernels.prefer_optimized(True)


@pytest.mark.parametrize("optimized", [True, False])
@pytest.mark.parametrize("activation, limit", [("silu", 0.0), ("clamped", 3.0), ("relu", 0.0)])
def test_a_feed_forward_with_weights_in_8_bits(activation, limit, optimized):
    """Against its own held weights, both products quantising their input: the second's input is taken from the first as it left, so the bound is one product's."""
    kernels.prefer_optimized(optimized)
    try:
        spec = SwiGLUSpec(hidden=144, intermediate=208, activation=activation, limit=limit, weight_format="fp8")
        part = filled(build("feed_forward", spec, prefix="m", dtype=torch.bfloat16, device="cuda"))
        assert part.gate_up.weight is None and part.down.codes.dtype == torch.float8_e4m3fn
        for rows in (1, 8, 20, 200):
            hidden = torch.randn(rows, 144, device="cuda").to(torch.bfloat16)
            inner = part.gate_up.forward_gated(hidden, part.limit) if part.fused else None
            found = part.forward(hidden, None).double().cpu()
            if inner is None:
                stacked = part.gate_up.forward(hidden)
                inner = torch.empty(rows, 208, device="cuda", dtype=torch.bfloat16)
                kernels.silu_mul(stacked, inner, relu=True)
            held = plain.held_rows(inner.cpu())[0]
            weight = part.down.codes.cpu().double() * part.down.scales.cpu().double().repeat_interleave(128, 0).repeat_interleave(128, 1)[:144, :208]
            wanted = held @ weight.T
            bound = (128 * 2.0 ** -23 + 5 * 2.0 ** -24) * (held.abs() @ weight.abs().T)
            assert bool(((found - wanted).abs() <= bound + 2.0 ** -8 * (wanted.abs() + bound) + 1e-37).all())
    finally:
        kernels.prefer_optimized(True)


def relative(found, wanted):
    return float((found.double() - wanted.double()).norm() / wanted.double().norm())


@pytest.fixture(scope="module")
def folders(tmp_path_factory):
    root = str(tmp_path_factory.mktemp("eight_bit"))
    return {which: tiny_configs.write_tiny(root, which, "bfloat16") for which in ("A", "B", "C")}


@pytest.mark.parametrize("which, weights, cache", [("A", "fp8", "fp8"), ("B", "fp8", "auto"), ("B", "auto", "fp8"), ("B", "fp8", "fp8"), ("C", "auto", "fp8")])
def test_an_engine_in_8_bits_is_near_the_16_bit_one_however_it_is_cut(folders, which, weights, cache):
    """An element held in e4m3 is off by at most 2^-4 of itself, evenly spread: 0.026 root mean square, 0.037 for a product of two.  Twelve products a model at most (three
    layers of four) and two reads of the cache a layer, adding as squares: 0.037 * sqrt(18) = 0.16 of the logits' norm, allowed twice.  Cuttings of the same run differ by bfloat16
    roundings (2^-8), which move some codes by a step (2^-3 of one element): allowed a quarter of the above."""
    tokens = helpers.random_prompts(tiny_configs.CONFIGS[which]["vocab_size"], [100], 4)[0]
    plain_engine = load_engine(folders[which], "bfloat16", max_tokens=1024)
    engine = load_engine(folders[which], "bfloat16", max_tokens=1024, weights=weights, cache=cache)
    wanted = helpers.run_whole(plain_engine, tokens)
    whole = helpers.run_whole(engine, tokens)
    assert relative(whole, wanted) < 0.32
    stepwise = helpers.run_tail_stepwise(engine, tokens, 40)
    assert relative(stepwise, whole[60:]) < 0.08
    engine.use_graphs = False
    launched = helpers.run_tail_stepwise(engine, tokens, 40)
    assert relative(launched, stepwise) < 0.08
    batched = helpers.run_batched(engine, [tokens, tokens[:50], tokens[10:90]], [60, 20, 70])
    assert relative(batched[0], whole[59:]) < 0.08
    engine.cache.check()
    if cache == "fp8":      # codes in the place of two bytes an element
        assert engine.cache.kv["attention"].keys.dtype == torch.float8_e4m3fn and engine.cache.bytes_per_token() <= plain_engine.cache.bytes_per_token() // 2 + 8
    if weights == "fp8":
        assert engine.model.weight_bytes() < plain_engine.model.weight_bytes()


def test_a_windowed_cache_in_8_bits_gives_pages_back(tmp_path):
    """A page that is taken again starts its scales afresh: portions and single tokens through four pages against one step with room for all."""
    from tau_rs_b200.config.registry import register_architecture
    from tau_rs_b200.weights import write_random_model

    try:
        register_architecture("ToyWindowForCausalLM", "toy_window", lambda raw: raw, helpers.window_spec)
    except ValueError:
        pass      # registered by another test
    folder = str(tmp_path / "toy")
    write_random_model(folder, helpers.WINDOW_CONFIG, seed=5, storage="bfloat16")
    model = load_model(folder, "bfloat16", enforce_declared_dtype=False)
    tokens = helpers.random_prompts(helpers.WINDOW_CONFIG["vocab_size"], [300], 6)[0]
    wanted = helpers.run_whole(Engine(model, 64 * 8, cache_format="fp8"), tokens)
    tight = Engine(model, 64 * 4, cache_format="fp8")
    slot = tight.open_sequence()
    found, position = [], 0
    for count in [50, 1, 64, 30, 1, 1, 64, 40] + [1] * 49:
        piece = tokens[position : position + count]
        found.append(tight.step([StepEntry(slot, piece, list(range(len(piece))))]).float().cpu().clone())
        position += count
        tight.cache.check()
    assert position == 300 and relative(torch.cat(found), wanted) < 0.08


def test_generating_with_both_formats(folders):
    prompts = helpers.random_prompts(500, [5, 90, 30], 8)
    output = tau_rs_b200.generate(folders["B"], prompts, max_new_tokens=12, stop_tokens=(), dtype="bfloat16", weights="fp8", cache="fp8")
    assert [len(result.tokens) for result in output] == [12, 12, 12]
    engine = load_engine(folders["B"], "bfloat16", max_tokens=1024, weights="fp8", cache="fp8")
    for prompt, result in zip(prompts, output):      # each token is near the greatest logit of the same run alone
        logits = helpers.run_whole(engine, list(prompt) + result.tokens)
        for index, token in enumerate(result.tokens):
            row = logits[len(prompt) - 1 + index]
            assert float(row.max() - row[token]) <= 0.08 * float(row.norm())
    with pytest.raises(ValueError, match="already"):
        tau_rs_b200.generate(engine, prompts, weights="fp8")
    with pytest.raises(ValueError, match="not held"):
        tau_rs_b200.generate(load_engine(folders["B"], "bfloat16", max_tokens=1024), prompts, cache="fp8")


def test_the_command_line_with_both_formats(folders):
    command = [sys.executable, os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "bin", "tau"), "--model", folders["B"], "--dtype", "bf16", "--weights", "fp8",
               "--cache", "fp8", "--prompt-ids", "1,2,3", "--max-tokens", "5", "--stop-ids", ""]
    result = subprocess.run(command, capture_output=True, text=True, timeout=600)
    assert result.returncode == 0, result.stderr
    assert len(json.loads(result.stdout.splitlines()[0])["tokens"]) == 5
    refused = subprocess.run(command[:4] + ["--dtype", "f32"] + command[6:], capture_output=True, text=True, timeout=600)
    assert refused.returncode != 0 and "bfloat16" in refused.stderr


def test_loading_weights_in_8_bits_never_holds_the_model_in_16(tmp_path):
    """From a folder and drawn on the device: the greatest memory in between is the codes' (half the products' bytes), embedding and head, and a stack or two; allowed three quarters of the products."""
    config = dict(tiny_configs.TINY_B, hidden_size=512, intermediate_size=1536, num_hidden_layers=10, num_attention_heads=8, num_key_value_heads=4, head_dim=64)
    from tau_rs_b200.api import random_model
    from tau_rs_b200.weights import write_random_model

    folder = str(tmp_path / "model")
    write_random_model(folder, config, seed=1, storage="bfloat16")
    for load in (lambda: load_model(folder, "bfloat16", weights="fp8"), lambda: random_model(config, weights="fp8")):
        torch.cuda.synchronize()
        torch.cuda.reset_peak_memory_stats()
        before = torch.cuda.memory_stats()["requested_bytes.all.current"]      # as asked for: the allocator may hand out larger blocks
        model = load()
        peak = torch.cuda.memory_stats()["requested_bytes.all.peak"] - before
        wide = {name: 2 * spec.shape[0] * spec.shape[1] for name, spec in model.tensor_specs().items() if spec.role == "matrix"}
        products = sum(size for name, size in wide.items() if "proj" in name)
        assert products > 60e6 and peak < 0.75 * products + sum(wide.values()) - products, (peak, products)
        del model
