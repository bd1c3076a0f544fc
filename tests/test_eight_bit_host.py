"""What the entry points of weights and caches in 8 bits refuse; no GPU is needed, the refusals come before any launch."""
from types import SimpleNamespace

import pytest
import torch

import plain_eight_bit
from tau_rs_b200.csrc import kernels

CODES = torch.float8_e4m3fn


def test_the_plain_statement_rounds_as_the_type_does():
    """Every value between codes, borders and subnormals: the statement in 64-bit against torch's own type, with a scale of one."""
    codes = torch.arange(0, 0x7F, dtype=torch.uint8).view(CODES).double()
    between = torch.cat([codes, (codes[1:] + codes[:-1]) / 2, (codes[1:] * 0.3 + codes[:-1] * 0.7), -codes])
    assert torch.equal(plain_eight_bit.to_e4m3(between, 1.0), between.float().to(CODES).double())


@pytest.mark.parametrize("greatest, power", [(448.0, 0), (448.5, 1), (1.75, -8), (1.7501, -7), (1.0, -8), (2.0 ** -140, -120), (0.0, -120), (3.3e38, 120)])
def test_the_scale_is_the_least_power_of_two_that_reaches(greatest, power):
    assert plain_eight_bit.power_of(greatest) == 2.0 ** power


def product_operands(rows=3, depth=32, features=16):
    return dict(values=torch.zeros(rows, depth, dtype=torch.bfloat16), codes=torch.zeros(features, depth, dtype=torch.uint8).view(CODES),
                scales=torch.ones(-(-features // 128), -(-depth // 128)), out=torch.zeros(rows, features, dtype=torch.bfloat16))


@pytest.mark.parametrize("change, message", [
    (dict(values=torch.zeros(3, 48, dtype=torch.bfloat16)), "shapes"),
    (dict(values=torch.zeros(3, 32, dtype=torch.float16)), "activations"),
    (dict(values=torch.zeros(3, 36, dtype=torch.bfloat16)[:, :32]), "16-byte"),
    (dict(values=torch.zeros(32, 3, dtype=torch.bfloat16).T), "activations"),
    (dict(codes=torch.zeros(16, 32, dtype=torch.uint8)), "float8_e4m3fn"),
    (dict(codes=torch.zeros(16, 64, dtype=torch.uint8).view(CODES)[:, :32]), "contiguous"),
    (dict(scales=torch.ones(1, 2)), "scales"),
    (dict(scales=torch.ones(1, 1, dtype=torch.float64)), "scales"),
    (dict(out=torch.zeros(3, 15, dtype=torch.bfloat16)), "output"),
    (dict(out=torch.zeros(3, 16, dtype=torch.float16)), "output"),
    (dict(out=torch.zeros(1, 16, dtype=torch.bfloat16).expand(3, 16)), "output"),
    (dict(bias=torch.zeros(16, dtype=torch.bfloat16)), "bias"),
    (dict(bias=torch.zeros(15)), "bias"),
    (dict(), "CUDA"),
])
def test_products_refuse(change, message):
    arguments = {**product_operands(), "bias": None, **change}
    with pytest.raises(kernels.KernelError, match=message):
        kernels.linear8(arguments["values"], arguments["codes"], arguments["scales"], arguments["bias"], arguments["out"])


def test_products_refuse_a_depth_of_no_whole_16_bytes():
    operands = product_operands(depth=24)
    operands["values"] = torch.zeros(3, 32, dtype=torch.bfloat16)[:, :24]
    with pytest.raises(kernels.KernelError, match="multiple of 16"):
        kernels.linear8(operands["values"], operands["codes"], operands["scales"], None, operands["out"])
    with pytest.raises(kernels.KernelError, match="multiple of 16"):
        kernels.quantize_blocks(torch.zeros(16, 24))


@pytest.mark.parametrize("features, out", [(24, torch.zeros(3, 12, dtype=torch.bfloat16)), (16, torch.zeros(3, 16, dtype=torch.bfloat16)), (16, torch.zeros(3, 8))])
def test_gated_products_refuse(features, out):
    operands = product_operands(features=features)
    with pytest.raises(kernels.KernelError):
        kernels.linear8_gated(operands["values"], operands["codes"], operands["scales"], out)


def cache_operands(tokens=5, pages=4, heads=2, dim=32, sequences=2):
    def ints(*values):
        return torch.tensor(values, dtype=torch.int32)

    step = SimpleNamespace(n_tokens=tokens, n_seqs=sequences, cu_seqlens=ints(0, 2, 5), seq_start=ints(0, 3), seq_len=ints(2, 6), all_single=False, max_len=6, decode_splits=0)
    return dict(keys=torch.zeros(tokens, heads, dim, dtype=torch.bfloat16), values=torch.zeros(tokens, heads, dim, dtype=torch.bfloat16),
                key_pages=torch.zeros(pages, heads, 64, dim, dtype=torch.uint8).view(CODES), value_pages=torch.zeros(pages, heads, 64, dim, dtype=torch.uint8).view(CODES),
                key_scales=torch.ones(pages, heads), value_scales=torch.ones(pages, heads), step=step, page_rows=torch.zeros(sequences, 2, dtype=torch.int32))


BAD_PAGES = [
    dict(key_pages=torch.zeros(4, 2, 64, 32, dtype=torch.bfloat16)),
    dict(value_pages=torch.zeros(3, 2, 64, 32, dtype=torch.uint8).view(CODES)),
    dict(key_pages=torch.zeros(4, 2, 32, 32, dtype=torch.uint8).view(CODES), value_pages=torch.zeros(4, 2, 32, 32, dtype=torch.uint8).view(CODES)),
    dict(key_pages=torch.zeros(4, 2, 64, 24, dtype=torch.uint8).view(CODES), value_pages=torch.zeros(4, 2, 64, 24, dtype=torch.uint8).view(CODES)),
    dict(key_scales=torch.ones(4, 3)),
    dict(value_scales=torch.ones(4, 2, dtype=torch.bfloat16)),
    dict(page_rows=torch.zeros(3, 2, dtype=torch.int32)),
    dict(page_rows=torch.zeros(2, 2, dtype=torch.int64)),
]


@pytest.mark.parametrize("change", BAD_PAGES + [dict(keys=torch.zeros(4, 2, 32, dtype=torch.bfloat16)), dict(values=torch.zeros(5, 2, 32)),
                                                dict(keys=torch.zeros(5, 2, 64, dtype=torch.bfloat16)[:, :, :32]), dict()])
def test_the_store_refuses(change):
    operands = {**cache_operands(), **change}
    with pytest.raises(kernels.KernelError):
        kernels.cache8_store(**operands)


@pytest.mark.parametrize("change", BAD_PAGES + [dict(queries=torch.zeros(5, 127, dtype=torch.bfloat16)), dict(queries=torch.zeros(5, 128)), dict(out=torch.zeros(5, 64, dtype=torch.bfloat16)),
                                                dict(heads=3), dict(kv_heads=4), dict(head_dim=64), dict(window=-1), dict()])
def test_attention_refuses(change):
    operands = {**cache_operands(), "queries": torch.zeros(5, 128, dtype=torch.bfloat16), "out": torch.zeros(5, 128, dtype=torch.bfloat16), "heads": 4, "kv_heads": 2, "head_dim": 32, "window": 0, **change}
    with pytest.raises(kernels.KernelError):
        kernels.attention8(operands["queries"], operands["key_pages"], operands["value_pages"], operands["key_scales"], operands["value_scales"], operands["out"], operands["step"],
                           operands["page_rows"], operands["heads"], operands["kv_heads"], operands["head_dim"], 1.0, operands["window"])


def test_page_rows_hold_the_longest_sequence():
    operands = cache_operands()
    operands["step"].max_len = 129      # two pages are listed
    with pytest.raises(kernels.KernelError, match="longest sequence"):
        kernels.cache8_store(**operands)


def test_rotation_tables_hold_the_longest_sequence():
    operands, tables = cache_operands(), [torch.zeros(5, 16) for _ in range(2)]      # six positions are there
    with pytest.raises(kernels.KernelError, match="rotation tables"):
        kernels.cache8_store(**operands, prepare=(torch.zeros(5, 128, dtype=torch.bfloat16), torch.zeros(5, 128, dtype=torch.bfloat16), None, None, 1e-6, *tables, 32, 4))


# ---- configuration, cache and budget: host logic ---------------------------------------------------------------------------------
def tiny_spec(which="B"):
    import tiny_configs
    from tau_rs_b200.config.registry import architecture_for

    entry = architecture_for(tiny_configs.CONFIGS[which])
    return entry.build_spec(entry.parse_config(tiny_configs.CONFIGS[which]))


def test_a_model_names_the_parts_whose_weights_are_held_in_8_bits():
    from tau_rs_b200 import DecoderModel
    from tau_rs_b200.config.specs import with_weight_format

    spec = tiny_spec("B")
    assert with_weight_format(spec, "") is spec
    changed = with_weight_format(spec, "fp8")
    assert all(block.mixer.weight_format == block.feed_forward.weight_format == "fp8" for block in changed.blocks) and spec.blocks[0].mixer.weight_format == ""
    model = DecoderModel(changed, torch.bfloat16, "cpu")
    assert model.tensor_specs() == DecoderModel(spec, torch.bfloat16, "cpu").tensor_specs()      # the folder is the same
    block = model.blocks[0]
    assert block.feed_forward.fused and block.mixer.qkv.weight_format == block.feed_forward.down.weight_format == "fp8"
    # 96 wide, 8 heads of 32 over one, 224 inner: bytes of codes and scales in the place of two bytes an element.
    held = [(320, 96), (96, 256), (448, 96), (96, 224)]
    saved = sum(rows * columns - 4 * -(-rows // 128) * -(-columns // 128) for rows, columns in held)
    plain = DecoderModel(spec, torch.bfloat16, "cpu")
    assert plain.weight_bytes() - model.weight_bytes() == 3 * saved
    with pytest.raises(ValueError, match="fp4"):
        with_weight_format(spec, "fp4")


def test_weights_in_8_bits_are_refused_where_they_are_not_served():
    import fasesun_models
    from tau_rs_b200 import DecoderModel
    from tau_rs_b200.api import random_model
    from tau_rs_b200.config.errors import UnsupportedDType
    from tau_rs_b200.config.specs import with_weight_format
    import tiny_configs

    with pytest.raises(ValueError, match="multiples of 16"):
        DecoderModel(with_weight_format(tiny_spec("C"), "fp8"), torch.bfloat16, "cpu")      # 120 wide
    with pytest.raises(ValueError, match="8 bits"):
        DecoderModel(with_weight_format(tiny_spec("B"), "fp8"), torch.float32, "cpu")
    with pytest.raises(UnsupportedDType, match="float32"):
        random_model(tiny_configs.TINY_B, dtype="float32", device=torch.device("cpu"), weights="fp8")
    with pytest.raises(UnsupportedDType, match="fp16"):
        random_model(tiny_configs.TINY_B, device=torch.device("cpu"), weights="fp16")
    with pytest.raises(UnsupportedDType, match="latent_attention|served"):
        random_model(fasesun_models.MIXED, device=torch.device("cpu"), weights="fp8")


def test_a_cache_in_8_bits_holds_codes_and_scales():
    from tau_rs_b200 import SequenceCache
    from tau_rs_b200.parts.base import CacheNeed

    groups = {"attention": (CacheNeed("kv", n_kv_heads=2, head_dim=32, eight_bit=True), 3), "state": (CacheNeed("state", state_shape=(4,)), 1)}
    cache = SequenceCache(groups, 64 * 5, 1024, torch.bfloat16, "cpu", cache_format="fp8")
    view = cache.layer_view("attention", 1)
    assert view.keys.dtype == view.values.dtype == CODES and view.keys.shape == (5, 2, 64, 32) and view.key_scales.shape == view.value_scales.shape == (5, 2)
    assert view.key_scales.dtype == torch.float32 and cache.layer_view("attention", 2).key_scales.data_ptr() != view.key_scales.data_ptr()
    assert cache.bytes_per_token() == 2 * 3 * 2 * 32 + 2 * 3 * 2 * 4 // 64
    wide = SequenceCache(groups, 64 * 5, 1024, torch.bfloat16, "cpu")
    assert wide.layer_view("attention", 1).key_scales is None and wide.layer_view("attention", 1).keys.dtype == torch.bfloat16
    slot = cache.open()
    cache.reserve(slot, 130)
    cache.advance(slot, 130)
    cache.check()


@pytest.mark.parametrize("need, dtype, cache_format, message", [
    (dict(kind="kv", n_kv_heads=2, head_dim=32), torch.bfloat16, "fp8", "run's dtype"),
    (dict(kind="rows", row_width=32), torch.bfloat16, "fp8", "run's dtype"),
    (dict(kind="state", state_shape=(4,)), torch.bfloat16, "fp8", "no keys"),
    (dict(kind="kv", n_kv_heads=2, head_dim=32, eight_bit=True), torch.float32, "fp8", "bfloat16 runs"),
    (dict(kind="kv", n_kv_heads=2, head_dim=32, eight_bit=True), torch.bfloat16, "int8", "unknown"),
])
def test_caches_in_8_bits_are_refused_where_they_are_not_served(need, dtype, cache_format, message):
    from tau_rs_b200 import SequenceCache
    from tau_rs_b200.parts.base import CacheNeed

    with pytest.raises(ValueError, match=message):
        SequenceCache({"g": (CacheNeed(**need), 1)}, 256, 256, dtype, "cpu", cache_format=cache_format)


def test_the_budget_counts_a_byte_an_element_and_the_scales():
    from tau_rs_b200.cache.budget import kv_bytes_per_token
    from tau_rs_b200.parts.base import CacheNeed

    groups = {"kv": (CacheNeed("kv", n_kv_heads=8, head_dim=128, eight_bit=True), 36)}
    assert kv_bytes_per_token(groups, 2) == 2 * 36 * 8 * 128 * 2
    assert kv_bytes_per_token(groups, 1) == 2 * 36 * 8 * 128 + 36      # 2 x 36 x 8 scales of 4 bytes to 64 positions


def test_the_command_line_names_both_formats():
    from tau_rs_b200.cli import build_parser

    parser = build_parser()
    assert parser.parse_args([]).weights == parser.parse_args([]).cache == "auto"
    assert parser.parse_args(["--weights", "fp8", "--cache", "fp8"]).weights == "fp8"
    with pytest.raises(SystemExit):
        parser.parse_args(["--cache", "fp4"])


def test_ranges_of_a_decode_over_8_bit_pages():
    """The rule's corners: never more ranges than pages, one where sequences fill the machine, numbers just above a cluster's eight become eight."""
    splits = kernels.decode8_splits
    assert splits(1, 1, 8, 148) == 1 and splits(1, 64, 8, 148) == 1 and splits(1, 300, 8, 148) == 8 and splits(8, 2048, 8, 148) == 4
    assert splits(64, 2048, 8, 148) == 1 and splits(40, 6000, 8, 148) == 2 and splits(2, 120000, 8, 148) == 37 and splits(4, 1000, 8, 148) == 4
    for n_seqs in (1, 3, 17, 64, 500):
        for length in (1, 65, 1000, 33000, 1 << 20):
            found = splits(n_seqs, length, 8, 148)
            assert 1 <= found <= 64 and found <= max(1, (1 << (length - 1).bit_length()) // 64)


def test_which_runs_are_worked_on_like_single_tokens():
    rule = kernels.runs8_like_single_tokens
    assert rule(4, 16, 4500, 32, 8, 128) and not rule(4, 17, 4500, 32, 8, 128)      # 64 and 68 columns
    assert rule(4, 76, 4500, 32, 8, 80) and not rule(4, 77, 4500, 32, 8, 80)        # 19 and 20 readings of 4 x 8 x 71 pages, for 700 x 63
    assert rule(64, 8, 2000, 32, 8, 256) and not rule(64, 9, 2000, 32, 8, 256)      # 32 and 36 columns
    assert rule(1, 64, 500, 32, 8, 128) and not rule(1, 256, 500, 32, 8, 128)       # 8 heads x 8 pages x 16 readings, x 64


@pytest.mark.parametrize("optimized", [True, False])
def test_products_refuse_codes_that_begin_between_borders(optimized):
    """Codes are read four and sixteen at a time, by the plain kernel too."""
    operands = product_operands()
    operands["codes"] = torch.zeros(16 * 32 + 1, dtype=torch.uint8)[1:].view(16, 32).view(CODES)
    assert operands["codes"].is_contiguous()
    kernels.prefer_optimized(optimized)
    try:
        with pytest.raises(kernels.KernelError, match="16-byte border"):
            kernels.linear8(operands["values"], operands["codes"], operands["scales"], None, operands["out"])
        with pytest.raises(kernels.KernelError, match="16-byte border"):
            kernels.linear8_gated(operands["values"], operands["codes"], operands["scales"], torch.zeros(3, 8, dtype=torch.bfloat16))
    finally:
        kernels.prefer_optimized(True)


def quantised_operands(rows=3, depth=272, features=16):
    return dict(x_codes=torch.zeros(rows, depth, dtype=torch.uint8).view(CODES), x_scales=torch.ones(-(-depth // 128), rows), codes=torch.zeros(features, depth, dtype=torch.uint8).view(CODES),
                scales=torch.ones(-(-features // 128), -(-depth // 128)), bias=None, out=torch.zeros(rows, features, dtype=torch.bfloat16))


BETWEEN_BORDERS = torch.zeros(3 * 272 + 1, dtype=torch.uint8)[1:].view(3, 272).view(CODES)


@pytest.mark.parametrize("product", [kernels.gemm8_simt, kernels.gemm8_skinny, kernels.gemm8_tc])
@pytest.mark.parametrize("change, message", [
    (dict(x_scales=torch.ones(2, 3)), "activations' scales"),
    (dict(x_scales=torch.ones(3, 2)), "activations' scales"),
    (dict(x_scales=torch.ones(3, 3, dtype=torch.float64)), "activations' scales"),
    (dict(x_scales=torch.ones(3, 6)[:, ::2]), "activations' scales"),
    (dict(x_codes=torch.zeros(3, 272, dtype=torch.bfloat16)), "activations"),
    (dict(x_codes=torch.zeros(3, 256, dtype=torch.uint8).view(CODES), x_scales=torch.ones(2, 3)), "shapes"),
    (dict(x_codes=torch.zeros(3, 288, dtype=torch.uint8).view(CODES)[:, :272]), "activations"),
    (dict(x_codes=BETWEEN_BORDERS), "16-byte border"),
    (dict(scales=torch.ones(1, 2)), "weight's scales"),
    (dict(scales=torch.ones(2, 3)), "weight's scales"),
    (dict(codes=torch.zeros(16, 272, dtype=torch.uint8)), "float8_e4m3fn"),
    (dict(codes=BETWEEN_BORDERS, out=torch.zeros(3, 3)), "16-byte border"),
    (dict(bias=torch.ones(15)), "bias"),
    (dict(out=torch.zeros(2, 16)), "output"),
    (dict(out=torch.zeros(3, 8)), "output"),
    (dict(out=torch.zeros(3, 16, dtype=torch.float16)), "output"),
    (dict(out=torch.zeros(16, 3).T), "output"),
    (dict(), "CUDA"),
])
def test_products_of_quantised_operands_refuse(product, change, message):
    with pytest.raises(kernels.KernelError, match=message):
        product(**{**quantised_operands(), **change})


def test_the_streaming_and_the_tiled_product_refuse():
    operands = product_operands()
    arguments = (operands["values"], operands["codes"], torch.ones(1, 2), None, operands["out"])
    with pytest.raises(kernels.KernelError, match="scales"):
        kernels.gemm8_stream(*arguments)
    with pytest.raises(kernels.KernelError, match="output"):
        kernels.gemm8_stream(operands["values"], operands["codes"], operands["scales"], None, operands["out"], gated=True)
    for wrong in (dict(features=64), dict(ranges=9), dict(ranges=-1)):
        with pytest.raises(kernels.KernelError, match="CUDA|tiles"):
            kernels.gemm8_tc(**quantised_operands(), **wrong)


@pytest.mark.parametrize("change", BAD_PAGES + [dict(queries=torch.zeros(5, 127, dtype=torch.bfloat16)), dict(out=torch.zeros(5, 64, dtype=torch.bfloat16)), dict(heads=3), dict(window=-1), dict()])
def test_attention_over_pages_as_they_are_held_refuses(change):
    operands = {**cache_operands(), "queries": torch.zeros(5, 128, dtype=torch.bfloat16), "out": torch.zeros(5, 128, dtype=torch.bfloat16), "heads": 4, "window": 0, **change}
    with pytest.raises(kernels.KernelError):
        kernels.attention_decode8(operands["queries"], operands["key_pages"], operands["value_pages"], operands["key_scales"], operands["value_scales"], operands["out"], operands["step"],
                                  operands["page_rows"], operands["heads"], 2, 32, 1.0, operands["window"])


def test_weights_are_brought_to_8_bits_as_the_tensors_arrive(monkeypatch):
    """Tensor by tensor as a loader hands them over: a stack's pieces are gone with its last one, whatever the order inside it, biases are kept for the end."""
    from tau_rs_b200 import DecoderModel
    from tau_rs_b200.config.specs import with_weight_format
    from tau_rs_b200.parts.linear import StackedLinear

    quantised = []
    monkeypatch.setattr(kernels, "quantize_blocks", lambda weight: quantised.append(weight.clone()) or (weight.to(CODES), torch.ones(1)))
    model = DecoderModel(with_weight_format(tiny_spec("B"), "fp8"), torch.bfloat16, "cpu")      # with biases
    stacks = [stack for block in model.blocks for stack in (block.mixer.qkv, block.mixer.out, block.feed_forward.gate_up, block.feed_forward.down)]
    for index, (name, spec) in enumerate(model.tensor_specs().items()):
        model.assign(name, torch.full(spec.shape, 1.0 + index % 50, dtype=torch.bfloat16 if spec.role == "matrix" else torch.float32))
        waiting = [stack for stack in stacks if any(part.dim() == 2 for part in stack._parts.values())]
        assert len(waiting) <= 1 and len(quantised) == sum(stack.codes is not None for stack in stacks)
    assert len(quantised) == len(stacks)
    model.finalize_weights()
    assert len(quantised) == len(stacks) and all(stack.weight is None and not stack._parts for stack in stacks)
    assert all((stack.bias is not None) == stack.has_bias for stack in stacks)
    late = StackedLinear([("a", 16), ("b", 16)], 32, True, torch.bfloat16, "cpu", interleave=0, weight_format="fp8")
    for name in ("b.bias", "b.weight", "a.bias", "a.weight"):
        late.assign(name, torch.full((16, 32) if "weight" in name else (16,), 1.0 if name[0] == "a" else 2.0))
    late.finalize_weights()
    assert torch.equal(quantised[-1][:, 0], late.bias) and late.bias.tolist() == [1.0] * 16 + [2.0] * 16
    with pytest.raises(KeyError):
        lacking = StackedLinear([("a", 16), ("b", 16)], 32, False, torch.bfloat16, "cpu", weight_format="fp8")
        lacking.assign("a.weight", torch.zeros(16, 32))
        lacking.finalize_weights()


@pytest.mark.parametrize("heads, kv_heads, dim, window", [(8, 8, 128, None), (32, 8, 128, None), (40, 8, 128, None), (28, 4, 128, None), (64, 4, 128, None), (64, 8, 64, None), (20, 1, 128, None), (16, 1, 256, None),
                                                          (24, 8, 96, None), (32, 8, 128, 1000), (40, 8, 64, 128)])
def test_an_engine_asks_for_the_ranges_that_a_call_by_itself_takes(heads, kv_heads, dim, window):
    """One answer for every length with the same next power of two, with a window as without: a captured step serves all of them."""
    from dataclasses import replace

    from tau_rs_b200 import DecoderModel

    spec = tiny_spec("B")
    spec = replace(spec, blocks=tuple(replace(block, mixer=replace(block.mixer, n_heads=heads, n_kv_heads=kv_heads, head_dim=dim, window=window, qk_norm=None, position=None)) for block in spec.blocks))
    model = DecoderModel(spec, torch.bfloat16, "cpu")
    passes = -(-(heads // kv_heads) // (16 if heads // kv_heads > 8 and dim <= 128 else 8))
    for n_seqs, length in [(1, 300), (4, 1000), (8, 2048), (8, 16000), (2, 120000), (40, 6000), (1, 64)]:
        wanted = kernels.decode8_splits(n_seqs, min(length, window) if window else length, kv_heads * passes)
        assert model.decode_splits(n_seqs, length, eight_bit=True) == wanted
        bucket = 1 << (length - 1).bit_length()
        assert all(model.decode_splits(n_seqs, other, eight_bit=True) == wanted for other in (bucket // 2 + 1, bucket))
    if (heads, kv_heads) == (40, 8) and not window:      # once half as many, from the blocks of the 16-bit kernel
        assert [model.decode_splits(n, length, eight_bit=True) for n, length in ((2, 120000), (8, 2048), (4, 1000), (8, 16000))] == [37, 4, 4, 8]


def test_a_model_of_several_windows_takes_the_ranges_of_the_layer_that_wants_most():
    from dataclasses import replace

    from tau_rs_b200 import DecoderModel

    spec = tiny_spec("B")
    blocks = [replace(block, mixer=replace(block.mixer, window=window)) for block, window in zip(spec.blocks, (64, None, 200))]
    schedule = [replace(entry, cache_group=f"g{index}", cache_layer=0) for index, entry in enumerate(spec.schedule)]
    model = DecoderModel(replace(spec, blocks=tuple(blocks), schedule=tuple(schedule)), torch.bfloat16, "cpu")
    assert model.decode_splits(1, 5000, eight_bit=True) == kernels.decode8_splits(1, 5000, 1) > kernels.decode8_splits(1, 200, 1)


@pytest.mark.parametrize("source", ["attention_decode8.cu", "eight_bit.cu", "gemm8_skinny.cu", "gemm8_tc.cu"])
def test_rules_of_launches_ask_the_device_for_its_multiprocessors(source):
    """No count of this machine stands in the code (comments say what was measured on it)."""
    import os
    import re

    path = os.path.join(os.path.dirname(os.path.abspath(kernels.__file__)), source)
    code = re.sub(r"//[^\n]*", "", open(path).read())
    assert not re.search(r"\b148", code) and "MultiProcessorCount" in code


def test_every_launch_is_booked_under_a_class():
    """A traced run shows milliseconds by class: what is launched under a name without one would count as something else."""
    import ast

    with open(kernels.__file__) as handle:
        tree = ast.parse(handle.read())
    names = {call.args[1].value for call in ast.walk(tree) if isinstance(call, ast.Call) and getattr(call.func, "id", "") == "_check" and isinstance(call.args[1], ast.Constant)}
    assert "linear8" in names and not names - set(kernels._CLASS_OF)


@pytest.mark.parametrize("order", [(0, 1, 0), (1, 0, 1), (0, 0, 1)])
def test_layers_of_two_kinds_share_a_cache_group(order):
    """Attention can work on a cache in 8 bits and masked attention cannot; what they keep is the same: one group, held in the run's dtype."""
    from dataclasses import replace

    from tau_rs_b200 import DecoderModel, SequenceCache
    from tau_rs_b200.config import MaskedAttentionSpec

    spec = tiny_spec("B")
    mixers = (replace(spec.blocks[0].mixer, n_heads=4, n_kv_heads=2, head_dim=64, qk_norm=None, position=None),
              MaskedAttentionSpec(hidden=spec.hidden, n_heads=4, n_kv_heads=2, dim=64, value_dim=64, softmax_scale=0.125))
    model = DecoderModel(replace(spec, blocks=tuple(replace(block, mixer=mixers[kind]) for block, kind in zip(spec.blocks, order))), torch.bfloat16, "cpu")
    (need, layers), = model.cache_groups().values()
    assert layers == 3 and not need.eight_bit
    SequenceCache(model.cache_groups(), 256, 256, torch.bfloat16, "cpu")
    with pytest.raises(ValueError, match="run's dtype"):
        SequenceCache(model.cache_groups(), 256, 256, torch.bfloat16, "cpu", cache_format="fp8")
    alone = DecoderModel(replace(spec, blocks=tuple(replace(block, mixer=mixers[0]) for block in spec.blocks)), torch.bfloat16, "cpu")
    assert all(need.eight_bit for need, _ in alone.cache_groups().values())
    narrow = replace(mixers[1], dim=32, value_dim=32)
    with pytest.raises(ValueError, match="different needs"):
        DecoderModel(replace(spec, blocks=tuple(replace(block, mixer=mixer) for block, mixer in zip(spec.blocks, (mixers[0], narrow, mixers[0])))), torch.bfloat16, "cpu")


def test_a_model_with_a_rule_of_its_own_for_ranges_serves_a_cache_in_16_bits():
    """`decode_splits(n_seqs, max_len)` is what an engine asks of any model; only a cache in 8 bits asks for more."""
    from tau_rs_b200 import DecoderModel, Engine

    class Fixed(DecoderModel):
        def decode_splits(self, n_seqs, max_len):
            return 3

    assert Engine(Fixed(tiny_spec("B"), torch.bfloat16, "cpu"), 256).decode_splits(2, 100) == 3
    engine = Engine(DecoderModel(tiny_spec("B"), torch.bfloat16, "cpu"), 256, cache_format="fp8")
    assert engine.decode_splits(1, 5000) == kernels.decode8_splits(1, 5000, 1)


def test_whoever_chooses_weights_in_8_bits_is_told_of_the_activations():
    from tau_rs_b200 import api
    from tau_rs_b200.cli import build_parser
    from tau_rs_b200.config.specs import with_weight_format

    help_text = " ".join(build_parser().format_help().split())
    assert "products' activations rounded to 8 bits" in help_text
    assert "round their inputs to 8 bits" in api.load_model.__doc__ and "activations" in api.generate.__doc__ and "activations" in with_weight_format.__doc__


@pytest.mark.parametrize("product, first", [(kernels.gemm8_stream, ()), (kernels.gemm8_tc, (torch.ones(1, 3),)), (kernels.linear8, ())])
def test_products_refuse_operands_of_one_dimension(product, first):
    operands = product_operands()
    values = operands["values"] if not first else torch.zeros(3, 32, dtype=torch.uint8).view(CODES)
    for wrong in ((values[0], operands["codes"]), (values, operands["codes"][0])):
        with pytest.raises(kernels.KernelError, match="shapes"):
            product(wrong[0], *first, wrong[1], operands["scales"], None, operands["out"])
