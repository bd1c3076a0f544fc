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
