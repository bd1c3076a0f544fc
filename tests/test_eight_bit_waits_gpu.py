"""Operands in 8 bits that never come: the kernels end within the limit, say so, and leave the output as it was."""
import pytest
import torch

import test_eight_bit_gpu as eight
from tau_rs_b200.csrc import build, kernels

pytestmark = pytest.mark.gpu


@pytest.fixture
def lost_rank(monkeypatch):
    """Every library that is loaded meanwhile is one in which nothing arrives in the second block of each cluster, and a wait gives up after a millisecond."""
    lost = ("TAU_LOST_COPIES", "TAU_WAIT_LIMIT_NS=1000000ull", "TAU_LOST_RANK=1")
    monkeypatch.setattr(build, "load_library", lambda source, defines=(), load=build.load_library: load(source, (*defines, *lost)))
    monkeypatch.setattr(kernels, "_functions", {})
    monkeypatch.setattr(kernels, "_decode8_functions", {})


@pytest.mark.parametrize("tile", [128, 192, 256])
def test_products_whose_ranges_meet_in_a_cluster(lost_rank, tile):
    """Four ranges of K, one of which gives up: no block of the cluster stores a sum that lacks it."""
    codes, w_codes = torch.zeros(64, 2048, device="cuda").to(eight.CODES), torch.zeros(256, 2048, device="cuda").to(eight.CODES)
    out = torch.full((64, 256), 7.0, device="cuda")
    kernels.gemm8_tc(codes, torch.ones(16, 64, device="cuda"), w_codes, torch.ones(2, 16, device="cuda"), None, out, features=tile, ranges=4)
    assert kernels.gemm8_tc_status() == 1 and bool((out == 7.0).all())


@pytest.mark.parametrize("heads, dim", [(8, 64), (32, 128)])
def test_attention_whose_ranges_meet_in_a_cluster(lost_rank, heads, dim):
    """Ranges of a sequence, and of a run of new tokens: the others wait for the one that gives up, and nobody stores."""
    pages = [torch.zeros(8, 2, 64, dim, device="cuda").to(eight.CODES) for _ in range(2)] + [torch.ones(8, 2, device="cuda") for _ in range(2)]
    table = torch.arange(8, dtype=torch.int32, device="cuda")[None]
    for run in ([(499, 1)], [(495, 2)]):
        queries = torch.zeros(run[0][1], heads * dim, device="cuda", dtype=torch.bfloat16)
        out, step = torch.full_like(queries, 7.0), eight.make_step(run)
        step.decode_splits = 4
        kernels.attention_decode8(queries, *pages, out, step, table, heads, 2, dim, dim ** -0.5, 0)
        assert build.load_library("attention_decode8.cu", (f"TAU_HEAD_DIM={dim}",)).tau_decode8_status() == 1 and bool((out == 7.0).all())


@pytest.mark.parametrize("heads, dim", [(8, 64), (32, 128)])
def test_attention_whose_ranges_meet_through_memory(monkeypatch, heads, dim):
    """Sixteen ranges leave records for a second kernel, and one of them gives up: what it is missing from stays as it was, a sequence that has no page there is complete."""
    lost = ("TAU_LOST_COPIES", "TAU_WAIT_LIMIT_NS=1000000ull", "TAU_LOST_RANGE=1")
    torch.manual_seed(0)
    pages = [torch.randn(33, 2, 64, dim, device="cuda").to(eight.CODES) for _ in range(2)] + [torch.ones(33, 2, device="cuda") for _ in range(2)]
    table = torch.zeros(3, 16, dtype=torch.int32, device="cuda")
    table[0], table[1, 0], table[2] = torch.arange(16), 16, torch.arange(17, 33)
    runs = [(1000, 1), (40, 1), (1023, 1)]
    queries = torch.randn(3, heads * dim, device="cuda").to(torch.bfloat16)
    out, wanted = (torch.full_like(queries, 7.0) for _ in range(2))
    step = eight.make_step(runs)
    step.decode_splits = 16
    kernels.attention_decode8(queries, *pages, wanted, step, table, heads, 2, dim, dim ** -0.5, 0)
    torch.cuda.synchronize()
    assert not bool((wanted == 7.0).all(1).any())
    monkeypatch.setattr(build, "load_library", lambda source, defines=(), load=build.load_library: load(source, (*defines, *lost)))
    monkeypatch.setattr(kernels, "_functions", {})
    monkeypatch.setattr(kernels, "_decode8_functions", {})
    kernels.attention_decode8(queries, *pages, out, step, table, heads, 2, dim, dim ** -0.5, 0)
    assert build.load_library("attention_decode8.cu", (f"TAU_HEAD_DIM={dim}",)).tau_decode8_status() == 1
    assert bool((out[0] == 7.0).all()) and bool((out[2] == 7.0).all()) and torch.equal(out[1], wanted[1])
