"""Products of weights in 8 bits, the cache in 8 bits and the attention over it, against plain statements in 64-bit."""
import pytest
import torch

import plain_eight_bit as plain
from tau_rs_b200.csrc import build, kernels
from tau_rs_b200.engine.batch import StepContext

pytestmark = pytest.mark.gpu
CODES = torch.float8_e4m3fn


def spread_values(*shape, seed, outliers=True):
    """Normal values whose rows, and a few of whose elements, differ by powers of ten."""
    random = torch.Generator().manual_seed(seed)
    values = torch.randn(*shape, generator=random) * torch.exp(2.0 * torch.randn(shape[0], *[1] * (len(shape) - 1), generator=random))
    if outliers:
        values = torch.where(torch.rand(*shape, generator=random) < 0.01, values * 300.0, values)
    return values


# ---- quantising --------------------------------------------------------------------------------------------------------------------
@pytest.mark.parametrize("rows, columns", [(1, 16), (128, 128), (130, 272), (300, 1040)])
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
def test_quantising_is_the_statement_bit_for_bit(rows, columns, dtype):
    """Whole and cut blocks, a block of zeros, magnitudes at the borders of a scale, infinities and NaN."""
    weight = spread_values(rows, columns, seed=rows).to(dtype)
    if rows > 2:
        weight[:128, :128] = 0.0
        weight[1, 5], weight[rows - 1, columns - 1], weight[rows - 1, 3] = 448.0, float("inf"), float("nan")
        weight[2, 20] = 2.0 ** -130
    for found, (held, scales), spread in (
            (kernels.quantize_blocks(weight.cuda()), plain.held_blocks(weight), lambda s: s.repeat_interleave(128, 0).repeat_interleave(128, 1)[:rows, :columns]),
            (kernels.quantize_rows(weight.cuda()), plain.held_rows(weight), lambda s: s.T.repeat_interleave(128, 1)[:, :columns])):
        codes, found_scales = found
        assert torch.equal(found_scales.cpu().double(), scales)
        assert torch.equal(torch.nan_to_num(codes.cpu().double() * spread(scales), nan=1e30), torch.nan_to_num(held, nan=1e30))


# ---- products ----------------------------------------------------------------------------------------------------------------------
def product_bound(x, w, exact, out_dtype):
    """Codes and products of two codes are exact in 32 bits.  Inside a block of 128 columns at most 128 sums lose a unit of 2^-23 of the sum of magnitudes (a tensor core may cut where
    a plain sum rounds); each block's sum is scaled and added, and the result stored."""
    blocks = -(-x.shape[1] // 128)
    lost = (128 * 2.0 ** -23 + (blocks + 3) * 2.0 ** -24) * (x.abs() @ w.abs().T)
    return lost + (2.0 ** -8 * (exact.abs() + lost) if out_dtype == torch.bfloat16 else 2.0 ** -24 * exact.abs()) + 1e-37


SIZES = [(1, 16, 16), (1, 1024, 4096), (3, 144, 130), (7, 2000, 257), (8, 4096, 528), (9, 272, 1000), (16, 1104, 384), (17, 128, 2048), (33, 1040, 300), (64, 2048, 512),
         (100, 416, 1500), (128, 256, 256), (129, 640, 272), (200, 4112, 640), (257, 1024, 1040), (600, 528, 2064), (4, 12416, 144), (14, 12416, 130)]


@pytest.mark.parametrize("rows, depth, features", SIZES)
@pytest.mark.parametrize("out_dtype, bias", [(torch.float32, True), (torch.bfloat16, False)])
def test_products(rows, depth, features, out_dtype, bias):
    x, w = spread_values(rows, depth, seed=depth).to(torch.bfloat16), spread_values(features, depth, seed=features).to(torch.bfloat16)
    offset = spread_values(features, seed=3, outliers=False) if bias else None
    wide = torch.full((rows, features + 24), 7.0, device="cuda", dtype=out_dtype)
    out = wide[:, :features]      # rows of a wider tensor
    kernels.linear8(x.cuda(), *kernels.quantize_blocks(w.cuda()), offset.cuda() if bias else None, out)
    held_x, held_w = plain.held_rows(x)[0].cuda(), plain.held_blocks(w)[0].cuda()
    exact = held_x @ held_w.T + (offset.double().cuda() if bias else 0.0)
    bound = product_bound(held_x, held_w, exact, out_dtype) + (2.0 ** -24 * exact.abs().max() if bias else 0.0)
    assert bool(((out.double() - exact).abs() <= bound).all()), float(((out.double() - exact).abs() / bound).max())
    assert bool((wide[:, features:] == 7.0).all())


@pytest.mark.parametrize("rows, depth, inner", [(1, 64, 8), (1, 1024, 1024), (5, 272, 200), (8, 1040, 1408), (13, 512, 264), (40, 1024, 520), (128, 144, 128), (300, 1104, 1000)])
@pytest.mark.parametrize("limit", [0.0, 2.0])
def test_gated_products(rows, depth, inner, limit):
    x = spread_values(rows, depth, seed=inner, outliers=False).to(torch.bfloat16)
    w = (spread_values(2 * inner, depth, seed=depth, outliers=False) * depth ** -0.5).to(torch.bfloat16)
    out = torch.full((rows, inner), 7.0, device="cuda", dtype=torch.bfloat16)
    kernels.linear8_gated(x.cuda(), *kernels.quantize_blocks(w.cuda()), out, limit=limit)
    held_x, held_w = plain.held_rows(x)[0].cuda(), plain.held_blocks(w)[0].cuda()
    pairs = (held_x @ held_w.T)
    slack = product_bound(held_x, held_w, pairs, torch.bfloat16)
    (gate, up), (gate_off, up_off) = ([t.view(rows, -1, 2, 8)[:, :, i].reshape(rows, -1) for i in (0, 1)] for t in (pairs, slack))
    if limit:      # g sigmoid(1.702 g) (u + 1): the slope of the first factor is below 1.1, the clamps have slope one at most
        g, u = gate.clamp(max=limit), up.clamp(-limit, limit) + 1.0
        first, second = g * torch.sigmoid(1.702 * g), u
    else:
        first, second = gate * torch.sigmoid(gate), up
    exact = first * second
    # The factors move by 1.1 times the gate's error (the greatest slope of x sigmoid(a x)) and by the up value's; fast exponential and quotient are good to 2^-20; one rounding.
    d1, d2 = 1.1 * gate_off + 2.0 ** -20 * first.abs(), up_off + 2.0 ** -23
    bound = d1 * second.abs() + d2 * first.abs() + d1 * d2
    bound = bound + 2.0 ** -8 * (exact.abs() + bound) + 1e-37
    assert bool(((out.double() - exact).abs() <= bound).all()), float(((out.double() - exact).abs() / bound).max())


@pytest.mark.parametrize("rows, depth, features", [(1, 16, 16), (100, 1040, 530), (300, 400, 272), (513, 1296, 800)])
@pytest.mark.parametrize("tile, ranges", [(128, 1), (128, 2), (128, 3), (128, 7), (128, 8), (192, 1), (192, 3), (192, 8), (256, 1), (256, 2), (256, 5)])
def test_every_tile_of_the_tensor_core_product(rows, depth, features, tile, ranges):
    """Each width of tile, ranges of K (more than there are blocks of K too), ungated in both types and gated, into rows of a wider tensor."""
    x, w = spread_values(rows, depth, seed=depth, outliers=False).to(torch.bfloat16), (spread_values(features, depth, seed=features, outliers=False) * depth ** -0.5).to(torch.bfloat16)
    x_codes, x_scales = kernels.quantize_rows(x.cuda())
    codes, scales = kernels.quantize_blocks(w.cuda())
    held_x, held_w = plain.held_rows(x)[0].cuda(), plain.held_blocks(w)[0].cuda()
    exact = held_x @ held_w.T
    for out_dtype, apart in ((torch.float32, 8), (torch.bfloat16, 3)):
        wide = torch.full((rows, features + apart), 7.0, device="cuda", dtype=out_dtype)
        kernels.gemm8_tc(x_codes, x_scales, codes, scales, None, wide[:, :features], features=tile, ranges=ranges)
        assert bool(((wide[:, :features].double() - exact).abs() <= product_bound(held_x, held_w, exact, out_dtype)).all()) and bool((wide[:, features:] == 7.0).all())
    if features % 16 == 0:
        stacked, out = torch.empty(rows, features, device="cuda", dtype=torch.bfloat16), torch.full((rows, features // 2 + 8), 7.0, device="cuda", dtype=torch.bfloat16)
        kernels.gemm8_tc(x_codes, x_scales, codes, scales, None, stacked, features=tile, ranges=ranges)
        kernels.gemm8_tc(x_codes, x_scales, codes, scales, None, out[:, : features // 2], gated=True, features=tile, ranges=ranges)
        pairs = stacked.double().view(rows, -1, 2, 8)
        gate, up = (pairs[:, :, i].reshape(rows, -1) for i in (0, 1))
        wanted = torch.nn.functional.silu(gate) * up
        # The same roundings before the activation.  __expf(x) is documented to be within 2 + 1.173 |x| units of 2^-23, the quotient within 2, the sum and the product are rounded once each
        # (2^-24), and the quotient of a denominator above 2^126 may be 0 (a gate below -87: the result is smaller than 2^-126 |g u|).
        bound = (2.0 ** -8 + 2.0 ** -23 * (6.0 + 1.173 * gate.abs())) * wanted.abs() + 2.0 ** -126 * (gate * up).abs() + 1e-37
        assert bool(((out[:, : features // 2].double() - wanted).abs() <= bound).all()), float(((out[:, : features // 2].double() - wanted).abs() / bound).max())
        assert bool((out[:, features // 2 :] == 7.0).all())
    assert kernels.gemm8_tc_status() == 0


@pytest.mark.parametrize("rows, depth, features", [(1, 16, 16), (8, 4096, 530), (3, 400, 4112), (7, 12288, 272), (5, 2064, 5000), (2, 12176, 40)])
def test_the_streaming_product(rows, depth, features):
    """One group of features and many to a block, fewer chunks of K than warps, a last chunk that is cut, the deepest K; against the statement, and gated against itself."""
    x, w = spread_values(rows, depth, seed=depth, outliers=False).to(torch.bfloat16), (spread_values(features, depth, seed=features, outliers=False) * depth ** -0.5).to(torch.bfloat16)
    offset = spread_values(features, seed=3, outliers=False).cuda()
    codes, scales = kernels.quantize_blocks(w.cuda())
    held_x, held_w = plain.held_rows(x)[0].cuda(), plain.held_blocks(w)[0].cuda()
    exact = held_x @ held_w.T + offset.double()
    wide = torch.zeros(rows, depth + 16, dtype=torch.bfloat16, device="cuda")
    wide[:, :depth] = x.cuda()
    assert build.load_library("gemm8_skinny.cu").tau_gemm8_stream_most_depth() >= kernels.STREAM8_MAX_DEPTH
    for out_dtype in (torch.float32, torch.bfloat16):
        out = torch.full((rows, features + 3), 7.0, device="cuda", dtype=out_dtype)
        kernels.gemm8_stream(wide[:, :depth], codes, scales, offset, out[:, :features])
        bound = product_bound(held_x, held_w, exact, out_dtype) + 2.0 ** -24 * exact.abs().max()
        assert bool(((out[:, :features].double() - exact).abs() <= bound).all()) and bool((out[:, features:] == 7.0).all())
    if features % 16 == 0:
        stacked, out = torch.empty(rows, features, device="cuda", dtype=torch.bfloat16), torch.empty(rows, features // 2, device="cuda", dtype=torch.bfloat16)
        kernels.gemm8_stream(wide[:, :depth], codes, scales, None, stacked)
        kernels.gemm8_stream(wide[:, :depth], codes, scales, None, out, gated=True)
        gate, up = (stacked.double().view(rows, -1, 2, 8)[:, :, i].reshape(rows, -1) for i in (0, 1))
        wanted = torch.nn.functional.silu(gate) * up
        bound = (2.0 ** -8 + 2.0 ** -23 * (6.0 + 1.173 * gate.abs())) * wanted.abs() + 2.0 ** -126 * (gate * up).abs() + 1e-37      # as above
        assert bool(((out.double() - wanted).abs() <= bound).all())


@pytest.mark.parametrize("rows", [1, 12, 40, 300])
def test_a_product_directly_behind_its_weights_quantising(rows):
    """Codes land where the weight before had its own: a product that asked for them too early would multiply with those."""
    x = torch.randn(rows, 4096, device="cuda").to(torch.bfloat16)
    weights = [(torch.randn(6144, 4096, device="cuda") * 4.0 ** turn).to(torch.bfloat16) for turn in range(4)]
    wanted = []
    for weight in weights:
        held = kernels.quantize_blocks(weight)
        torch.cuda.synchronize()
        out = torch.empty(rows, 6144, device="cuda")
        kernels.linear8(x, *held, None, out)
        wanted.append(out)
        del held
    for weight, result in zip(weights, wanted):
        out = torch.empty(rows, 6144, device="cuda")
        held = kernels.quantize_blocks(weight)
        kernels.linear8(x, *held, None, out)
        del held
        assert torch.equal(out, result)


def test_a_row_that_is_not_finite_stays_alone():
    """An infinity and a NaN in two rows make those rows' results NaN and leave the others as they are; so does a NaN in a weight's row for its feature."""
    for rows in (4, 40, 300):
        x, w = torch.randn(rows, 512, device="cuda").to(torch.bfloat16), torch.randn(256, 512, device="cuda").to(torch.bfloat16)
        clean, out = (torch.empty(rows, 256, device="cuda") for _ in range(2))
        kernels.linear8(x, *kernels.quantize_blocks(w), None, clean)
        x[1, 7], x[2, 500] = float("inf"), float("nan")
        kernels.linear8(x, *kernels.quantize_blocks(w), None, out)
        assert bool(out[1:3].isnan().all()) and torch.equal(out[0], clean[0]) and torch.equal(out[3:], clean[3:])
        w[9, 100] = float("nan")
        kernels.linear8(x, *kernels.quantize_blocks(w), None, out)
        assert bool(out[:, 9].isnan().all()) and torch.equal(out[3:, 10:], clean[3:, 10:])


def test_products_without_rows_and_scales_that_are_no_powers_of_two():
    codes, scales = kernels.quantize_blocks(torch.randn(256, 256, device="cuda"))
    kernels.linear8(torch.empty(0, 256, device="cuda", dtype=torch.bfloat16), codes, scales, None, torch.empty(0, 256, device="cuda"))
    kernels.linear8_gated(torch.empty(0, 256, device="cuda", dtype=torch.bfloat16), codes, scales, torch.empty(0, 128, device="cuda", dtype=torch.bfloat16))
    scales = torch.rand_like(scales) + 0.3
    for rows in (2, 50, 300):
        x = torch.randn(rows, 256, device="cuda").to(torch.bfloat16)
        out = torch.empty(rows, 256, device="cuda")
        kernels.linear8(x, codes, scales, None, out)
        held_x, held_w = plain.held_rows(x.cpu())[0].cuda(), codes.double() * scales.double().repeat_interleave(128, 0).repeat_interleave(128, 1)
        exact = held_x @ held_w.T
        assert bool(((out.double() - exact).abs() <= 2.0 * product_bound(held_x, held_w, exact, torch.float32)).all())      # the scales' product is rounded too


def test_activations_in_32_bits_and_a_captured_product():
    """float32 activations; a captured call replayed on new inputs, on another stream than it was captured on, beside an eager call of the same kernel."""
    w = kernels.quantize_blocks(torch.randn(512, 1024, device="cuda"))
    for rows in (3, 24, 260):
        x = torch.randn(rows, 1024, device="cuda")
        wide, narrow = (torch.empty(rows, 512, device="cuda") for _ in range(2))
        kernels.linear8(x.to(torch.bfloat16).float(), *w, None, wide)
        kernels.linear8(x.to(torch.bfloat16), *w, None, narrow)
        assert torch.allclose(wide, narrow, rtol=1e-5, atol=1e-4 * float(narrow.abs().max()))
        held, out = torch.empty(rows, 1024, device="cuda", dtype=torch.bfloat16), torch.empty(rows, 512, device="cuda")
        held.copy_(x)
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            kernels.linear8(held, *w, None, out)
        other = torch.cuda.Stream()
        held.copy_(-x)
        other.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(other):
            graph.replay()
        again = torch.empty_like(out)
        kernels.linear8(held, *w, None, again)
        torch.cuda.synchronize()
        assert torch.equal(out, again)


# ---- the cache ---------------------------------------------------------------------------------------------------------------------
def ints(values):
    return torch.tensor(values, dtype=torch.int32, device="cuda")


def make_step(runs):
    bounds = [0]
    for _, new in runs:
        bounds.append(bounds[-1] + new)
    positions = [p for start, new in runs for p in range(start, start + new)]
    owners = [i for i, (_, new) in enumerate(runs) for _ in range(new)]
    lengths = [start + new for start, new in runs]
    return StepContext(n_tokens=bounds[-1], n_seqs=len(runs), n_wanted=0, token_ids=ints(positions), positions=ints(positions), token_seq=ints(owners), want_rows=ints([]),
                       cu_seqlens=ints(bounds), seq_slot=ints(range(len(runs))), seq_start=ints([s for s, _ in runs]), seq_len=ints(lengths), page_rows={}, max_new=max(n for _, n in runs),
                       max_len=max(lengths), all_single=all(n == 1 for _, n in runs), min_new=min(n for _, n in runs), all_fresh=all(s == 0 for s, _ in runs))


class Cache:
    """Pages of the library beside the plain statement's; what nobody wrote is NaN in the codes and in the scales."""

    def __init__(self, pages, heads, dim, counts, seed=0):
        self.keys, self.values = (torch.full((pages, heads, 64, dim), 0x7F, dtype=torch.uint8, device="cuda").view(CODES) for _ in range(2))
        self.key_scales, self.value_scales = (torch.full((pages, heads), float("nan"), device="cuda") for _ in range(2))
        self.plain_keys, self.plain_values = plain.Pages(pages, heads, dim), plain.Pages(pages, heads, dim)
        order = torch.randperm(pages, generator=torch.Generator().manual_seed(seed)).tolist()
        self.table = torch.zeros(len(counts), max(max(counts), 1), dtype=torch.int32)
        for index, count in enumerate(counts):
            self.table[index, :count] = torch.tensor([order.pop() for _ in range(count)], dtype=torch.int32)
        self.rows = self.table.cuda()

    @property
    def pages(self):
        return self.keys, self.values, self.key_scales, self.value_scales

    def store(self, runs, keys, values, **more):
        kernels.cache8_store(keys.cuda(), values.cuda(), *self.pages, make_step(runs), self.rows, **more)
        first = 0
        for index, (start, new) in enumerate(runs):
            self.plain_keys.store_run(self.table[index], start, keys[first : first + new])
            self.plain_values.store_run(self.table[index], start, values[first : first + new])
            first += new

    def check(self, runs):
        keys, values = kernels.cache8_read(*self.pages, make_step(runs), self.rows)
        stride = self.table.shape[1]
        for index, (start, new) in enumerate(runs):
            length = start + new
            for found, wanted in ((keys, self.plain_keys), (values, self.plain_values)):
                mine = found[index * stride : (index + 1) * stride].cpu().double().transpose(0, 1).reshape(found.shape[1], -1, found.shape[3])
                held = wanted.sequence(self.table[index], length)
                assert torch.equal(torch.nan_to_num(mine[:, :length], nan=1e30), torch.nan_to_num(held, nan=1e30)), index
                assert bool((mine[:, length:] == 0).all()), index


def random_rows(tokens, heads, dim, seed):
    return spread_values(tokens, heads, dim, seed=seed).to(torch.bfloat16), spread_values(tokens, heads, dim, seed=seed + 1).to(torch.bfloat16)


@pytest.mark.parametrize("heads, dim", [(1, 16), (2, 48), (3, 80), (8, 128), (2, 256)])
def test_the_store_is_the_statement_bit_for_bit(heads, dim):
    """Runs that start and end inside pages, single tokens, a run over several pages, scales that grow, one that stays, zeros, infinities and NaN, forty sequences."""
    runs = [(0, 1), (0, 64), (0, 65), (0, 200), (0, 7)] + [(0, 1 + index % 5) for index in range(35)]
    cache = Cache(90, heads, dim, [5] * 5 + [1] * 35)
    lengths = [0] * 40
    for turn, news in enumerate([[new for _, new in runs], [63, 1, 1, 55, 120] + [2] * 35, [1] * 40, [40, 3, 130, 1, 9] + [1] * 35]):
        now = [(length, new) for length, new in zip(lengths, news)]
        keys, values = random_rows(sum(news), heads, dim, 10 * turn)
        if turn == 1:
            keys[5, 0, 3], values[70, 0, 1], keys[80:90] = float("inf"), float("nan"), 0.0
        cache.store(now, keys, values)
        cache.check(now)
        lengths = [length + new for length, new in zip(lengths, news)]


def test_the_store_reads_keys_and_values_inside_wider_rows_and_leaves_other_pages_alone():
    cache = Cache(6, 2, 32, [2, 2])
    runs = [(0, 70), (0, 3)]
    wide = spread_values(73, 256, seed=4).to(torch.bfloat16).cuda()
    keys, values = wide[:, 64:128].view(73, 2, 32), wide[:, 128:192].view(73, 2, 32)
    kernels.cache8_store(keys, values, *cache.pages, make_step(runs), cache.rows)
    straight = Cache(6, 2, 32, [2, 2])
    straight.store(runs, keys.cpu(), values.cpu())
    straight.check(runs)
    for found, wanted in zip(cache.pages, straight.pages):
        assert torch.equal(found.view(torch.uint8), wanted.view(torch.uint8))
    used = set(cache.table[0].tolist()) | {int(cache.table[1, 0])}
    for page in set(range(6)) - used:
        assert bool((cache.keys[page].view(torch.uint8) == 0x7F).all()) and bool(cache.key_scales[page].isnan().all())


@pytest.mark.parametrize("n_heads, n_kv_heads, dim, rotary, normed", [(4, 2, 32, 32, True), (6, 2, 80, 40, True), (8, 8, 128, 128, True), (2, 1, 64, 0, False), (9, 3, 256, 256, False), (4, 4, 64, 64, True), (4, 2, 96, 96, True), (2, 2, 256, 256, True)])
def test_preparing_and_storing_equals_the_prepare_kernel_and_a_store(n_heads, n_kv_heads, dim, rotary, normed):
    runs = [(0, 75), (30, 1), (64, 2), (100, 60)]
    tokens = sum(new for _, new in runs)
    step = make_step(runs)
    projected = torch.randn(tokens, (n_heads + 2 * n_kv_heads) * dim, device="cuda").to(torch.bfloat16)
    weights = [torch.rand(dim, device="cuda") + 0.5 if normed else None for _ in range(2)]
    angles = torch.rand(256, rotary // 2, device="cuda") * 6 if rotary else None
    cos, sin = (angles.cos(), angles.sin()) if rotary else (None, None)
    queries, wanted_queries = (torch.empty(tokens, n_heads * dim, device="cuda", dtype=torch.bfloat16) for _ in range(2))
    cache, straight = Cache(12, n_kv_heads, dim, [3] * 4), Cache(12, n_kv_heads, dim, [3] * 4)
    for each in (cache, straight):      # what the later runs continue
        each.store([(0, 1), (0, 30), (0, 64), (0, 100)], *random_rows(195, n_kv_heads, dim, 1))
    split = (projected[:, n_heads * dim : (n_heads + n_kv_heads) * dim].view(tokens, n_kv_heads, dim), projected[:, (n_heads + n_kv_heads) * dim :].view(tokens, n_kv_heads, dim))
    kernels.cache8_store(*split, *cache.pages, step, cache.rows, prepare=(projected, queries, *weights, 1e-6, cos, sin, rotary, n_heads))
    plain_pages = [torch.zeros(12, n_kv_heads, 64, dim, device="cuda", dtype=torch.bfloat16) for _ in range(2)]
    kernels.attention_prepare(projected, wanted_queries, *plain_pages, True, *weights, 1e-6, cos, sin, rotary, step.positions, step.token_seq, straight.rows, n_heads, n_kv_heads, dim)
    place = [(int(straight.table[index, p // 64]), p % 64) for index, (start, new) in enumerate(runs) for p in range(start, start + new)]
    pages, slots = torch.tensor(place).T
    kernels.cache8_store(*(t[pages.cuda(), :, slots.cuda()].contiguous() for t in plain_pages), *straight.pages, step, straight.rows)
    assert torch.equal(queries, wanted_queries)
    for found, wanted in zip(cache.pages, straight.pages):
        assert torch.equal(found.view(torch.uint8), wanted.view(torch.uint8))


# ---- attention ---------------------------------------------------------------------------------------------------------------------
def check_attention(runs, heads, kv_heads, dim, window, seed=0, dirty=True, splits=0):
    """Against the statement.  A weight of the softmax is rounded to 16 bits before it meets a value (2^-8 at most); a score is a sum of `dim` exact products in 32 bits (a unit of 2^-23
    of the sum of magnitudes each) times the scale, and moves the weights by twice its error; exponentials are good to 2^-20 and sums of weights to 2^-20; the result is rounded once."""
    counts = [-(-(start + new) // 64) for start, new in runs]
    cache = Cache(sum(counts) + 1, kv_heads, dim, counts, seed)
    whole = [(0, start + new) for start, new in runs]
    random = torch.Generator().manual_seed(seed)
    tokens = sum(length for _, length in whole)
    keys, values = torch.randn(tokens, kv_heads, dim, generator=random).to(torch.bfloat16), spread_values(tokens, kv_heads, dim, seed=seed + 5).to(torch.bfloat16)
    cache.store(whole, keys, values)
    if dirty and window:      # what a window has left behind may be anything
        for index, (start, _) in enumerate(runs):
            for position in range(0, max(0, start + 1 - window)):
                cache.keys[int(cache.table[index, position // 64]), :, position % 64].view(torch.uint8).fill_(0x7F)
                cache.values[int(cache.table[index, position // 64]), :, position % 64].view(torch.uint8).fill_(0xFF)
    new_tokens = sum(new for _, new in runs)
    queries = torch.randn(new_tokens, heads * dim, generator=random).to(torch.bfloat16)
    out = torch.full((new_tokens, heads * dim), float("nan"), device="cuda", dtype=torch.bfloat16)
    step = make_step(runs)
    step.decode_splits = splits
    scale = dim ** -0.5
    kernels.attention8(queries.cuda(), *cache.pages, out, step, cache.rows, heads, kv_heads, dim, scale, window)
    first = 0
    for index, (start, new) in enumerate(runs):
        length = start + new
        wanted, spread, reach = plain.attention(queries[first : first + new].view(new, heads, dim), cache.plain_keys.sequence(cache.table[index], length),
                                                cache.plain_values.sequence(cache.table[index], length), start, scale, window)
        found = out[first : first + new].cpu().double().view(new, heads, dim)
        lost = 2.0 ** -8 + 2.0 * (dim + 4) * 2.0 ** -23 * reach + 2.0 ** -18
        bound = lost * spread + 2.0 ** -8 * (wanted.abs() + lost * spread)
        assert bool(((found - wanted).abs() <= bound).all()), (index, float(((found - wanted).abs() / bound).max()))
        first += new


@pytest.mark.parametrize("heads, kv_heads, dim", [(1, 1, 16), (2, 2, 48), (6, 2, 80), (16, 2, 64), (8, 8, 128), (32, 8, 128), (5, 1, 96), (20, 1, 128), (4, 2, 256)])
@pytest.mark.parametrize("window", [0, 1, 70])
def test_single_tokens(heads, kv_heads, dim, window):
    """Lengths of one, around a page and over several; groups of one to twenty query heads."""
    check_attention([(length - 1, 1) for length in (1, 2, 63, 64, 65, 127, 129, 300)], heads, kv_heads, dim, window)


@pytest.mark.parametrize("splits", [1, 2, 5, 8, 16, 17, 40, 64])
def test_single_tokens_with_a_given_number_of_splits(splits):
    """More splits than pages, ranges without a position, one sequence far longer than the others."""
    check_attention([(1500, 1), (0, 1), (64, 1), (700, 1)], 8, 2, 64, 0, seed=splits, splits=splits)
    check_attention([(1500, 1), (3, 1)], 4, 1, 128, 333, seed=splits, splits=splits)
    check_attention([(600, 1), (3, 1)], 3, 3, 16, 0, seed=splits, splits=splits)


@pytest.mark.parametrize("heads, kv_heads, dim", [(4, 2, 32), (6, 2, 80), (8, 2, 64), (32, 8, 128), (12, 1, 128), (2, 1, 256)])
@pytest.mark.parametrize("window", [0, 1, 90])
def test_runs(heads, kv_heads, dim, window):
    """Fresh prompts, portions behind cached ones, single tokens among them."""
    check_attention([(0, 70), (100, 1), (60, 9), (0, 1), (130, 66), (64, 64)], heads, kv_heads, dim, window)


@pytest.mark.parametrize("directly", [0, 1])
@pytest.mark.parametrize("heads, kv_heads, dim, window", [(4, 2, 32, 0), (6, 2, 80, 90), (8, 2, 64, 1), (32, 8, 128, 0), (9, 3, 128, 33), (2, 1, 256, 70), (17, 1, 96, 0)])
def test_runs_by_either_kernel(monkeypatch, directly, heads, kv_heads, dim, window):
    """Runs worked on like single tokens and runs over pages laid out in 16 bits, whichever the rule would take: runs of one and of many tokens, a token over two blocks, ranges that no
    column of a block sees."""
    monkeypatch.setattr(kernels, "runs8_like_single_tokens", lambda *sizes: bool(directly))
    check_attention([(0, 7), (100, 1), (60, 9), (130, 66), (500, 3)], heads, kv_heads, dim, window)
    check_attention([(3000, 5), (0, 2)], heads, kv_heads, dim, window, seed=4)


@pytest.mark.parametrize("heads, kv_heads, dim, window", [(4, 2, 48, 0), (8, 2, 64, 90), (4, 1, 128, 0)])
def test_runs_whose_pages_are_read_back_a_few_sequences_at_a_time(monkeypatch, heads, kv_heads, dim, window):
    """Room for two sequences at a time, then for less than one: the result of each is that of all at once."""
    monkeypatch.setattr(kernels, "runs8_like_single_tokens", lambda *sizes: False)
    for room in (2, 0):
        monkeypatch.setattr(kernels, "READ8_BYTES", room * 4 * 4 * 64 * kv_heads * dim)      # the longest has four pages
        check_attention([(0, 70), (100, 1), (60, 9), (0, 1), (130, 66)], heads, kv_heads, dim, window)


@pytest.mark.parametrize("directly", [0, 1])
@pytest.mark.parametrize("kv_heads, dim", [(2, 32), (1, 64), (2, 128), (1, 256)])
def test_what_later_tokens_hold_reaches_no_earlier_one(monkeypatch, directly, kv_heads, dim):
    """A key and a value of new tokens that are not finite: the tokens before them are as without them, those behind see NaN."""
    monkeypatch.setattr(kernels, "runs8_like_single_tokens", lambda *sizes: bool(directly))
    torch.manual_seed(dim)
    for at, what in ((40, "key"), (41, "value")):
        results = []
        for spoiled in (False, True):
            cache = Cache(4, kv_heads, dim, [2, 1])
            keys, values = random_rows(110, kv_heads, dim, 3)
            if spoiled:
                (keys if what == "key" else values)[at] = float("nan")
            cache.store([(0, 100), (0, 10)], keys, values)
            queries = torch.randn(110, 2 * kv_heads * dim, generator=torch.Generator().manual_seed(1)).to(torch.bfloat16).cuda()
            out = torch.empty_like(queries)
            kernels.attention8(queries, *cache.pages, out, make_step([(0, 100), (0, 10)]), cache.rows, 2 * kv_heads, kv_heads, dim, dim ** -0.5, 0)
            results.append(out.float())
        assert torch.equal(results[0][:at], results[1][:at]) and torch.equal(results[0][100:], results[1][100:]) and bool(results[1][at:100].isnan().all())


def test_many_single_tokens_and_a_long_context():
    check_attention([(index * 7 % 150, 1) for index in range(70)], 8, 4, 64, 0, seed=2)
    check_attention([(9000, 1)], 2, 1, 64, 0, seed=3)


@pytest.mark.parametrize("sequences", [2, 31, 33, 100, 257, 1000, 1024, 1025])
def test_sequences_of_unequal_lengths(sequences):
    """The longest may start first: every sequence is still worked on once, whatever their lengths, in every class of lengths."""
    check_attention([((37 * index * index + 64 * index) % (700 if sequences > 100 else 3000), 1) for index in range(sequences)], 2, 1, 32, 0)


@pytest.mark.parametrize("n_heads, n_kv_heads, dim, rotary, normed, window", [(4, 2, 32, 32, True, 0), (8, 8, 128, 128, True, 70), (32, 4, 64, 64, True, 0), (6, 2, 80, 40, True, 1), (16, 1, 128, 0, False, 0),
                                                                               (8, 1, 256, 256, True, 100), (3, 3, 16, 8, False, 0)])
@pytest.mark.parametrize("splits", [0, 1, 3, 8, 20])
def test_single_tokens_stored_and_attended_in_one_kernel(n_heads, n_kv_heads, dim, rotary, normed, window, splits):
    """Against the store and the attention one after the other, bit for bit: pages that start, end and are in the middle, scales that grow, several steps behind each other, and a run that
    only reads what another stored."""
    lengths = [0, 1, 62, 63, 64, 130, 300]
    cache, straight = (Cache(7 * 5, n_kv_heads, dim, [5] * 7) for _ in range(2))
    keys, values = random_rows(sum(lengths), n_kv_heads, dim, 2)
    for each in (cache, straight):
        if sum(lengths):
            kernels.cache8_store(keys.cuda(), values.cuda(), *each.pages, make_step([(0, length) for length in lengths]), each.rows)
    weights = [torch.rand(dim, device="cuda") + 0.5 if normed else None for _ in range(2)]
    angles = torch.rand(512, rotary // 2, device="cuda") * 6 if rotary else None
    cos, sin = (angles.cos(), angles.sin()) if rotary else (None, None)
    for turn in range(3):
        step = make_step([(length + turn, 1) for length in lengths])
        step.decode_splits = splits
        projected = torch.randn(7, (n_heads + 2 * n_kv_heads) * dim + 8, device="cuda").to(torch.bfloat16)[:, : (n_heads + 2 * n_kv_heads) * dim] * (4.0 ** turn)
        queries, wanted, found = (torch.empty(7, n_heads * dim, device="cuda", dtype=torch.bfloat16) for _ in range(3))
        split = [projected[:, (n_heads + i * n_kv_heads) * dim : (n_heads + (i + 1) * n_kv_heads) * dim].unflatten(1, (n_kv_heads, dim)) for i in (0, 1)]
        kernels.cache8_store(*split, *straight.pages, step, straight.rows, prepare=(projected, queries, *weights, 1e-6, cos, sin, rotary, n_heads))
        kernels.attention8(queries, *straight.pages, wanted, step, straight.rows, n_heads, n_kv_heads, dim, dim ** -0.5, window)
        numbers = (*weights, 1e-6, cos, sin, rotary, n_heads, n_kv_heads, dim, dim ** -0.5, window)
        assert kernels.attention8_decode_fused(projected, *cache.pages, found, step, cache.rows, True, *numbers)
        assert torch.equal(found, wanted)
        for mine, theirs in zip(cache.pages, straight.pages):
            assert torch.equal(mine.view(torch.uint8), theirs.view(torch.uint8))
        assert kernels.attention8_decode_fused(projected[:, : n_heads * dim], *cache.pages, found.zero_(), step, cache.rows, False, *numbers) and torch.equal(found, wanted)
    assert not kernels.attention8_decode_fused(projected, *cache.pages, found, make_step([(0, 2)] * 7), cache.rows, True, *numbers)


def test_attention_of_a_captured_step():
    """Captured over one set of lengths and replayed over another on another stream, beside an eager call."""
    runs = [(150, 1), (3, 1), (64, 1)]
    cache = Cache(12, 2, 64, [4, 4, 4])
    cache.store([(0, 256)] * 3, *random_rows(768, 2, 64, 9))
    queries = torch.randn(3, 8 * 64, device="cuda").to(torch.bfloat16)
    out, again = torch.empty_like(queries), torch.empty_like(queries)
    for splits in (4, 40):
        step = make_step(runs)
        step.decode_splits = splits
        arguments = (cache.rows, 8, 2, 64, 0.125, 0)
        kernels.attention8(queries, *cache.pages, out, step, *arguments)
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            kernels.attention8(queries, *cache.pages, out, step, *arguments)
        step.seq_len.copy_(ints([200, 64, 1]))
        step.seq_start.copy_(ints([199, 63, 0]))
        other = torch.cuda.Stream()
        other.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(other):
            graph.replay()
        kernels.attention8(queries, *cache.pages, again, step, *arguments)
        torch.cuda.synchronize()
        assert torch.equal(out, again)


def most_asked_for(call) -> int:
    """The most bytes that `call` holds at once: as they are asked for (the allocator may hand out up to a mebibyte more, if it has a block that is just too large)."""
    torch.cuda.synchronize()
    torch.cuda.reset_peak_memory_stats()
    before = torch.cuda.memory_stats()["requested_bytes.all.current"]
    call()
    return torch.cuda.memory_stats()["requested_bytes.all.peak"] - before


@pytest.fixture
def plain_kernels():
    kernels.prefer_optimized(False)
    yield
    kernels.prefer_optimized(True)


@pytest.mark.parametrize("heads, kv_heads, dim, window", [(1, 1, 16, 0), (6, 2, 80, 90), (8, 2, 64, 1), (20, 1, 128, 0), (4, 2, 256, 70)])
def test_the_plain_kernel(plain_kernels, heads, kv_heads, dim, window):
    """Single tokens and runs against the statement, and bit for bit what the plain kernel of a 16-bit cache makes of the pages read back."""
    check_attention([(length - 1, 1) for length in (1, 64, 65, 300)], heads, kv_heads, dim, window)
    check_attention([(0, 70), (100, 1), (60, 9), (0, 1)], heads, kv_heads, dim, window)
    cache, runs = Cache(9, kv_heads, dim, [3, 2, 4]), [(120, 40), (0, 70), (199, 1)]
    cache.store([(0, 160), (0, 70), (0, 200)], *random_rows(430, kv_heads, dim, 5))
    queries = torch.randn(111, heads * dim, device="cuda").to(torch.bfloat16)
    found, wanted = torch.empty_like(queries), torch.empty_like(queries)
    step = make_step(runs)
    kernels.attention8(queries, *cache.pages, found, step, cache.rows, heads, kv_heads, dim, dim ** -0.5, window)
    keys, values = kernels.cache8_read(*cache.pages, step, cache.rows)
    places = torch.arange(12, dtype=torch.int32, device="cuda").view(3, 4)
    kernels.attention_generic(queries, keys, values, wanted, step.positions, step.token_seq, places, heads, kv_heads, dim, dim ** -0.5, window)
    assert torch.equal(found, wanted)


def test_the_plain_kernel_needs_no_workspace(plain_kernels):
    """A captured step lists as many pages as a sequence may ever have: memory goes by none of them (laid out in 16 bits these would take 671 MB)."""
    cache = Cache(40, 2, 64, [1] * 40)
    cache.store([(0, 30)] * 40, *random_rows(1200, 2, 64, 5))
    rows = torch.zeros(40, 512, dtype=torch.int32, device="cuda")
    rows[:, :1] = cache.rows
    queries = torch.randn(40, 8 * 64, device="cuda").to(torch.bfloat16)
    out, wanted = torch.empty_like(queries), torch.empty_like(queries)
    step = make_step([(29, 1)] * 40)
    kernels.attention8(queries, *cache.pages, wanted, step, cache.rows, 8, 2, 64, 0.125, 0)
    assert most_asked_for(lambda: kernels.attention8(queries, *cache.pages, out, step, rows, 8, 2, 64, 0.125, 0)) < 1 << 20
    assert torch.equal(out, wanted)


@pytest.mark.parametrize("dim", [32, 128])
def test_runs_behind_a_window_lay_out_the_pages_that_they_see(monkeypatch, dim):
    """A window of 100 and runs of up to 60 tokens see four pages wherever they begin, of the 63 that the longest sequence has: the workspace goes by the four."""
    monkeypatch.setattr(kernels, "runs8_like_single_tokens", lambda *sizes: False)
    for window in (1, 63, 64, 65, 100):
        check_attention([(3950, 60), (0, 2), (129, 60), (64, 3), (3903, 60), (99, 1)], 4, 2, dim, window)
    cache, runs = Cache(63, 2, dim, [63]), [(3950, 60)]
    cache.store([(0, 4010)], *random_rows(4010, 2, dim, 5))
    queries = torch.randn(60, 4 * dim, device="cuda").to(torch.bfloat16)
    out, step = torch.empty_like(queries), make_step(runs)
    arguments = (queries, *cache.pages, out, step, cache.rows, 4, 2, dim, dim ** -0.5, 100)
    kernels.attention8(*arguments)
    assert most_asked_for(lambda: kernels.attention8(*arguments)) <= 2 * 4 * 2 * 64 * dim * 2 + 4096      # and the table of their places


@pytest.mark.parametrize("heads, kv_heads, dim, at_once", [(6, 3, 48, 2), (8, 4, 64, 3), (3, 3, 128, 1), (8, 2, 256, 1)])
def test_runs_whose_pages_are_read_back_a_few_heads_at_a_time(monkeypatch, heads, kv_heads, dim, at_once):
    """Less room than one sequence takes: heads are read a few at a time, results are the same bit for bit, and memory stays within the room."""
    monkeypatch.setattr(kernels, "runs8_like_single_tokens", lambda *sizes: False)
    cache, runs = Cache(40, kv_heads, dim, [33, 5]), [(2000, 90), (255, 65)]
    cache.store([(0, 2090), (0, 320)], *random_rows(2410, kv_heads, dim, 5))
    queries = torch.randn(155, heads * dim, device="cuda").to(torch.bfloat16)
    out, wanted, step = torch.full_like(queries, 7.0), torch.full_like(queries, 7.0), make_step(runs)
    for window in (0, 100):
        kernels.attention8(queries, *cache.pages, wanted, step, cache.rows, heads, kv_heads, dim, dim ** -0.5, window)
        span = 33 if window == 0 else 4      # 189 positions, wherever they begin
        room = at_once * span * 4 * 64 * dim
        with monkeypatch.context() as patch:
            patch.setattr(kernels, "READ8_BYTES", room)
            most = most_asked_for(lambda: kernels.attention8(queries, *cache.pages, out, step, cache.rows, heads, kv_heads, dim, dim ** -0.5, window))
            assert most <= room + 2 * queries.numel() * 2 + 4096      # queries and results of those heads, and the table of the pages' places
        assert torch.equal(out, wanted)


@pytest.mark.parametrize("directly", [0, 1])
@pytest.mark.parametrize("longest", [600, 9000])
def test_rows_behind_the_last_run_stay_as_they_were(monkeypatch, directly, longest):
    """More rows than the runs have tokens: keys, values, queries and results behind the last run are neither read nor written, by a few ranges of a sequence or by many."""
    monkeypatch.setattr(kernels, "runs8_like_single_tokens", lambda *sizes: bool(directly))
    runs, counts = [(longest - 3, 3), (40, 2)], [-(-longest // 64), 1]
    cache, padded = Cache(sum(counts), 2, 64, counts), Cache(sum(counts), 2, 64, counts)
    keys, values = random_rows(longest + 42, 2, 64, 3)
    queries = torch.randn(9, 4 * 64, device="cuda").to(torch.bfloat16)
    new = torch.cat([torch.arange(longest - 3, longest), torch.arange(longest + 40, longest + 42)])
    results = []
    for each, rows in ((cache, 5), (padded, 9)):
        kernels.cache8_store(torch.cat([keys[: longest - 3], keys[longest : longest + 40]]).cuda(), torch.cat([values[: longest - 3], values[longest : longest + 40]]).cuda(), *each.pages,
                             make_step([(0, longest - 3), (0, 40)]), each.rows)
        step = make_step(runs)
        step.n_tokens = rows
        more = [torch.cat([each_[new], torch.full((rows - 5, 2, 64), float("nan"), dtype=torch.bfloat16)]).cuda() for each_ in (keys, values)]
        kernels.cache8_store(*more, *each.pages, step, each.rows)
        out = torch.full((rows, 4 * 64), 7.0, device="cuda", dtype=torch.bfloat16)
        kernels.attention8(queries[:rows], *each.pages, out, step, each.rows, 4, 2, 64, 0.125, 0)
        results.append(out)
    assert directly == 0 or (kernels.decode8_splits(2, longest, 2) > 8) == (longest == 9000)
    assert torch.equal(results[1][:5], results[0]) and bool((results[1][5:] == 7.0).all())
    for found, wanted in zip(padded.pages, cache.pages):
        assert torch.equal(found.view(torch.uint8), wanted.view(torch.uint8))
