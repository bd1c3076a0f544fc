"""Timed cases of the operators that serve a model with weights and cache in 8 bits (e4m3).

Product: activations in bfloat16 meet weights held as e4m3 codes with one 32-bit scale for each 128 x 128 block; within the call the
activations are quantised with a scale for each row and 128 columns.  Store: the keys and values of new tokens enter pages of 64
positions, a scale for each page and head, and the pages are read back as the values that they stand for, as a prompt's attention needs
them.  Attention: queries over such pages, one token a sequence or runs of them.

A block's scale is the least power of two `s >= 2^-120` with `max |x| <= 448 s` over its finite elements; a code is `x / s` rounded to e4m3; what is
not finite becomes NaN.  A page's scale grows when later tokens need it, and the codes that are there are rounded to the new one.

Sizes are those of the dense shapes of `bench.py` (1,024, 4,096 and 5,120 wide; 16, 32 and 64 query heads over 8 key/value heads) and
odd ones between them.  Weights and inputs are random.
"""
import math

import torch

own = False

PAGE = 64
BLOCK = 128


def listed():
    return [
        # One request alone on the small shape: q, k and v of the next token; launches and latency count.
        {"name": "product_1x1024x4096", "kind": "product", "rows": 1, "depth": 1024, "features": 4096, "gated": False, "bias": False, "out": "bfloat16"},
        # The benchmark's decode step of 8 requests: gate and up of the 4,096-wide shape, with the activation.
        {"name": "product_8x4096x24576_gated", "kind": "product", "rows": 8, "depth": 4096, "features": 24576, "gated": True, "bias": False, "out": "bfloat16"},
        # A busy server's decode step: the down product of 64 requests.
        {"name": "product_64x12288x4096", "kind": "product", "rows": 64, "depth": 12288, "features": 4096, "gated": False, "bias": False, "out": "bfloat16"},
        # Odd sizes: a last block of 80 columns, features that fill no tile, a bias, 32-bit results.
        {"name": "product_333x2000x1500_bias", "kind": "product", "rows": 333, "depth": 2000, "features": 1500, "gated": False, "bias": True, "out": "float32"},
        # The benchmark's prompt: 2,048 tokens through gate and up.
        {"name": "product_2048x4096x24576_gated", "kind": "product", "rows": 2048, "depth": 4096, "features": 24576, "gated": True, "bias": False, "out": "bfloat16"},
        # The next token of 64 requests enters the cache, most of them in the middle of a page.
        {"name": "store_64_tokens", "kind": "store", "sequences": 64, "longest": 200, "new": 1, "ragged": True, "heads": 8, "kv_heads": 8, "dim": 128, "window": 0},
        # The benchmark's prompt enters it beside another that continues.
        {"name": "store_prompts", "kind": "store", "sequences": 3, "longest": 2048, "new": 1500, "ragged": True, "heads": 8, "kv_heads": 8, "dim": 128, "window": 0},
        # One request's next token, a short chat.
        {"name": "decode_1x300", "kind": "attention", "sequences": 1, "longest": 300, "new": 1, "ragged": False, "heads": 16, "kv_heads": 8, "dim": 128, "window": 0},
        # The benchmark's decode step.
        {"name": "decode_8x2048", "kind": "attention", "sequences": 8, "longest": 2048, "new": 1, "ragged": False, "heads": 32, "kv_heads": 8, "dim": 128, "window": 0},
        # A busy server: 40 requests of unequal lengths, eight query heads to a key/value head.
        {"name": "decode_40_ragged_h64", "kind": "attention", "sequences": 40, "longest": 6000, "new": 1, "ragged": True, "heads": 64, "kv_heads": 8, "dim": 128, "window": 0},
        # Two long documents.
        {"name": "decode_2x120000", "kind": "attention", "sequences": 2, "longest": 120000, "new": 1, "ragged": False, "heads": 32, "kv_heads": 8, "dim": 128, "window": 0},
        # Portions of several prompts in one step, behind what is cached of them.
        {"name": "runs_ragged", "kind": "attention", "sequences": 4, "longest": 4500, "new": 600, "ragged": True, "heads": 32, "kv_heads": 8, "dim": 128, "window": 0},
    ]


def _between(rng, low, high, step=1):
    """A multiple of `step` between `low` and `high`, spread over the logarithm."""
    value = math.exp(rng.uniform(math.log(low), math.log(high)))
    return min(high, max(low, int(round(value / step)) * step))


def draw(rng):
    kind = rng.choice(["product", "product", "store", "attention", "attention", "attention"])
    if kind == "product":
        gated = rng.random() < 0.3
        rows, depth, features = _between(rng, 1, 2048), _between(rng, 256, 12288, 16), _between(rng, 256, 24576, 16 if gated else 4)
        rows = max(1, min(rows, 2048 * 4096 * 24576 // (depth * features)))
        return {"kind": "product", "rows": rows, "depth": depth, "features": features, "gated": gated, "bias": not gated and rng.random() < 0.4,
                "out": "bfloat16" if gated else rng.choice(["bfloat16", "float32"])}
    kv_heads = rng.choice([1, 2, 4, 8])
    heads = kv_heads * rng.choice([1, 2, 3, 4, 8, 16])
    dim = rng.choice([64, 80, 96, 128, 128, 128, 256])
    if kind == "store":
        new = 1 if rng.random() < 0.5 else _between(rng, 2, 1500)
        sequences = _between(rng, 1, 64 if new == 1 else 4)
        return {"kind": "store", "sequences": sequences, "longest": max(new, _between(rng, 1, 2048 if new > 1 else 200)), "new": new, "ragged": rng.random() < 0.7,
                "heads": kv_heads, "kv_heads": kv_heads, "dim": dim, "window": 0}
    if rng.random() < 0.65:
        sequences = _between(rng, 1, 64)
        longest = _between(rng, 1, min(120000, 240000 // sequences))
        return {"kind": "attention", "sequences": sequences, "longest": longest, "new": 1, "ragged": rng.random() < 0.6, "heads": heads, "kv_heads": kv_heads, "dim": dim,
                "window": rng.choice([0, 0, 0, _between(rng, 1, longest)])}
    sequences = _between(rng, 1, 4)
    new = _between(rng, 2, 600)
    longest = _between(rng, new, 4500)
    return {"kind": "attention", "sequences": sequences, "longest": longest, "new": new, "ragged": rng.random() < 0.6, "heads": min(heads, 32), "kv_heads": kv_heads, "dim": dim,
            "window": rng.choice([0, 0, _between(rng, 1, longest)])}


def _runs(case):
    """(positions cached before, new tokens) of each sequence; the first sequence is the longest and brings the most."""
    runs = []
    for index in range(case["sequences"]):
        share = 1.0 if index == 0 or not case["ragged"] else (index * 0.6180339887 + 0.11) % 1.0
        new = max(1, int(case["new"] * share))
        length = max(new, int(case["longest"] * share))
        runs.append((length - new, new))
    return runs


def _scale(greatest):
    """The block's scale, from the greatest magnitude of its finite elements (32- or 64-bit)."""
    mantissa, exponent = torch.frexp(greatest)      # greatest = mantissa * 2^exponent, mantissa in [0.5, 1)
    steps = torch.where(mantissa > 0.875, exponent - 8, exponent - 9)
    return torch.ldexp(torch.ones_like(greatest), torch.where(greatest > 0, steps, torch.full_like(steps, -120)).clamp(min=-120))


def _greatest(values, dims):
    return torch.where(torch.isfinite(values), values.abs(), torch.zeros_like(values)).amax(dims, keepdim=True)


def _codes(values, scale):
    return torch.where(torch.isfinite(values), values / scale, torch.full_like(values, float("nan"))).float().to(torch.float8_e4m3fn)


def _generator(seed):
    return torch.Generator(device="cuda").manual_seed(seed)


def _quantized_weight(weight):
    """Codes [features, depth] and scales [blocks of features, blocks of depth] of a weight, block by block of 128 x 128."""
    features, depth = weight.shape
    down, across = -(-features // BLOCK), -(-depth // BLOCK)
    padded = torch.zeros(down * BLOCK, across * BLOCK, device=weight.device)
    padded[:features, :depth] = weight
    blocks = padded.view(down, BLOCK, across, BLOCK)
    scale = _scale(_greatest(blocks, (1, 3)))
    codes = _codes(blocks, scale).view(torch.uint8).view(down * BLOCK, across * BLOCK)[:features, :depth].contiguous()
    return codes.view(torch.float8_e4m3fn), scale.view(down, across).contiguous()


def _step(runs, page_rows):
    """The step's metadata, as the engine's steps bring it."""
    from tau_rs_b200.engine.batch import StepContext

    def ints(values):
        return torch.tensor(values, dtype=torch.int32, device="cuda")

    bounds, positions, owners = [0], [], []
    for index, (start, new) in enumerate(runs):
        bounds.append(bounds[-1] + new)
        positions += range(start, start + new)
        owners += [index] * new
    return StepContext(
        n_tokens=bounds[-1], n_seqs=len(runs), n_wanted=0, token_ids=ints(positions), positions=ints(positions), token_seq=ints(owners), want_rows=ints([]),
        cu_seqlens=ints(bounds), seq_slot=ints(range(len(runs))), seq_start=ints([start for start, _ in runs]), seq_len=ints([start + new for start, new in runs]),
        page_rows={"attention": page_rows}, max_new=max(new for _, new in runs), max_len=max(start + new for start, new in runs),
        all_single=all(new == 1 for _, new in runs), min_new=min(new for _, new in runs), all_fresh=all(start == 0 for start, _ in runs))


def prepare(case, seed):
    random = _generator(seed)

    def normal(*shape):
        return torch.randn(*shape, device="cuda", generator=random)

    state = {"case": case, "own": own}
    if case["kind"] == "product":
        rows, depth, features = case["rows"], case["depth"], case["features"]
        # Behind a norm: channels of unequal size, some of them far above the others.
        channels = torch.exp(0.5 * normal(depth)) * torch.where(torch.rand(depth, device="cuda", generator=random) < 0.01, 8.0, 1.0)
        state["values"] = (normal(rows, depth) * channels).to(torch.bfloat16)
        state["codes"], state["scales"] = _quantized_weight(normal(features, depth) * 0.02)
        state["bias"] = normal(features) * 0.1 if case["bias"] else None
        return state
    runs, heads, kv_heads, dim = _runs(case), case["heads"], case["kv_heads"], case["dim"]
    counts = [-(-(start + new) // PAGE) for start, new in runs]
    stride, used = max(counts), sum(counts)
    order = torch.randperm(used, device="cuda", generator=random).tolist()
    table = torch.zeros(len(runs), stride, dtype=torch.int32)
    cursor = 0
    for index, count in enumerate(counts):
        table[index, :count] = torch.tensor(order[cursor : cursor + count], dtype=torch.int32)
        cursor += count
    state["runs"], state["counts"], state["page_rows"] = runs, counts, table.cuda()
    # Keys behind a norm over the head and a rotation, values as a projection leaves them, some heads several times larger than others.
    for name in ("key", "value"):
        sizes = torch.exp(0.5 * normal(1, kv_heads, 1, dim if name == "key" else 1))
        codes, scales = torch.empty(used, kv_heads, PAGE, dim, dtype=torch.uint8, device="cuda"), torch.empty(used, kv_heads, 1, 1, device="cuda")
        for first in range(0, used, 512):
            pages = (normal(min(512, used - first), kv_heads, PAGE, dim) * sizes).to(torch.bfloat16).float()
            scales[first : first + 512] = _scale(_greatest(pages, (2, 3)))
            codes[first : first + 512] = _codes(pages, scales[first : first + 512]).view(torch.uint8)
        state[name + "_pages"], state[name + "_scales"] = codes.view(torch.float8_e4m3fn), scales.view(used, kv_heads)
    tokens = sum(new for _, new in runs)
    if case["kind"] == "store":
        state["keys"], state["values"] = normal(tokens, kv_heads, dim).to(torch.bfloat16), (normal(tokens, kv_heads, dim) * torch.exp(normal(tokens, 1, 1))).to(torch.bfloat16)
        # What the pages hold behind the positions cached before belongs to nobody: zeros here, so that whole pages can be compared.
        for index, (start, _) in enumerate(runs):
            for page in range(start // PAGE, counts[index]):
                for name in ("key", "value"):
                    state[name + "_pages"][int(table[index, page]), :, max(0, start - page * PAGE) :] = 0
    else:
        state["queries"] = normal(tokens, heads * dim).to(torch.bfloat16)
    if own:
        state["step"] = _step(runs, state["page_rows"])
    return state


def run(state):
    case = state["case"]
    if state["own"]:
        return _run_own(case, state)
    if case["kind"] == "product":
        out = torch.bfloat16 if case["out"] == "bfloat16" else torch.float32
        return _product(state, torch.float32, True).to(out)
    if case["kind"] == "store":
        return _store(state, torch.float32)
    return _attention(state, torch.float32).to(torch.bfloat16)


def _run_own(case, state):
    from tau_rs_b200.csrc import kernels

    if case["kind"] == "product":
        values, features = state["values"], case["features"]
        out = torch.empty(values.shape[0], features // 2 if case["gated"] else features, dtype=torch.bfloat16 if case["out"] == "bfloat16" else torch.float32, device="cuda")
        if case["gated"]:
            kernels.linear8_gated(values, state["codes"], state["scales"], out)
        else:
            kernels.linear8(values, state["codes"], state["scales"], state["bias"], out)
        return out
    pages = (state["key_pages"], state["value_pages"], state["key_scales"], state["value_scales"])
    if case["kind"] == "store":
        kernels.cache8_store(state["keys"], state["values"], *pages, state["step"], state["page_rows"])
        keys, values = kernels.cache8_read(*pages, state["step"], state["page_rows"])
        return {"keys": keys, "values": values, "key_scales": state["key_scales"], "value_scales": state["value_scales"]}
    out = torch.empty_like(state["queries"])
    kernels.attention8(state["queries"], *pages, out, state["step"], state["page_rows"], case["heads"], case["kv_heads"], case["dim"], case["dim"] ** -0.5, case["window"])
    return out


def _product(state, dtype, round_pairs):
    """The product in its plain form: both operands as the values that their codes stand for."""
    case, values = state["case"], state["values"].to(dtype)
    rows, depth = values.shape
    across = -(-depth // BLOCK)
    padded = torch.zeros(rows, across * BLOCK, dtype=dtype, device=values.device)
    padded[:, :depth] = values
    blocks = padded.view(rows, across, BLOCK)
    scale = _scale(_greatest(blocks, (2,)))
    held = (_codes(blocks, scale).to(dtype) * scale).view(rows, across * BLOCK)[:, :depth]
    spread = state["scales"].to(dtype).repeat_interleave(BLOCK, 0).repeat_interleave(BLOCK, 1)[: case["features"], :depth]
    result = held @ (state["codes"].to(dtype) * spread).T
    if case["bias"]:
        result = result + state["bias"].to(dtype)
    if case["gated"]:      # groups of 8 gate rows and their 8 up rows; both are rounded as an ungated product would store them
        pairs = (result.to(torch.bfloat16).to(dtype) if round_pairs else result).view(rows, -1, 2, 8)
        gate, up = pairs[:, :, 0].reshape(rows, -1), pairs[:, :, 1].reshape(rows, -1)
        result = gate / (1 + torch.exp(-gate)) * up
    return result


def _store(state, dtype):
    """Page by page: the scale over what is new and the page's own (none for a page that starts here), older codes rounded to it."""
    runs, table, counts = state["runs"], state["page_rows"].tolist(), state["counts"]
    stride = len(table[0])
    result = {}
    for name, new in (("key", state["keys"].to(dtype)), ("value", state["values"].to(dtype))):
        codes, scales = state[name + "_pages"], state[name + "_scales"]
        cursor = 0
        for index, (start, count) in enumerate(runs):
            for page in range(start // PAGE, counts[index]):
                low, high = max(start, page * PAGE), min(start + count, (page + 1) * PAGE)
                number, before = table[index][page], low - page * PAGE
                rows = new[cursor + low - start : cursor + high - start].transpose(0, 1)
                wanted = _scale(_greatest(rows, (1, 2)))
                if before:
                    old = scales[number].to(dtype).view(-1, 1, 1)
                    wanted = torch.maximum(wanted, old)
                    codes[number, :, :before] = _codes(codes[number, :, :before].to(dtype) * old, wanted)
                codes[number, :, before : before + high - low] = _codes(rows, wanted)
                scales[number] = wanted.view(-1).float()
            cursor += count
        result[name + "s"], result[name + "_scales"] = _read(codes, scales, table, counts, stride, dtype), scales
    return result


def _read(codes, scales, table, counts, stride, dtype):
    """The pages of the sequences, one sequence behind the other, as the values that they stand for; zeros where a sequence has no page."""
    pages = torch.zeros(len(table) * stride, *codes.shape[1:], dtype=torch.bfloat16 if dtype == torch.float32 else dtype, device=codes.device)
    numbers = torch.tensor([table[index][page] for index, count in enumerate(counts) for page in range(count)], device=codes.device)
    places = torch.tensor([index * stride + page for index, count in enumerate(counts) for page in range(count)], device=codes.device)
    pages[places] = (codes[numbers].to(dtype) * scales[numbers].to(dtype)[:, :, None, None]).to(pages.dtype)
    return pages


def _attention(state, dtype):
    """Sequence by sequence: every key and value as the value it stands for, a whole matrix of scores, its softmax, the weighted sum."""
    case = state["case"]
    heads, kv_heads, dim, window = case["heads"], case["kv_heads"], case["dim"], case["window"]
    group = heads // kv_heads
    out = torch.empty(state["queries"].shape, dtype=dtype, device="cuda")
    cursor = 0
    for index, (start, new) in enumerate(state["runs"]):
        length, count = start + new, state["counts"][index]
        numbers = state["page_rows"][index, :count].long()
        # One token sees only its window; more of them see the window before the first.
        first = max(0, start + 1 - window) // PAGE if window else 0
        held = []
        for name in ("key", "value"):
            pages = state[name + "_pages"][numbers[first:]].to(dtype) * state[name + "_scales"][numbers[first:]].to(dtype)[:, :, None, None]
            held.append(pages.transpose(0, 1).reshape(kv_heads, -1, dim)[:, : length - first * PAGE])
        keys, values = held
        queries = state["queries"][cursor : cursor + new].to(dtype).view(new, kv_heads, group, dim).transpose(0, 1).reshape(kv_heads, new * group, dim)
        place = torch.arange(first * PAGE, length, device="cuda")
        own_place = torch.arange(start, length, device="cuda")
        hidden = place[None] > own_place[:, None]
        if window:
            hidden = hidden | (place[None] <= own_place[:, None] - window)
        scores = (queries @ keys.transpose(1, 2)).view(kv_heads, new, group, -1) * dim ** -0.5
        scores = scores.masked_fill(hidden[None, :, None], float("-inf"))
        weights = torch.exp(scores - scores.amax(-1, keepdim=True))
        result = (weights.view(kv_heads, new * group, -1) @ values).view(kv_heads, new, group, dim) / weights.sum(-1, keepdim=True)
        out[cursor : cursor + new] = result.transpose(0, 1).reshape(new, heads * dim)
        cursor += new
    return out


def _visible(case):
    """(query, key) pairs, and the cached positions that any query of each sequence sees."""
    pairs = seen = 0
    window = case["window"]
    for start, new in _runs(case):
        last = start + new
        seen += min(last, window + new - 1) if window else last
        pairs += sum(min(position + 1, window) if window else position + 1 for position in range(start, last))
    return pairs, seen


def work(case):
    if case["kind"] == "product":
        rows, depth, features = case["rows"], case["depth"], case["features"]
        scales = -(-depth // BLOCK) * -(-features // BLOCK)
        out = rows * (features // 2 if case["gated"] else features) * (2 if case["out"] == "bfloat16" else 4)
        return {"bytes": 2 * rows * depth + features * depth + 4 * scales + (4 * features if case["bias"] else 0) + out, "flops": 2 * rows * depth * features}
    runs, kv_heads, dim = _runs(case), case["kv_heads"], case["dim"]
    tokens = sum(new for _, new in runs)
    if case["kind"] == "store":      # new tokens in, codes out, then the sequences' pages read and laid out in 16 bits
        pages = sum(-(-(start + new) // PAGE) for start, new in runs)
        return {"bytes": 2 * tokens * kv_heads * dim * 3 + 2 * pages * kv_heads * (PAGE * dim * 3 + 4), "flops": 0}
    pairs, seen = _visible(case)
    return {"bytes": 2 * 2 * tokens * case["heads"] * dim + 2 * seen * kv_heads * dim + 8 * kv_heads * -(-seen // PAGE), "flops": 4 * pairs * case["heads"] * dim}


# ---- the same in 64 bits, from the definitions -------------------------------------------------------------------------------------
def _held64(values, dims):
    """Values as e4m3 with a power of two for each block of `dims` would hold them, without the type: 4 significant bits down to 2^-6, steps of 2^-9 below."""
    magnitude = values.abs()
    top = torch.where(torch.isfinite(magnitude), magnitude, torch.zeros_like(magnitude)).amax(dims, keepdim=True)
    return _round64(values, _power64(top)), _power64(top)


def _power64(top):
    exponent = torch.ceil(torch.log2(top.clamp(min=2.0 ** -300) / 448.0))
    exponent = torch.where(448.0 * torch.exp2(exponent - 1) >= top, exponent - 1, exponent)      # the logarithm may lie on the wrong side of a border
    exponent = torch.where(448.0 * torch.exp2(exponent) < top, exponent + 1, exponent)
    return torch.exp2(exponent.clamp(min=-120))


def _round64(values, power):
    scaled = values / power
    step = torch.exp2(torch.floor(torch.log2(scaled.abs().clamp(min=2.0 ** -6))).clamp(min=-6) - 3)
    return torch.where(torch.isfinite(values), torch.round(scaled / step) * step * power, torch.full_like(values, float("nan")))      # ties to even


def exact(case, seed):
    global own
    kept, own = own, False
    try:
        state = prepare(case, seed)
    finally:
        own = kept
    if case["kind"] == "product":
        values = state["values"].double()
        result = torch.zeros(case["rows"], case["features"], dtype=torch.float64, device="cuda")
        for block in range(-(-case["depth"] // BLOCK)):
            columns = slice(block * BLOCK, (block + 1) * BLOCK)
            held, _ = _held64(values[:, columns], (1,))
            part = held @ state["codes"][:, columns].double().T
            result += part * state["scales"][:, block].double().repeat_interleave(BLOCK)[: case["features"]]
        if case["bias"]:
            result += state["bias"].double()
        if case["gated"]:
            pairs = result.view(case["rows"], -1, 2, 8)
            gate, up = pairs[:, :, 0].reshape(case["rows"], -1), pairs[:, :, 1].reshape(case["rows"], -1)
            result = gate * torch.sigmoid(gate) * up
        return result
    if case["kind"] == "store":
        return _store64(state)
    return _attention64(state)


def _store64(state):
    table, stride = state["page_rows"].tolist(), state["page_rows"].shape[1]
    result = {}
    for name in ("key", "value"):
        held = state[name + "_pages"].double() * state[name + "_scales"].double()[:, :, None, None]
        scales = state[name + "_scales"].double().clone()
        new = state[name + "s"].double()
        first = 0
        for index, (start, count) in enumerate(state["runs"]):
            for position in range(start, start + count):      # grouped by page: the positions of one page at a time
                if position != start and position % PAGE:
                    continue
                number, low = table[index][position // PAGE], position % PAGE
                high = min(PAGE, low + start + count - position)
                rows = new[first + position - start : first + position - start + high - low].permute(1, 0, 2)
                power = _power64(rows.abs().amax((1, 2), keepdim=True))
                if low:
                    power = torch.maximum(power, scales[number][:, None, None])
                    held[number, :, :low] = _round64(held[number, :, :low], power)
                held[number, :, low:high] = _round64(rows, power)
                scales[number] = power[:, 0, 0]
            first += count
        pages = torch.zeros(len(table) * stride, *held.shape[1:], dtype=torch.float64, device="cuda")
        for index, count in enumerate(state["counts"]):
            pages[index * stride : index * stride + count] = held[state["page_rows"][index, :count].long()]
        result[name + "s"], result[name + "_scales"] = pages, scales
    return result


def _attention64(state):
    case = state["case"]
    heads, kv_heads, dim, window = case["heads"], case["kv_heads"], case["dim"], case["window"]
    rows = []
    first = 0
    for index, (start, new) in enumerate(state["runs"]):
        numbers = state["page_rows"][index, : state["counts"][index]].long()
        result = torch.empty(new, heads, dim, dtype=torch.float64, device="cuda")
        for head in range(heads):
            shared = head // (heads // kv_heads)
            keys = (state["key_pages"][numbers, shared].double() * state["key_scales"][numbers, shared].double()[:, None, None]).reshape(-1, dim)[: start + new]
            values = (state["value_pages"][numbers, shared].double() * state["value_scales"][numbers, shared].double()[:, None, None]).reshape(-1, dim)[: start + new]
            queries = state["queries"][first : first + new].view(new, heads, dim)[:, head].double()
            scores = queries @ keys.T / math.sqrt(dim)
            distance = torch.arange(start, start + new, device="cuda")[:, None] - torch.arange(start + new, device="cuda")[None]
            visible = (distance >= 0) & (distance < window) if window else distance >= 0
            result[:, head] = torch.softmax(torch.where(visible, scores, torch.full_like(scores, -math.inf)), -1) @ values
        rows.append(result.view(new, heads * dim))
        first += new
    return torch.cat(rows)
