"""Plain statements of what the 8-bit kernels compute, in 64-bit, with numpy-like torch operations on the CPU; shares nothing with the library.

A block's scale is the least power of two s >= 2^-120 with max |x| <= 448 s over its finite elements, a code is x / s rounded to e4m3 (a sign, four bits of exponent, three
of mantissa, steps of 2^-9 below 2^-6, ties to even, greatest number 448); what is not finite becomes NaN.
"""
import math

import torch

PAGE = 64
BLOCK = 128


def power_of(greatest: float) -> float:
    """The scale of a block whose greatest finite magnitude is `greatest`, by search from the formula."""
    exponent = -120
    if greatest > 0:
        exponent = max(-120, math.frexp(greatest)[1] - 10)
        while greatest > 448.0 * 2.0 ** exponent:
            exponent += 1
    return 2.0 ** exponent


def to_e4m3(values, scale: float):
    """The values (not the codes) that e4m3 with this scale holds for `values` (float64)."""
    scaled = values / scale
    step = torch.exp2(torch.floor(torch.log2(scaled.abs().clamp(min=2.0 ** -6))).clamp(min=-6) - 3)
    held = torch.round(scaled / step) * step * scale
    return torch.where(torch.isfinite(values), held, torch.full_like(values, float("nan")))


def greatest_of(values) -> float:
    finite = values[torch.isfinite(values)]
    return float(finite.abs().max()) if finite.numel() else 0.0


def held_blocks(weight):
    """(values held, scales) of a weight cut into blocks of 128 x 128."""
    weight = weight.double()
    rows, columns = weight.shape
    held, scales = torch.empty_like(weight), torch.empty(-(-rows // BLOCK), -(-columns // BLOCK), dtype=torch.float64)
    for i in range(scales.shape[0]):
        for j in range(scales.shape[1]):
            part = (slice(i * BLOCK, (i + 1) * BLOCK), slice(j * BLOCK, (j + 1) * BLOCK))
            scales[i, j] = power_of(greatest_of(weight[part]))
            held[part] = to_e4m3(weight[part], float(scales[i, j]))
    return held, scales


def held_rows(values):
    """(values held, scales [blocks, rows]) of activations with a scale for each row and 128 columns."""
    values = values.double()
    rows, columns = values.shape
    held, scales = torch.empty_like(values), torch.empty(-(-columns // BLOCK), rows, dtype=torch.float64)
    for i in range(rows):
        for j in range(scales.shape[0]):
            part = (i, slice(j * BLOCK, (j + 1) * BLOCK))
            scales[j, i] = power_of(greatest_of(values[part]))
            held[part] = to_e4m3(values[part], float(scales[j, i]))
    return held, scales


class Pages:
    """A cache of one layer, position by position: `held[page][head]` [64, dim] float64 and `scale[page][head]`, for keys or values."""

    def __init__(self, pages, heads, dim):
        self.held = torch.zeros(pages, heads, PAGE, dim, dtype=torch.float64)
        self.scale = torch.ones(pages, heads, dtype=torch.float64)

    def store(self, page: int, low: int, rows):
        """`rows` [count, heads, dim] enter positions low, low + 1, ... of `page` together."""
        rows = rows.double()
        for head in range(rows.shape[1]):
            scale = power_of(greatest_of(rows[:, head]))
            if low:
                scale = max(scale, float(self.scale[page, head]))
                self.held[page, head, :low] = to_e4m3(self.held[page, head, :low], scale)
            self.held[page, head, low : low + rows.shape[0]] = to_e4m3(rows[:, head], scale)
            self.scale[page, head] = scale

    def store_run(self, table, start: int, rows):
        done = 0
        while done < rows.shape[0]:
            position = start + done
            count = min(PAGE - position % PAGE, rows.shape[0] - done)
            self.store(int(table[position // PAGE]), position % PAGE, rows[done : done + count])
            done += count

    def sequence(self, table, length: int):
        """[heads, length, dim]"""
        pages = [self.held[int(table[j])] for j in range(-(-length // PAGE))]
        return torch.cat(pages, dim=1)[:, :length] if pages else self.held.new_zeros(self.held.shape[1], 0, self.held.shape[3])


def attention(queries, keys, values, start: int, scale: float, window: int):
    """queries [new, heads, dim] at positions start, start + 1, ...; keys and values [kv heads, length, dim].  Returns (results, sums of weight times |value|, greatest
    sums of |query| times |key| of each query and head): what a bound on rounding needs."""
    new, heads, dim = queries.shape
    group = heads // keys.shape[0]
    out, spread, reach = (torch.zeros(new, heads, dim, dtype=torch.float64) for _ in range(3))
    for token in range(new):
        position = start + token
        first = max(0, position + 1 - window) if window else 0
        for head in range(heads):
            k, v = keys[head // group, first : position + 1], values[head // group, first : position + 1]
            q = queries[token, head].double()
            weights = torch.softmax(k @ q * scale, 0)
            out[token, head], spread[token, head] = weights @ v, weights @ v.abs()
            reach[token, head] = (k.abs() @ q.abs()).max() * scale
    return out, spread, reach
