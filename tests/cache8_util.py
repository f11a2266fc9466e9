"""A paged cache of 8 bits for the tests: e4m3 rounding, the append and the values that a cache
holds, in 64 bits on the CPU."""
import math

import torch

E4M3, BLOCK = torch.float8_e4m3fn, 16
LEAST = {torch.bfloat16: -117, torch.float16: -15}  # exponent of the smallest scale
MOST = {torch.bfloat16: 1.875 * 2.0 ** 127, torch.float16: 61440.0}  # largest value held


def e4m3(z):
    """z (at most 448) to the nearest of four significant bits, multiples of 2^-9 below 2^-6, ties to
    even; NaN stays."""
    step = torch.exp2(torch.floor(torch.log2(z.abs().clamp(min=2.0 ** -6))) - 3)
    return torch.where(z.isnan(), z, torch.round(z / step) * step)


def exponent(amax, dtype):
    """The least e, from LEAST on, with amax <= 448 * 2^e."""
    m, e = math.frexp(amax)  # 448 = 0.875 * 2^9
    return max(e - 9 + (m > 0.875), LEAST[dtype]) if amax else LEAST[dtype]


def per_row(scales, page):
    """scales [pages, heads, 2, blocks] -> keys' and values' [pages, heads, page, 1]."""
    return [scales[:, :, side].repeat_interleave(BLOCK, -1)[..., None] for side in range(2)]


def held(k_pages, v_pages, scales, dtype=torch.float64):
    """The keys and values of a cache, on the CPU."""
    scales = per_row(scales.cpu().double(), k_pages.shape[2])
    return [(x.cpu().double() * s).to(dtype) for x, s in zip((k_pages, v_pages), scales)]


def random_cache(gen, pages, heads, page, dim, dtype, spread=3.0):
    """Pages and scales of random values, each block of a magnitude of its own (2^-spread .. 2^spread)."""
    blocks = page // BLOCK
    kv = [torch.randn(pages, heads, page, dim, generator=gen) for _ in range(2)]
    scales = torch.exp2(torch.randint(-int(spread) - 6, int(spread) - 5, (pages, heads, 2, blocks),
                                      generator=gen).float())
    kv = [(x * 64).clamp(-448, 448).to(E4M3) for x in kv]
    return kv[0], kv[1], scales


def append(values, scales, rows, base, table, page, dtype):
    """Appends rows [n, heads, dim] (64 bits) at positions base .. of one side: values [pages, heads,
    page, dim] and scales [pages, heads, blocks] in 64 bits, in place.  A block's old exponent counts
    unless the block begins with these rows; returns for each row and head its block's scale."""
    n, heads, _ = rows.shape
    used = torch.zeros(n, heads, dtype=torch.float64)
    rows = torch.where(rows.isfinite(), rows.clamp(-MOST[dtype], MOST[dtype]), math.nan)
    i = 0
    while i < n:
        p = base + i
        count = min(BLOCK - p % BLOCK, n - i)
        if p < 0:
            i += 1
            continue
        number, at, block = table[p // page], p % page, p % page // BLOCK
        for h in range(heads):
            x = rows[i:i + count, h]
            size = float(x.abs().nan_to_num(0.0).amax())
            e = exponent(size, dtype)
            if p % BLOCK:
                e = max(e, int(math.log2(scales[number, h, block])))
            scale, start = 2.0 ** e, at - p % BLOCK
            old = values[number, h, start:at]
            old.copy_(e4m3(old / scale) * scale)
            # rows behind keep their bits
            values[number, h, at + count:start + BLOCK] *= scale / float(scales[number, h, block])
            values[number, h, at:at + count] = e4m3(x / scale) * scale
            scales[number, h, block] = scale
            used[i:i + count, h] = scale
        i += count
    return used


def assert_keys(got, want, slack, scale, what):
    """Held values within one rounding to e4m3 (half a step: 2^-4 of the value, or 2^-10 of the scale
    below 2^-6 of it) of a value within slack of want."""
    tol = torch.maximum(2.0 ** -4 * (want.abs() + slack), 2.0 ** -10 * scale) + slack
    bad = ~((got - want).abs() <= tol)
    assert not bad.any(), (f'{what}: {int(bad.sum())} of {bad.numel()} values, first at '
                           f'{bad.nonzero()[0].tolist()}')
