"""Batches over a paged cache for the attention tests, and the operators in 64 bits
on the CPU, sequence by sequence."""
import math

import torch

EPS = 1e-6
HALF_STEP = {torch.bfloat16: 2.0 ** -8, torch.float16: 2.0 ** -11}


def frequencies(pairs, base=1e7):
    return (base ** (-torch.arange(pairs, dtype=torch.float64) / pairs)).float()


def batch(lens, page, seed=0, spare=3, columns=0):
    """lens: (new, length) of each sequence.  Returns starts, lengths, table (int32; pages in
    random order, entries past a sequence's pages out of range) and the page count."""
    g = torch.Generator().manual_seed(seed)
    need = [-(-length // page) for _, length in lens]
    pages = sum(need) + spare
    order = torch.randperm(pages, generator=g).tolist()
    columns = max(columns, max(need, default=1), 1)
    table = torch.full((len(lens), columns), -7, dtype=torch.int32)
    for s, n in enumerate(need):
        table[s, :n] = torch.tensor([order.pop() for _ in range(n)], dtype=torch.int32)
    starts = torch.tensor([0] + [n for n, _ in lens]).cumsum(0).to(torch.int32)
    return starts, torch.tensor([n for _, n in lens], dtype=torch.int32), table, pages


def norm_rope(x, weight, positions, inv_freq, eps=EPS):
    """(result, bound on its fp32 error before the last rounding) in 64 bits."""
    z = x.double()
    if weight is not None:
        z = z / torch.sqrt(z.square().mean(-1, keepdim=True) + eps) * (1 + weight.double())
    # fp32: the sum of squares (each of D / 8 * 8 additions and products half a step, all of one
    # sign), root, quotient and two products; then two products, a sum and sine and cosine (4 ulp)
    slack = z.abs() * (2 * x.shape[-1] + 16) * 2.0 ** -24
    if inv_freq is not None:
        h = inv_freq.numel()
        a = positions.double()[:, None, None] * inv_freq.double()
        c, s = torch.cos(a), torch.sin(a)
        lo, hi = z[..., :h].clone(), z[..., h:2 * h].clone()
        size = lo.abs() + hi.abs()
        z = torch.cat([lo * c - hi * s, hi * c + lo * s, z[..., 2 * h:]], -1)
        turned = size * (2 * x.shape[-1] + 32) * 2.0 ** -24
        slack = torch.cat([turned, turned, slack[..., 2 * h:]], -1)
    return z, slack


def assert_rows(got, want, slack, dtype, what):
    """got within one rounding of a value within slack of want."""
    got = got.double().cpu()
    tol = HALF_STEP[dtype] * (want.abs() + slack) + slack + (6e-8 if dtype == torch.float16 else 0)
    bad = ~((got - want).abs() <= tol)
    assert not bad.any(), (f'{what}: {int(bad.sum())} of {bad.numel()} values, first at '
                           f'{bad.nonzero()[0].tolist()}, error / tolerance '
                           f'{float(((got - want).abs() / tol).nan_to_num(9e9).max()):.3g}')


def gather(pages, row, length, page, h):
    used = row[:-(-length // page)].long() if length else row[:0].long()
    return pages[used, h].reshape(-1, pages.shape[-1])[:length]


def attention(q, k_pages, v_pages, starts, lengths, table, scale=None, gate=None):
    """(result, tolerance) of the rows of sequences, NaN elsewhere, in 64 bits on the CPU."""
    dim, page, hk = q.shape[-1], k_pages.shape[2], k_pages.shape[1]
    g, u = q.shape[1] // hk, HALF_STEP[q.dtype]
    scale = dim ** -0.5 if scale is None else scale
    out = torch.full(q.shape, math.nan, dtype=torch.float64)
    tol = torch.zeros(q.shape, dtype=torch.float64)
    for s in range(lengths.numel()):
        a, b, n = int(starts[s]), int(starts[s + 1]), int(lengths[s])
        for h in range(hk):
            k = gather(k_pages, table[s], n, page, h).double()
            v = gather(v_pages, table[s], n, page, h).double()
            for t in range(a, b):
                seen = max(min(n - (b - a) + (t - a) + 1, n), 0)
                rows = q[t, h * g:(h + 1) * g].double()
                if seen == 0:
                    out[t, h * g:(h + 1) * g] = 0
                    continue
                x = rows @ k[:seen].t() * scale
                w = torch.softmax(x, -1)
                o, size = w @ v[:seen], w @ v[:seen].abs()
                # scores: D products and sums, the scale, the running maximum's subtraction and
                # exp2 of a rounded argument; two of them in a weight (its own and the sum's)
                err = (rows.abs() @ k[:seen].abs().t()).amax(-1, keepdim=True) * abs(scale)
                err = 2 * ((dim + 8) * err + 2 * x.abs().amax(-1, keepdim=True) + 8) * 2.0 ** -24
                # weights are rounded to the type; sums of weights and products in fp32
                lost = size * (u + err + (seen + 64) * 2.0 ** -24)
                if q.dtype == torch.float16:  # weights below the smallest normal, of a sum >= 1
                    lost = lost + 2.0 ** -25 * v[:seen].abs().sum(0)
                out[t, h * g:(h + 1) * g], tol[t, h * g:(h + 1) * g] = o, lost
    if gate is not None:
        # the exponent -x log2(e) is off by half a step of its size, |x| 2^-24 of e^-x; exp2, the
        # sum, the reciprocal (a step each) and the product add 4 steps of 2^-24 (of 1 ulp: 2^-23)
        s, x = torch.sigmoid(gate.double()), gate.double().abs()
        out, tol = out * s, tol * s + out.nan_to_num().abs() * s * (2 * x + 8) * 2.0 ** -24
    return out, tol


def assert_attention(got, want, what, before=None):
    """got against attention()'s (result, tolerance); rows of no sequence hold `before`."""
    ref, slack = want
    got = got.cpu()
    none = ref[:, 0, 0].isnan() & ref.isnan().flatten(1).all(1)
    if before is not None:
        assert torch.equal(got[none], before.cpu()[none]), f'{what}: rows of no sequence'
    assert_rows(got[~none], ref[~none], slack[~none], got.dtype, what)
