"""GPU tests of attention over a cache in 8 bits whose values or scales are beyond the rows' type: they
reach the rows that see them and no others."""
import pytest
import torch

from localmoe35ba3b_amd.operators import attention as A
from tests import attention_util as U
from tests import cache8_util as C
from tests.conftest import seeded
from tests.test_gpu_attention import rand, to

pytestmark = pytest.mark.gpu

BF16, FP16 = torch.bfloat16, torch.float16
TYPES = pytest.mark.parametrize('dtype', [BF16, FP16])


def block_of(table, position, page):
    return int(table[0, position // page]), position % page // C.BLOCK


@TYPES
@pytest.mark.parametrize('dim', [64, 128, 256])
@pytest.mark.parametrize('new', [1, 3, 40])
def test_attention_values_beyond_the_type_reach_the_rows_that_see_them(dev, new, dim, dtype):
    """Under the largest scale the code 0x78 is an infinity of the type: at a position inside the last
    block it shows in the rows from that position on, in its heads and channel, and nowhere else."""
    gen, length, bad = seeded(dim + new), 85, 83
    lens = [(new, length), (new, 70)]
    starts, lengths, table, pages = U.batch(lens, 16)
    q = rand(gen, 2 * new, 4, dim, dtype=dtype, scale=0.05)  # no weight below the type's least
    kp, vp, scales = C.random_cache(gen, pages, 2, 16, dim, dtype)
    at, b = block_of(table, bad, 16)
    scales[at, :, 1, b] = 2.0 ** (120 if dtype == BF16 else 8)
    vb = vp.view(torch.uint8)
    vb[at] = torch.randint(0, 2, vb[at].shape, generator=gen).to(torch.uint8)  # tiny
    want = U.attention(q, *C.held(kp, vp, scales, dtype), starts, lengths, table)
    vb[at, 0, bad % 16, 3], vb[at, 0, bad % 16, dim - 1] = 0x78, 0xF8
    got = A.paged_attention(*to(dev, q, kp, vp, starts, lengths, table), scales=scales.to(dev)).cpu()
    rows = slice(max(0, new - (length - bad)), new)
    assert rows.stop - rows.start == min(new, 2)
    assert (got[rows, :2, 3] == float('inf')).all() and (got[rows, :2, dim - 1] == float('-inf')).all()
    for c in (3, dim - 1):
        got[rows, :2, c] = want[0][rows, :2, c].to(dtype)
    U.assert_attention(got, want, 'the others')


@TYPES
@pytest.mark.parametrize('dim', [64, 128, 256])
@pytest.mark.parametrize('new', [1, 40])
def test_attention_scales_beyond_the_largest(dev, new, dim, dtype):
    """Of a scale the exponent counts, and one beyond the largest counts as that: in blocks that rows see,
    and behind the end, where neither it nor NaN shows."""
    gen, most = seeded(dim + 3), 120 if dtype == BF16 else 8
    starts, lengths, table, pages = U.batch([(new, 85)], 32)
    q = rand(gen, new, 4, dim, dtype=dtype)
    kp, vp, scales = C.random_cache(gen, pages, 2, 32, dim, dtype)
    at, b = block_of(table, 84, 32)  # positions 80 .. 84 of it are seen
    vb, kb = vp.view(torch.uint8), kp.view(torch.uint8)
    vb[at, :, 16:] = torch.randint(0, 2, vb[at, :, 16:].shape, generator=gen).to(torch.uint8)
    kb[at, :, 16:] = 0
    vb[at, :, 21:], kb[at, :, 21:] = 0x7F, 0xFF  # behind the end
    assert b == 1
    scales[at, :, 1, b] = 2.0 ** most
    values = C.held(kp, vp, scales, dtype)
    values[0][at, :, 21:], values[1][at, :, 21:] = 0, 0
    want = U.attention(q, *values, starts, lengths, table)
    inf, nan = float('inf'), float('nan')
    for v_scale in (2.0 ** most, 2.0 ** (most + 1), 1.5 * 2.0 ** most, -(2.0 ** (most + 3)), inf, nan):
        scales[at, :, 1, b], scales[at, :, 0, b] = v_scale, 1.0 if new > 1 else abs(v_scale)
        got = A.paged_attention(*to(dev, q, kp, vp, starts, lengths, table), scales=scales.to(dev))
        U.assert_attention(got, want, f'{v_scale}')
