"""GPU tests of what a cache in 8 bits keeps: rows that an append finds held already, rows behind its
last and whole blocks that it does not write, on both sides of the cache, against 64-bit results."""
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
I32 = torch.int32


def ints(*v):
    return torch.tensor(v, dtype=I32)


def both_sides(kp, vp, scales, want, scale64, what):
    """The whole cache against values and scales in 64 bits."""
    for side, got in enumerate(C.held(kp, vp, scales)):
        assert torch.equal(scales[:, :, side].cpu().double(), scale64[side]), (what, side)
        assert torch.equal(got, want[side]), (what, side)


def plain_append(cache, want, scale64, k, v, base, table, page, dtype):
    """Appends keys without norm and rotation, which are held as values are, and the same in 64 bits."""
    kp, vp, scales = cache
    n = k.shape[0]
    A.append(kp, vp, *to(kp.device, k, v, ints(0, n), ints(base + n), ints(*table).view(1, -1)),
             scales=scales)
    for side, x in enumerate((k, v)):
        C.append(want[side], scale64[side], x.double(), base, table, page, dtype)
    both_sides(kp, vp, scales, want, scale64, (base, n))


@TYPES
@pytest.mark.parametrize('dim,heads,page', [(64, 1, 16), (64, 3, 64), (128, 2, 32), (256, 5, 16)])
def test_append_leaves_what_is_held(dev, dim, heads, page, dtype):
    """Tokens of growing and falling sizes, alone and in parts of blocks: the bits of both sides."""
    gen = seeded(dim + page)
    kp, vp, scales = to(dev, *C.random_cache(gen, 8, heads, page, dim, dtype))
    want, scale64 = C.held(kp, vp, scales), [scales[:, :, s].cpu().double() for s in range(2)]
    table = [6, 1, 4, 0, 7]
    length = 0
    for i, n in enumerate([1, 1, 1, 2, 1, 3, 5, 1, 1, 6, 20, 1, 1, 7, 1, 19, 1, 8]):
        if length + n > 5 * page:
            break
        sizes = torch.exp2(torch.randint(-7, 8, (2, n, heads, 1), generator=gen).float())
        k, v = ((torch.randn(n, heads, dim, generator=gen) * s).to(dtype) for s in sizes)
        plain_append((kp, vp, scales), want, scale64, k, v, length, table, page, dtype)
        length += n


@pytest.mark.parametrize('dim,heads', [(64, 20), (128, 9), (256, 12)])
def test_append_of_many_blocks_and_heads(dev, dim, heads):
    """Workgroups that take several sides of a block, one after another: a chunk that goes on inside a
    block of other sizes, and one behind it."""
    gen, page = seeded(dim + heads), 64
    kp, vp, scales = to(dev, *C.random_cache(gen, 28, heads, page, dim, BF16))
    want, scale64 = C.held(kp, vp, scales), [scales[:, :, s].cpu().double() for s in range(2)]
    table, length = torch.randperm(28, generator=gen)[:26].tolist(), 0
    for n in (5, 1500, 90):
        sizes = torch.exp2(torch.randint(-7, 8, (2, n, heads, 1), generator=gen).float())
        k, v = ((torch.randn(n, heads, dim, generator=gen) * s).to(BF16) for s in sizes)
        plain_append((kp, vp, scales), want, scale64, k, v, length, table, page, BF16)
        length += n


@TYPES
@pytest.mark.parametrize('dim,page', [(64, 16), (128, 64), (256, 32)])
def test_append_leaves_what_is_held_beside_normed_keys(dev, dim, page, dtype):
    """Keys with norm and rotation, of which some rows have strong channels, so that scales grow: rows
    held are those of the kernel's own scales, and the scales the oracle's, or twice or half of them
    where the largest value is at a border."""
    gen, heads = seeded(dim), 3
    kp, vp, scales = to(dev, *C.random_cache(gen, 6, heads, page, dim, dtype))
    kw, freq = torch.randn(dim, generator=gen) * 0.2, U.frequencies(dim // 4)
    table, length, grown = [5, 2, 0, 3], 0, 0
    for n in [1] * 20 + [3, 4, 9, 1, 1]:
        k, v = rand(gen, n, heads, dim, dtype=dtype), rand(gen, n, heads, dim, dtype=dtype)
        k[..., dim - 1] *= torch.exp2(torch.randint(-1, 8, (n, heads), generator=gen).float())
        before, old = C.held(kp, vp, scales)[0], scales[:, :, 0].cpu().double()
        bits = kp.cpu().view(torch.uint8)
        A.append(kp, vp, *to(dev, k, v, ints(0, n), ints(length + n), ints(*table).view(1, -1)),
                 inv_freq=freq.to(dev), k_weight=kw.to(dev), scales=scales)
        now, new, after = C.held(kp, vp, scales)[0], scales[:, :, 0].cpu().double(), kp.cpu().view(torch.uint8)
        k64, _ = U.norm_rope(k, kw, torch.arange(length, length + n), freq)
        oracle, value64 = old.clone(), before.clone()
        C.append(value64, oracle, k64, length, table, page, dtype)
        ratio = new / oracle
        assert ((ratio == 1) | (ratio == 2) | (ratio == 0.5)).all()
        for number in range(6):
            first = table.index(number) * page if number in table else None
            for at in range(page):
                p = None if first is None else first + at
                if p is not None and length <= p < length + n:
                    continue  # a new row
                b = at // C.BLOCK
                if p is None or p >= length or not torch.equal(new[number, :, b], old[number, :, b]):
                    if p is not None and p < length:  # held, in a block whose scale grew
                        grown += 1
                        scale = new[number, :, b][:, None]
                        rounded = C.e4m3(before[number, :, at] / scale) * scale
                        assert torch.equal(now[number, :, at], rounded), (length, number, at)
                        continue
                assert torch.equal(after[number, :, at], bits[number, :, at]), (length, number, at)
        length += n
    assert grown > 0


@TYPES
@pytest.mark.parametrize('dim', [64, 128, 256])
def test_append_into_blocks_of_small_scales(dev, dim, dtype):
    """Scales below the least that an append makes, as another program may have written them: rows held
    under them stay the values that attention reads, rounded under the new scale."""
    gen, heads, page = seeded(dim + 7), 2, 32
    exps = [-118, -121, -126] if dtype == BF16 else [-16, -20, -27]
    for size in (0.0, 1e-6, 1.0):  # new rows that need the least scale, or more
        kp, vp, scales = to(dev, *C.random_cache(gen, 4, heads, page, dim, dtype))
        for number, e in zip((2, 0, 3), exps):
            scales[number] = 2.0 ** e
        want, scale64 = C.held(kp, vp, scales), [scales[:, :, s].cpu().double() for s in range(2)]
        table = [2, 0, 3]
        for base, n in ((5, 1), (6, 3), (page + 15, 2), (2 * page + 20, 4)):
            k, v = ((torch.randn(n, heads, dim, generator=gen) * size).to(dtype) for _ in range(2))
            plain_append((kp, vp, scales), want, scale64, k, v, base, table, page, dtype)


def test_attention_before_and_after_an_append_to_a_small_scale(dev):
    """What a row sees of the keys held before is the same before and after the append that lifts their
    block's scale: fp16 values that 2^-15 still holds exactly."""
    gen, page, dim = seeded(4), 16, 64
    kp, vp, scales = to(dev, *C.random_cache(gen, 2, 1, page, dim, FP16))
    vp[0] = (torch.randint(1, 15, (1, page, dim), generator=gen) * 32.0).to(dev).to(C.E4M3)  # 2^-15 of steps of 1
    scales[0] = 2.0 ** -20
    q = torch.zeros(1, 2, dim, dtype=FP16, device=dev)  # equal weights
    batch = to(dev, ints(0, 1), ints(4), ints(0).view(1, 1))
    a = A.paged_attention(q, kp, vp, *batch, scales=scales)
    zero = torch.zeros(1, 1, dim, dtype=FP16, device=dev)
    A.append(kp, vp, zero, zero, *to(dev, ints(0, 1), ints(5), ints(0).view(1, 1)), scales=scales)
    assert scales[0].cpu().eq(2.0 ** -15).all()
    assert torch.equal(A.paged_attention(q, kp, vp, *batch, scales=scales), a) and a.any()
