"""Attention over the 4-bit cache at the ends of what it can be given: bytes of
scales that no row is written with, scales of scores and queries whose product
leaves 32 bits, weights that fp16 holds without all of its bits."""
import math

import pytest
import torch

from gpu_util import gen, normal
from kv4_util import numbers

pytestmark = pytest.mark.gpu

HALF = {torch.float16: 2.0 ** -11, torch.bfloat16: 2.0 ** -8}  # half a step of the type, relative


def ints(dev, *v):
    return torch.tensor(v, dtype=torch.int32, device=dev)


def cache_of(pkg, dev, k, v, block=16):
    """A cache of rows k and v [tokens, heads, d], its table, and what it holds in 64 bits."""
    n, heads, d = k.shape
    blocks = -(-n // block)
    cache = pkg.KVCache4.empty(blocks, heads, d, block, device=dev)
    pkg.kv_append(cache, k.to(dev), v.to(dev), torch.arange(n, device=dev))
    return cache, torch.arange(blocks, dtype=torch.int32, device=dev).view(1, blocks), [numbers(cache, x)[:n] for x in "kv"]


@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
@pytest.mark.parametrize("rows, heads", [(3, 4), (130, 32)])  # a tile of 16 rows, tiles of 128
@pytest.mark.parametrize("byte", [226, 227, 240, 247, 248, 255])
@pytest.mark.parametrize("d", [64, 128])
def test_scales_past_the_largest_leave_rows_that_do_not_see_them(pkg, dev, d, byte, rows, heads, dtype):
    """A value of six of a scale past 10240 is no fp16 number: rows of the tile
    before it get what they get without it, to the bit."""
    kv_heads, n = 1, 241
    g = gen(byte)
    k, v = (torch.randn((n, kv_heads, d), generator=g).half() for _ in range(2))
    cache, table, _ = cache_of(pkg, dev, k, v)
    q = normal((rows + 1, heads, d), 50, 1.5, dtype=dtype).to(dev)
    cu = ints(dev, 0, rows + 1)
    want = pkg.kv_attention(q, cache, table, ints(dev, n), cu=cu)
    # the last token, which only the last row sees
    cache.v_scale[15, ..., 0] = byte
    for code in (7, 15):  # 6 and -6
        cache.v[15] = (cache.v[15] & 0xf0) | torch.where(torch.arange(8, device=dev) == 0, code, cache.v[15] & 15).to(torch.uint8)
        got = pkg.kv_attention(q, cache, table, ints(dev, n), cu=cu)
        assert torch.equal(got[:rows], want[:rows]), code
        if byte > 247:
            assert torch.isnan(got[rows]).all()
        if byte == 226:  # a number still: 61440
            ks, vs, qd = numbers(cache, "k")[:n, 0], numbers(cache, "v")[:n, 0], q[rows].cpu().double()
            w = ((qd @ ks.t()) * d ** -0.5).softmax(-1)
            ref = w @ vs
            # a weight is off by half an fp16 step, its score by 130 roundings of at most its terms' magnitudes;
            # the sum of the weights by as much; a weight below fp16's normal range by 2^-32 of the largest
            by = 2.0 ** -12 + 130 * 2.0 ** -24 * (qd.abs() @ ks.abs().t()).amax() * d ** -0.5 + 2.0 ** -20
            room = 2 * by * (w @ vs.abs()) + n * 2.0 ** -31 * vs.abs().amax() + 2.0 ** -25
            assert ((got[rows].cpu().double() - ref).abs() <= HALF[dtype] * ref.abs() + room * (1 + HALF[dtype])).all()


@pytest.mark.parametrize("d", [64, 128])
@pytest.mark.parametrize("rows", [1, 130])  # tiles of 16 rows and of 128
def test_scores_that_a_scale_makes_nothing(pkg, dev, rows, d):
    """bf16 queries of 2^-60 to 2^-126 under a scale of 2^-40 and less: every
    score is 0 beside a weight's bits, so a row is the mean of what it sees."""
    heads, n = 32, 381
    g = gen(91)
    k, v = (torch.randn((n, 1, d), generator=g).half() for _ in range(2))
    cache, table, (_, vs) = cache_of(pkg, dev, k, v)
    vs = vs[:, 0]
    for by, scale in ((-60, 2.0 ** -40), (-110, 2.0 ** -40), (-126, 2.0 ** -40), (-110, 2.0 ** -126), (-126, 1.0)):
        q = (torch.randn((rows, heads, d), generator=g).clamp(-4, 4).double() * 2.0 ** by).to(torch.bfloat16).to(dev)
        got = pkg.kv_attention(q, cache, table, ints(dev, n), cu=ints(dev, 0, rows), scale=scale).cpu().double()
        for i in {0, rows // 2, rows - 1}:
            seen = vs[:n - rows + i + 1]
            want = seen.mean(0)
            # weights are equal powers of two, sums of them exact, sums of values by 2^-24 of their magnitudes each
            room = HALF[torch.bfloat16] * want.abs() + len(seen) * 2.0 ** -24 * seen.abs().mean(0)
            assert ((got[i] - want).abs() <= room * (1 + 2.0 ** -8)).all(), (by, scale, i)


@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
@pytest.mark.parametrize("rows", [1, 130])  # tiles of 16 rows and of 128
def test_scores_past_32_bits(pkg, dev, rows, dtype):
    """Scores whose size is no 32-bit number: the key with the largest one is all
    that remains, keys of zeros share where every score is 0."""
    heads, n, d = 32, 381, 64
    g = gen(93)
    k, v = (torch.randn((n, 1, d), generator=g).half() for _ in range(2))
    cache, table, (ks, vs) = cache_of(pkg, dev, k, v)
    zeros, _, (_, vz) = cache_of(pkg, dev, torch.zeros_like(k), v)
    q = torch.randn((rows, heads, d), generator=g).to(dtype)
    for by, scale in ((0, 2.0 ** 100), (0, 2.0 ** 127), *(((100, 2.0 ** 60), (120, 2.0 ** 127)) if dtype == torch.bfloat16 else ())):
        qs = (q.double() * 2.0 ** by).to(dtype)
        got = pkg.kv_attention(qs.to(dev), cache, table, ints(dev, n), cu=ints(dev, 0, rows), scale=scale).cpu().double()
        none = pkg.kv_attention(qs.to(dev), zeros, table, ints(dev, n), cu=ints(dev, 0, rows), scale=scale).cpu().double()
        for i in {0, rows - 1}:
            seen = n - rows + i + 1
            s = q[i].double() @ ks[:seen, 0].t()
            two = s.topk(2).values
            # (the kernel's own scores are off by less than 2^-13: 64 roundings of sums below 2^7 in 2^-24)
            clear = two[:, 0] - two[:, 1] > 2.0 ** -12
            assert clear.sum() > heads // 2
            assert torch.equal(got[i, clear], vs[s.argmax(-1), 0][clear]), (by, scale, i)
            want = vz[:seen, 0].mean(0)
            room = HALF[dtype] * want.abs() + seen * 2.0 ** -24 * vz[:seen, 0].abs().mean(0)
            assert ((none[i] - want).abs() <= room * (1 + 2.0 ** -8)).all(), (by, scale, i)


@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
@pytest.mark.parametrize("d", [64, 128])
@pytest.mark.parametrize("rows, kv_heads", [(1, 1), (130, 1), (130, 16)])  # 16 rows; 128, keys shared out; 128, most tiles whole
def test_thousands_of_weights_below_fp16s_normal_range(pkg, dev, rows, kv_heads, d, dtype):
    """A key 21.5 or 22 bits above 32000 others, whose weights together are about
    one percent: they count in the sum as they do in the values."""
    heads, n = 32 * kv_heads, 32011
    k = torch.zeros((n, kv_heads, d), dtype=torch.float16)
    v = torch.full((n, kv_heads, d), 0.75, dtype=torch.float16)  # (held as it is: 6 * 2^-3)
    k[5], v[5] = 0.75, 0.0
    v[5, :, 1] = 0.75  # of every key: what comes out there is the weights' sum over itself
    cache, table, (ks, vs) = cache_of(pkg, dev, k, v, 64)
    assert torch.equal(ks, k.double()) and torch.equal(vs, v.double())
    q = torch.full((rows, heads, d), 0.5, dtype=dtype, device=dev)
    for bits in (21.5, 22.0):
        scale = bits * math.log(2) / (0.375 * d)
        got = pkg.kv_attention(q, cache, table, ints(dev, n), cu=ints(dev, 0, rows), scale=scale).cpu().double()
        rest = (n - rows + torch.arange(rows)[:, None].double()) * 2.0 ** -bits
        want = 0.75 * rest / (1 + rest)
        # a weight of 2^-22 is off by 2^-32 of the largest at most, 2^-10 of itself, by its score's 2^-24 of 2^5
        # less, and the sum of the weights (other than the largest, which is a power of two) by as much
        assert ((got[..., 0] - want).abs() <= (HALF[dtype] + 2.0 ** -9 + 2.0 ** -14) * want).all(), bits
        assert ((got[..., 1] - 0.75).abs() <= 0.75 * (HALF[dtype] + 2.0 ** -11)).all(), bits
