"""Attention over the 4-bit cache at the ends of what it can be given: bytes of
scales that no row is written with."""
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
