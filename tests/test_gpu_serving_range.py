"""Attention over the 8-bit cache at the ends of its range: pages whose value
scales lie far apart or are zero, scores of any size, against the definition in
64 bits."""
import pytest
import torch

from gpu_util import gen, normal
from test_gpu_serving import check_attention, ints

pytestmark = pytest.mark.gpu


def codes(shape, seed, std=36):
    return (torch.randn(shape, generator=gen(seed)) * std).round().clamp(-127, 127)


def cache_of(pkg, dev, kc, vc, ks, vs, block):
    """A cache of the given codes [blocks * block, heads, d] and scales [blocks,
    heads] (numbers of 11 significant bits), and its values in 64 bits."""
    blocks, heads = ks.shape
    d = kc.shape[-1]
    cache = pkg.KVCache.empty(blocks, heads, d, block, device=dev)
    cache.k[..., :d] = kc.view(blocks, block, heads, d).transpose(1, 2).to(torch.int8).to(dev)
    cache.v[..., :d, :] = vc.view(blocks, block // 16, 16, heads, d).permute(0, 3, 1, 4, 2).to(torch.int8).to(dev)
    cache.k_scale.copy_(ks)
    cache.v_scale.copy_(vs)
    assert torch.equal(cache.v_scale.cpu().double(), vs.double())  # (held exactly)
    return cache, [c.double() * s.double().repeat_interleave(block, 0)[..., None] for c, s in ((kc, ks), (vc, vs))]


# Rows of a request and heads of its key head: tiles of 16 rows, alone (keys
# shared out) and a few together, and of 128.
ROWS = [(1, 16), (3, 7), (450, 10)]


@pytest.mark.parametrize("rows, heads", ROWS)
@pytest.mark.parametrize("d, block", [(64, 16), (128, 32), (40, 64)])
@pytest.mark.parametrize("powers", [
    [None, 26], [26, None], [None, 30, 60], [110, None, 0], [None, 110, None, 80], [-60, 66], [66, -60, None], [-90, 90, -90],
    [None, None, None], [-95, None, -95], [0, 31, 0, -31, None, 0], [None] * 5 + [100] + [0] * 6,
])
def test_attention_over_value_scales_far_apart(pkg, dev, rows, heads, d, block, powers):
    """Pages of values around 2^power (None: zeros) under scores of a few units:
    every key has its part of the sum of weights, whatever its page's scale."""
    blocks = 3 * len(powers) if rows < 400 else max(3, 512 // block // len(powers) + 1) * len(powers)
    n = blocks * block
    vs = torch.tensor([0.0 if p is None else 2.0 ** (p - 6) for p in powers]).repeat(blocks // len(powers))[:, None]
    kc, vc = codes((n, 1, d), 1), codes((n, 1, d), 2)
    cache, (k, v) = cache_of(pkg, dev, kc, vc, torch.full((blocks, 1), 2.0 ** -6), vs, block)
    table = torch.arange(blocks, dtype=torch.int32, device=dev).view(1, blocks)
    q = normal((rows, heads, d), 3, 1.5, dtype=torch.bfloat16).to(dev)
    lens, cu = ints(dev, n - 3), [0, rows]
    got = pkg.kv_attention(q, cache, table, lens, cu=ints(dev, *cu))
    if rows > 400:  # (the first and last rows of the tiles, for the definition's time)
        at = torch.tensor(sorted({0, 1, 12, 13, 200, rows - 2, rows - 1}))
        for i in at.tolist():
            check_attention(got[i:i + 1], q[i:i + 1], k, v, block, table, ints(dev, n - 3 - rows + i + 1), [0, 1], d ** -0.5,
                            blocks, (powers, i))
    else:
        check_attention(got, q, k, v, block, table, lens, cu, d ** -0.5, blocks, powers)


@pytest.mark.parametrize("rows, heads", ROWS)
@pytest.mark.parametrize("d, block", [(64, 16), (128, 32)])
@pytest.mark.parametrize("power, dtype", [(14, torch.float16), (19, torch.float16), (23, torch.float16), (27, torch.float16),
                                          (33, torch.float16), (37, torch.float16), (30, torch.bfloat16), (90, torch.bfloat16)])
@pytest.mark.parametrize("sign", [1, -1])
def test_attention_of_large_scores(pkg, dev, rows, heads, d, block, power, dtype, sign):
    """Scores that are whole multiples of 2^power: the keys of a row's largest
    one share it, on pages of unlike value scales, and no weight overflows."""
    blocks = max(5, 600 // block)
    n = blocks * block
    kc, vc = torch.zeros((n, 1, d)), codes((n, 1, d), 12)
    kc[..., 0] = torch.randint(-9, 10, (n, 1), generator=gen(11)).float()
    vs = torch.exp2(torch.arange(blocks) % 4 - 6.0)[:, None]
    cache, (k, v) = cache_of(pkg, dev, kc, vc, torch.ones((blocks, 1)), vs, block)
    table = torch.randperm(blocks, generator=gen(13)).to(torch.int32).view(1, blocks).to(dev)
    half = min(power // 2, 15)
    q = torch.zeros((rows, heads, d))
    q[..., 0] = sign * 2.0 ** half
    q[..., 1:] = normal((rows, heads, d - 1), 14, dtype=torch.float32)  # (meets zero codes)
    q, scale = q.to(dtype).to(dev), 2.0 ** (power - half)
    got = pkg.kv_attention(q, cache, table, ints(dev, n - 3), cu=ints(dev, 0, rows), scale=scale)
    for i in {0, rows // 2, rows - 1}:
        check_attention(got[i:i + 1], q[i:i + 1], k, v, block, table, ints(dev, n - 3 - rows + i + 1), [0, 1], scale, blocks,
                        (power, i))


def test_attention_of_rows_with_infinities(pkg, dev):
    """An infinity or a NaN in a row of q makes that row NaN and no other."""
    heads, d, block, blocks = 10, 128, 32, 16
    kc, vc = codes((blocks * block, 1, d), 15), codes((blocks * block, 1, d), 16)
    ones = torch.full((blocks, 1), 2.0 ** -6)
    cache, (k, v) = cache_of(pkg, dev, kc, vc, ones, ones, block)
    table = torch.arange(blocks, dtype=torch.int32, device=dev).view(1, blocks)
    for dtype in (torch.float16, torch.bfloat16):
        for rows in (3, 450):
            q = normal((rows, heads, d), 17, 1.5, dtype=dtype).to(dev)
            want = pkg.kv_attention(q, cache, table, ints(dev, 500), cu=ints(dev, 0, rows))
            q[0, 3, 5], q[1, 0, 127], q[rows - 1, 9, 0] = float("inf"), float("nan"), float("-inf")
            got = pkg.kv_attention(q, cache, table, ints(dev, 500), cu=ints(dev, 0, rows))
            bad = torch.zeros((rows, heads), dtype=torch.bool, device=dev)
            bad[0, 3] = bad[1, 0] = bad[rows - 1, 9] = True
            assert torch.isnan(got[bad]).all() and torch.isfinite(got[~bad]).all(), (dtype, rows)
            off = (got[~bad].double() - want[~bad].double()).abs()
            assert (off <= 2.0 ** -7 * want[~bad].double().abs() + 2.0 ** -9).all(), (dtype, rows)
