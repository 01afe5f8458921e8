"""Attention over the 8-bit cache at the ends of its range: pages whose value
scales lie far apart or are zero, against the definition in 64 bits."""
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
