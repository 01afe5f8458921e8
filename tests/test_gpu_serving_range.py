"""Attention over the 8-bit cache at the ends of its range: pages whose value
scales lie far apart or are zero, scores of any size, keys far above the others,
against the definition in 64 bits."""
import pytest
import torch

from gpu_util import gen, normal
from test_gpu_serving import HALF, check_attention, ints

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


def weights64(q, k, n, scale):
    return (q.double() @ k[:n, 0].T * scale).softmax(-1)


@pytest.mark.parametrize("tiles", [16, 128])
@pytest.mark.parametrize("spread", [0.0, 0.3])
@pytest.mark.parametrize("bits", [12, 18, 20, 22, 24.4])
@pytest.mark.parametrize("n", [1000, 8000])
def test_attention_of_one_key_far_above_the_rest(pkg, dev, tiles, spread, bits, n):
    """One key `bits` bits above all others whose values are zero, as a first
    token often is: the others carry the output, and keep their weights' bits.
    A weight is rounded to 11 bits, or to 2^-32 of the row's largest weight times
    value scale; no term grows with the number of keys beyond that."""
    d, block, group = 64, 64, 8
    blocks = -(-n // block)
    # 64 requests of a row and a key head for each query head, or one of many rows (keys up to them)
    requests, rows, kv_heads = (64, 1, 8) if tiles == 16 else (1, min(n, 4200), 1)
    kc, vc = (codes((blocks * block, 1, d), 21) * (spread / 8)).round(), codes((blocks * block, 1, d), 22, 12) + 60
    kc[..., 0], kc[0], vc[0] = 0, 0, 0
    kc[0, 0, 0] = 127
    every = lambda t: t.expand(-1, kv_heads, *t.shape[2:]).contiguous()  # noqa: E731
    one = torch.full((blocks, 1), 2.0 ** -6)
    cache, (k, v) = cache_of(pkg, dev, every(kc), every(vc), every(one), every(one), block)
    q = normal((1, 1, d), 23, dtype=torch.float32).expand(requests * rows, group, d).clone()
    scale = 0.125
    q[..., 0] = bits * 0.6931471805599453 / (127 / 64 * scale)
    q = q.half().to(dev)
    table = torch.arange(blocks, dtype=torch.int32, device=dev).expand(requests, blocks).contiguous()
    lens = torch.full((requests,), n, dtype=torch.int32, device=dev)
    cu = torch.arange(0, requests * rows + 1, rows, dtype=torch.int32, device=dev)
    got = pkg.kv_attention(q, cache, table, lens, cu=None if tiles == 16 else cu, scale=scale).cpu().double()
    qh = q[0, 0].cpu()
    for t in ([0, 63] if tiles == 16 else [rows // 2, rows - 2, rows - 1]):
        keys = n if tiles == 16 else n - rows + t + 1
        w, x = weights64(qh, k, keys, scale), v[:keys, 0]
        assert w[0] / w[1:].max() > 2.0 ** (bits - 2)
        want = w @ x
        # the output's half step; scores (fp32 sums of 64 products up to 20: 2^-13) and weights
        # (half a step of 11 bits); weights below 2^-14 of fp16 in steps of 2^-24, times up to 127
        room = HALF[torch.float16] * want.abs() + (2.0 ** -11 + 2.0 ** -13) * (w @ x.abs()) + \
            2.0 ** -32 * w.max() * x.abs().sum(0) + 2.0 ** -25
        off = (got[t] - want).abs() - room
        assert off.max() <= 0, (t, float(((got[t] - want).abs() / want.abs()).max()))
