"""The serving operators on the GPU: block tables and slots, the 8-bit
key/value cache, attention over it and sampling, each against a plain
implementation in 64 bits (or in lists and whole numbers), at the sizes and
masks where they can go wrong, and all of them together in a serving loop."""
import math

import numpy as np
import pytest
import torch

from gpu_util import gen, normal

pytestmark = pytest.mark.gpu

HALF = {torch.float16: 2.0 ** -11, torch.bfloat16: 2.0 ** -8}  # half a step of the type, relative


def ints(dev, *v, dtype=torch.int32):
    return torch.tensor(v, dtype=dtype, device=dev)


# ---- kv_plan -------------------------------------------------------------------------

class Pool:
    """What kv_plan does, with lists."""

    def __init__(self, requests, width, block, free):
        self.rows, self.lens = [[] for _ in range(requests)], [0] * requests
        self.width, self.block, self.free = width, block, list(free)

    def step(self, new, tokens):
        need = lambda r, n: -(-(self.lens[r] + n) // self.block) - len(self.rows[r])  # noqa: E731
        for r, n in enumerate(new):
            if n < 0:
                self.free += self.rows[r]
                self.rows[r], self.lens[r] = [], 0
        left, cu, slots, positions = len(self.free), [0], [-1] * tokens, [0] * tokens
        for r, n in enumerate(new):
            cu.append(cu[-1] + max(n, 0))
            if n <= 0 or len(self.rows[r]) + need(r, n) > self.width or cu[-1] > tokens:
                continue
            left -= need(r, n)
            if need(r, n) and left < 0:
                continue
            for _ in range(need(r, n)):
                self.rows[r].append(self.free.pop())
            for i in range(n):
                p = self.lens[r] + i
                slots[cu[r] + i] = self.rows[r][p // self.block] * self.block + p % self.block
                positions[cu[r] + i] = p
            self.lens[r] += n
        return slots, positions, cu


@pytest.mark.parametrize("requests, width, block, blocks, most, seed", [
    (1, 4, 16, 5, 70, 0), (7, 3, 32, 9, 40, 1), (65, 5, 16, 150, 9, 2), (300, 4, 64, 500, 130, 3),
    (1500, 3, 16, 2000, 3, 4), (4096, 2, 16, 3000, 2, 5),
])
def test_plan_over_many_steps(pkg, dev, requests, width, block, blocks, most, seed):
    """Requests that start, grow, idle and end, on a pool that runs short:
    every step's slots, and the table, lengths and stack it leaves."""
    rng = np.random.default_rng(seed)
    order = rng.permutation(blocks).tolist()
    pool = Pool(requests, width, block, order)
    free = ints(dev, *order)
    count, lens = ints(dev, blocks), torch.zeros(requests, dtype=torch.int32, device=dev)
    table = torch.full((requests, width + 3), -7, dtype=torch.int32, device=dev)[:, :width]
    for step in range(12):
        new = np.where(rng.random(requests) < 0.2, -1, rng.integers(0, most + 1, requests)).tolist()
        tokens = int(rng.integers(0, 2 * requests * most + 2))
        p = pkg.kv_plan(lens, ints(dev, *new), table, free, count, block_size=block, tokens=tokens)
        slots, positions, cu = pool.step(new, tokens)
        assert p.slots.tolist() == slots and p.positions.tolist() == positions and p.cu.tolist() == cu, step
        assert p.lens.tolist() == pool.lens and p.free_count.tolist() == [len(pool.free)], step
        assert free.tolist()[:len(pool.free)] == pool.free, step
        host = table.tolist()
        assert all(host[r][:len(row)] == row for r, row in enumerate(pool.rows)), step
        lens.copy_(p.lens)
        count.copy_(p.free_count)
    assert (table.as_strided((requests, 3), (width + 3, 1), width) == -7).all()  # (past the table's width)


def test_plan_without_requests_or_rows(pkg, dev):
    none, table = ints(dev), torch.zeros((0, 4), dtype=torch.int32, device=dev)
    p = pkg.kv_plan(none, none, table, ints(dev, 3, 1), ints(dev, 2), block_size=16, tokens=5)
    assert p.slots.tolist() == [-1] * 5 and p.positions.tolist() == [0] * 5
    assert p.cu.tolist() == [0] and p.free_count.tolist() == [2]
    p = pkg.kv_plan(ints(dev, 0), ints(dev, 1), torch.zeros((1, 0), dtype=torch.int32, device=dev), ints(dev, 3),
                    ints(dev, 1), block_size=16, tokens=1)
    assert p.slots.tolist() == [-1] and p.lens.tolist() == [0] and p.cu.tolist() == [0, 1]
    p = pkg.kv_plan(ints(dev, 5), ints(dev, 4), ints(dev, 2).view(1, 1), none, ints(dev, 0), block_size=16, tokens=0)
    assert p.slots.numel() == 0 and p.lens.tolist() == [5]


def test_plan_takes_numbers_out_of_range_as_the_nearest(pkg, dev):
    """Lengths past the table, a count past the stack, tokens past 2^31 in all."""
    table = ints(dev, 4, 5, 6, 7).view(2, 2)
    p = pkg.kv_plan(ints(dev, -3, 1000), ints(dev, 1, 1), table, ints(dev, 9, 8), ints(dev, 77), block_size=16, tokens=2)
    assert p.lens.tolist() == [1, 32] and p.slots.tolist() == [8 * 16, -1] and p.free_count.tolist() == [1]
    big = 2 ** 31 - 1
    p = pkg.kv_plan(ints(dev, 0, 0, 0), ints(dev, big, big, 3), torch.zeros((3, 2), dtype=torch.int32, device=dev),
                    ints(dev, 9, 8), ints(dev, 2), block_size=16, tokens=4)
    assert p.cu.tolist() == [0, big, big, big] and p.lens.tolist() == [0, 0, 0] and p.slots.tolist() == [-1] * 4


# ---- kv_append and kv_read -----------------------------------------------------------

def up11(x):
    """The smallest number of 11 significant bits that is at least x > 0 (float64, exact)."""
    m, e = np.frexp(x)
    return np.ldexp(np.ceil(np.ldexp(m, 11)), e - 11)


class Held:
    """A cache's values for one of K and V, in 64 bits: codes [cells, heads, d] and scales [blocks, heads]."""

    def __init__(self, blocks, heads, d, block):
        self.codes, self.scale = np.zeros((blocks * block, heads, d)), np.zeros((blocks, heads))
        self.block = block

    def append(self, x, slots):
        x = x.double().numpy()
        for b in sorted({s // self.block for s in slots if 0 <= s < len(self.codes)}):
            rows = [i for i, s in enumerate(slots) if s // self.block == b]
            cells = slice(b * self.block, (b + 1) * self.block)
            for h in range(x.shape[1]):
                v = x[rows, h]
                amax = np.abs(v).max()
                old = 0.0 if any(slots[i] % self.block == 0 for i in rows) else self.scale[b, h]
                now = old
                if not np.isfinite(amax):
                    now = math.nan
                elif amax > 127 * old:
                    now = max(up11(amax / 127), 2.0 ** -100)
                    if 127 * (now - np.ldexp(1.0, np.frexp(now)[1] - 11)) >= amax:
                        now -= np.ldexp(1.0, np.frexp(now)[1] - 11)  # (amax / 127 itself was rounded)
                    now = max(now, 2.0 ** -100)
                    self.codes[cells, h] = np.rint(self.codes[cells, h] * old / now)
                with np.errstate(all="ignore"):
                    self.codes[[slots[i] for i in rows], h] = np.nan_to_num(np.rint(v / now))
                self.scale[b, h] = now

    def at(self, slots):
        return self.codes[slots] * self.scale[[s // self.block for s in slots]][..., None]


def same_cache(cache, k, v):
    """The cache's tensors hold exactly the codes and scales of k and v."""
    n, h, b, dp = cache.k.shape
    d = cache.head_dim
    kc = cache.k.cpu().transpose(1, 2).reshape(n * b, h, dp)
    vc = cache.v.cpu().permute(0, 2, 4, 1, 3).reshape(n * b, h, dp)
    for codes, scale, want in ((kc, cache.k_scale, k), (vc, cache.v_scale, v)):
        np.testing.assert_array_equal(scale.cpu().double().numpy(), want.scale)
        live = np.repeat(np.isfinite(want.scale), b, 0)  # (a NaN block's codes say nothing)
        np.testing.assert_array_equal(codes[..., :d].double().numpy()[live], want.codes[live])
        assert not codes[..., d:].any()


APPENDS = [  # kv heads, head dim, block, dtype
    (1, 8, 16, torch.float16), (2, 64, 16, torch.bfloat16), (3, 40, 32, torch.float16), (8, 128, 64, torch.bfloat16),
    (4, 80, 128, torch.float16), (1, 96, 256, torch.bfloat16), (5, 120, 64, torch.float16),
]


@pytest.mark.parametrize("heads, d, block, dtype", APPENDS)
def test_append_in_pieces_of_every_length(pkg, dev, heads, d, block, dtype):
    """A request's tokens come one, two, many at a time, across blocks, with
    magnitudes that grow (codes rounded again) and a restart of its first
    block: codes and scales to the bit, k and v views of one projection."""
    blocks = 6
    cache = pkg.KVCache.empty(blocks, heads, d, block, device=dev)
    k, v = Held(blocks, heads, d, block), Held(blocks, heads, d, block)
    pages, at, g = [4, 1, 5, 0], 0, gen(d)
    for i, n in enumerate([1, 1, 2, 1, 13, 3, block - 7, block, 5, 1, block + 3]):
        kv = torch.randn((n, 2, heads, d), generator=g) * (0.3 * 1.4 ** i)
        kv = kv.to(dtype)
        if i == 3:
            at = 0  # the first block is begun again
        slots = [pages[p // block] * block + p % block for p in range(at, min(at + n, 4 * block))]
        n = len(slots)
        at += n
        kv = kv[:n]
        gpu = kv.to(dev)
        pkg.kv_append(cache, gpu[:, 0], gpu[:, 1], ints(dev, *slots, dtype=torch.int64))
        k.append(kv[:, 0], slots)
        v.append(kv[:, 1], slots)
        same_cache(cache, k, v)
    slots = [pages[p // block] * block + p % block for p in range(at)]
    kr, vr = pkg.kv_read(cache, ints(dev, *slots, dtype=torch.int64), dtype=dtype)
    for got, want in ((kr, k), (vr, v)):
        torch.testing.assert_close(got.cpu(), torch.from_numpy(want.at(slots)).to(dtype), rtol=0, atol=0)


@pytest.mark.parametrize("tokens, heads, d, block, dtype", [
    (1, 4, 64, 64, torch.float16), (700, 2, 72, 32, torch.bfloat16), (2100, 8, 64, 16, torch.float16),
    (5000, 4, 128, 256, torch.bfloat16),
])
def test_append_of_many_requests(pkg, dev, tokens, heads, d, block, dtype):
    """Runs of ragged lengths on a shuffled pool, some rows without a slot
    (padding, or past the cache), rows apart from each other in memory."""
    rng = np.random.default_rng(tokens)
    blocks = 2 * (tokens // block + 2)
    order, slots = rng.permutation(blocks).tolist(), []
    while len(slots) < tokens:
        a = int(rng.integers(0, block))
        b = order.pop()
        slots += list(range(b * block + a, b * block + int(rng.integers(a + 1, block + 1))))
        if rng.random() < 0.2:
            slots += [-1, blocks * block + 3][: int(rng.integers(1, 3))]
        if not order:
            slots += [-1] * tokens
    slots = slots[:tokens]
    wide = normal((tokens, heads, d + 7), 3, dtype=dtype)
    x, y = wide[..., 3:3 + d], normal((heads, tokens, d), 4, 5.0, dtype=dtype).transpose(0, 1)
    cache = pkg.KVCache.empty(blocks, heads, d, block, device=dev)
    k, v = Held(blocks, heads, d, block), Held(blocks, heads, d, block)
    gw, gy = wide.to(dev), y.transpose(0, 1).contiguous().to(dev)
    pkg.kv_append(cache, gw[..., 3:3 + d], gy.transpose(0, 1), ints(dev, *slots, dtype=torch.int64))
    k.append(x, slots)
    v.append(y, slots)
    same_cache(cache, k, v)
    kr, vr = pkg.kv_read(cache, ints(dev, *slots, dtype=torch.int64), dtype=dtype)
    inside = [i for i, s in enumerate(slots) if 0 <= s < blocks * block]
    at = [slots[i] for i in inside]
    outside = sorted(set(range(tokens)) - set(inside))
    for got, want in ((kr, k), (vr, v)):
        assert torch.equal(got.cpu()[inside], torch.from_numpy(want.at(at)).to(dtype))
        assert not got[outside].any()


@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
def test_append_of_extreme_values(pkg, dev, dtype):
    """Zero rows, the type's smallest and largest magnitudes, ties of two
    codes, infinities and NaN: exact, or a NaN scale until the block begins
    anew; other heads and blocks stay as they are."""
    top, tiny = torch.finfo(dtype).max, torch.finfo(dtype).smallest_normal
    sub = 2.0 ** -24 if dtype == torch.float16 else 2.0 ** -133
    d, block = 16, 16
    steps = torch.arange(d).double()
    rows = [steps * 0, steps * 0 + sub, steps * sub, steps * tiny, steps / 2, steps + 0.5, 127 - steps / 2, -steps * 254,
            steps * (top / 15), -steps * (top / 15)]
    cache = pkg.KVCache.empty(4, 2, d, block, device=dev)
    k, v = Held(4, 2, d, block), Held(4, 2, d, block)
    for i, row in enumerate(rows):
        x = torch.stack([row, row.flip(0) * (0.5 if i < 8 else 1)]).to(dtype)[None]
        pkg.kv_append(cache, x.to(dev), -x.to(dev), ints(dev, 2 * block + i, dtype=torch.int64))
        k.append(x, [2 * block + i])
        v.append(-x, [2 * block + i])
        same_cache(cache, k, v)
    kr, _ = pkg.kv_read(cache, ints(dev, *range(2 * block, 2 * block + 10), dtype=torch.int64), dtype=dtype)
    assert torch.isfinite(kr).all() and kr.abs().max() == top  # (held 127 * scale may be above it)
    for bad in (math.inf, -math.inf, math.nan):
        x = torch.ones((1, 2, d), dtype=dtype)
        x[0, 1, 5] = bad
        slot = ints(dev, 3 * block + 0, dtype=torch.int64)
        pkg.kv_append(cache, x.to(dev), x.to(dev), slot)
        assert torch.isnan(cache.k_scale[3, 1]) and torch.isnan(cache.v_scale[3, 1])
        assert torch.isfinite(cache.k_scale[3, 0])
        pkg.kv_append(cache, torch.ones_like(x).to(dev), torch.ones_like(x).to(dev), slot + 1)
        assert torch.isnan(cache.k_scale[3, 1]) and torch.isnan(pkg.kv_read(cache, slot + 1)[0][0, 1]).all()
        pkg.kv_append(cache, torch.ones_like(x).to(dev), torch.ones_like(x).to(dev), slot)
        assert torch.isfinite(cache.k_scale[3]).all() and (pkg.kv_read(cache, slot)[0] - 1).abs().max() < 2.0 ** -7
    np.testing.assert_array_equal(cache.k_scale[:3].cpu().double().numpy(), k.scale[:3])


# ---- kv_attention --------------------------------------------------------------------

def filled(pkg, dev, blocks, heads, d, block, seed, std=36):
    """A cache of random codes and scales, and its values [blocks * block, heads, d] in 64 bits."""
    g = gen(seed)
    cache = pkg.KVCache.empty(blocks, heads, d, block, device=dev)
    codes = [(torch.randn((blocks * block, heads, d), generator=g) * std).round().clamp(-127, 127) for _ in range(2)]
    scale = [((0.005 + 0.03 * torch.rand((blocks, heads), generator=g)).view(torch.int32) & ~0x1FFF).view(torch.float32)
             for _ in range(2)]
    cache.k[..., :d] = codes[0].view(blocks, block, heads, d).transpose(1, 2).to(torch.int8).to(dev)
    cache.v[..., :d, :] = codes[1].view(blocks, block // 16, 16, heads, d).permute(0, 3, 1, 4, 2).to(torch.int8).to(dev)
    cache.k_scale.copy_(scale[0])
    cache.v_scale.copy_(scale[1])
    values = [c.double() * s.double().repeat_interleave(block, 0)[..., None] for c, s in zip(codes, scale)]
    return cache, values


def attention64(q, k, v, block, table, lens, cu, scale, blocks):
    """The definition, row by row; and what a weight's rounding can move an output by."""
    out, room = torch.full(q.shape, math.nan, dtype=torch.float64), torch.zeros(q.shape, dtype=torch.float64)
    group = q.shape[1] // k.shape[1]
    for r in range(len(lens)):
        for i, t in enumerate(range(cu[r], cu[r + 1])):
            n = min(lens[r], table.shape[1] * block) - (cu[r + 1] - cu[r]) + i + 1
            p = torch.arange(max(n, 0))
            page = table[r, p // block].long()
            page, p = page[(page >= 0) & (page < blocks)], p[(page >= 0) & (page < blocks)]
            cells = page * block + p % block
            out[t] = 0
            for h in range(q.shape[1]) if len(cells) else ():
                w = (q[t, h].double() @ k[cells, h // group].T * scale).softmax(-1)
                x = v[cells, h // group]
                out[t, h] = w @ x
                # a weight is off by half an fp16 step of itself (2^-11), a score by 128 fp32
                # roundings of sums up to 50 (another 2^-11), and a weight below fp16's normal
                # range by 2^-25 of the largest weighted scale (twice: of the largest value it has)
                room[t, h] = 2 * 2.0 ** -11 * (w @ x.abs()) + len(cells) * 2.0 ** -24 * (w[:, None] * x.abs()).max()
    return out, room


def check_attention(got, q, k, v, block, table, lens, cu, scale, blocks, name=""):
    want, room = attention64(q.cpu(), k, v, block, table.cpu(), lens.tolist(), cu, scale, blocks)
    got = got.cpu().double()
    live = ~torch.isnan(want)
    # (65520 and more is infinity in fp16, whose largest number is 65504; 2^128 is in bf16)
    top = torch.finfo(q.dtype).max * (1 + HALF[q.dtype] / 2)
    over = live & (want.abs() - room > top)
    assert (got[over] == want[over].sign() * math.inf).all(), name
    live &= want.abs() + room < top
    off = (got - want).abs() - HALF[q.dtype] * want.abs() - room
    assert live.any() and off[live].max() <= 2.0 ** -25, (name, float(off[live].max()))


LENS = [0, 1, 2, 15, 16, 17, 31, 63, 64, 65, 100, 127, 128, 129, 255, 257, 300, 511, 513, 600]

SHAPES = [  # heads, kv heads, head dim, block, dtype
    (8, 2, 64, 16, torch.float16), (14, 2, 64, 64, torch.bfloat16), (4, 4, 128, 32, torch.float16),
    (32, 4, 128, 64, torch.bfloat16), (3, 1, 40, 128, torch.float16), (6, 2, 80, 16, torch.bfloat16),
    (40, 1, 96, 256, torch.float16), (1, 1, 8, 16, torch.bfloat16), (5, 5, 120, 32, torch.float16),
    (33, 1, 72, 64, torch.bfloat16),
]


@pytest.mark.parametrize("heads, kv_heads, d, block, dtype", SHAPES)
def test_attention_of_one_token_each(pkg, dev, heads, kv_heads, d, block, dtype):
    blocks, R = 60 * 16 // block * 16 + 40, len(LENS)
    cache, (k, v) = filled(pkg, dev, blocks, kv_heads, d, block, 7)
    width = -(-max(LENS) // block)
    table = torch.randint(0, blocks, (R, width), generator=gen(8), dtype=torch.int32).to(dev)
    lens = ints(dev, *LENS)
    q = normal((R, heads, d), 9, 1.5, dtype=dtype).to(dev)
    got = pkg.kv_attention(q, cache, table, lens)
    check_attention(got, q, k, v, block, table, lens, list(range(R + 1)), d ** -0.5, blocks)
    assert not got[0].any()  # no key: zeros
    for r in (1, 9, 19):  # alone: the keys shared out over workgroups, or not
        one = pkg.kv_attention(q[r:r + 1], cache, table[r:r + 1], lens[r:r + 1], scale=0.3)
        check_attention(one, q[r:r + 1], k, v, block, table[r:r + 1], lens[r:r + 1], [0, 1], 0.3, blocks, r)


RAGGED = [  # rows of each request, its tokens
    ([1, 0, 3, 2], [5, 7, 64, 2]), ([17], [17]), ([5, 1, 4, 0, 2], [200, 0, 4, 9, 130]), ([70, 3], [333, 3]),
    ([1] * 9, [1, 2, 30, 64, 65, 100, 0, 7, 63]), ([0, 0], [5, 5]), ([130, 33, 64], [130, 400, 64]), ([6], [4]),
]


@pytest.mark.parametrize("heads, kv_heads, d, block, dtype", SHAPES[:8])
def test_attention_of_ragged_rows(pkg, dev, heads, kv_heads, d, block, dtype):
    blocks = 64
    cache, (k, v) = filled(pkg, dev, blocks, kv_heads, d, block, 17)
    for rows, held in RAGGED:
        width = -(-max(held) // block) + 1
        table = torch.randint(0, blocks, (len(rows), width), generator=gen(18), dtype=torch.int32).to(dev)
        cu = [0] + np.cumsum(rows).tolist()
        q = normal((cu[-1] + 5, heads, d), 19, 1.5, dtype=dtype).to(dev)  # five rows of no request
        out = torch.full_like(q, 7.0)
        lens = ints(dev, *held)
        got = pkg.kv_attention(q, cache, table, lens, cu=ints(dev, *cu), out=out)
        assert got is out and (out[cu[-1]:] == 7).all(), rows  # left as they were
        if cu[-1]:
            check_attention(out, q, k, v, block, table, lens, cu, d ** -0.5, blocks, rows)


@pytest.mark.parametrize("heads, kv_heads, d, block, dtype", SHAPES)
def test_attention_of_many_rows(pkg, dev, heads, kv_heads, d, block, dtype):
    """Tiles of 128 rows: requests that end inside one, an empty one, a prompt
    without a context, a context that ends inside a page; rows of no request."""
    a = 2200 // heads + 1
    rows, held = [a, 0, a + 3], [a + 37, 5, a + 3]
    cu = [0] + np.cumsum(rows).tolist()
    blocks, width = 48, -(-max(held) // block)
    cache, (k, v) = filled(pkg, dev, blocks, kv_heads, d, block, 23)
    table = torch.randint(0, blocks, (3, width), generator=gen(24), dtype=torch.int32).to(dev)
    q = normal((cu[-1] + 7, heads, d), 25, 1.5, dtype=dtype).to(dev)
    out = torch.full_like(q, 7.0)
    lens = ints(dev, *held)
    pkg.kv_attention(q, cache, table, lens, cu=ints(dev, *cu), out=out)
    assert (out[cu[-1]:] == 7).all()
    check_attention(out, q, k, v, block, table, lens, cu, d ** -0.5, blocks)


def test_attention_of_a_prompt(pkg, dev):
    """Rows in the hundreds over a longer context: several tiles a request, in both types."""
    for dtype, heads, kv_heads, d in ((torch.float16, 8, 2, 128), (torch.bfloat16, 6, 1, 64)):
        blocks, block = 80, 32
        cache, (k, v) = filled(pkg, dev, blocks, kv_heads, d, block, 27)
        table = torch.randperm(blocks, generator=gen(28))[:60].view(2, 30).to(torch.int32).to(dev)
        lens, cu = ints(dev, 941, 777), [0, 333, 500]
        q = normal((500, heads, d), 29, 1.5, dtype=dtype).to(dev)
        got = pkg.kv_attention(q, cache, table, lens, cu=ints(dev, *cu))
        check_attention(got, q, k, v, block, table, lens, cu, d ** -0.5, blocks)


def test_attention_reads_any_view_and_writes_any_rows(pkg, dev):
    """q a view of a projection (odd offset), tables and out with rows apart,
    out over q itself, out over other elements of q's buffer, operands of
    other strides."""
    heads, kv_heads, d, block, blocks = 6, 2, 64, 16, 40
    cache, (k, v) = filled(pkg, dev, blocks, kv_heads, d, block, 37)
    lens = ints(dev, 40, 100, 7)
    wide = torch.randint(0, blocks, (3, 20), generator=gen(38), dtype=torch.int32).to(dev)
    table = wide[:, 5:12]
    buf = normal((3, 1 + 2 * heads * d), 39, 1.5).to(dev)
    q = buf[:, 1:1 + heads * d].view(3, heads, d)
    want = pkg.kv_attention(q.contiguous(), cache, table.contiguous(), lens)
    check_attention(want, q, k, v, block, table, lens, [0, 1, 2, 3], d ** -0.5, blocks)
    assert torch.equal(pkg.kv_attention(q, cache, table, lens), want)
    assert torch.equal(pkg.kv_attention(q.transpose(1, 2).contiguous().transpose(1, 2), cache, table, lens), want)
    out = torch.zeros((heads, 3, d + 3), dtype=q.dtype, device=dev)[..., 3:].transpose(0, 1)
    assert pkg.kv_attention(q, cache, table, lens, out=out) is out and torch.equal(out, want)
    beside = buf[:, 1 + heads * d:].view(3, heads, d)
    assert torch.equal(pkg.kv_attention(q, cache, table, lens, out=beside), want)
    back = torch.zeros((3, heads, 2 * d), dtype=q.dtype, device=dev)[..., ::2]
    assert torch.equal(pkg.kv_attention(q, cache, table, lens, out=back), want)
    shifted = buf[:, 65:65 + heads * d].view(3, heads, d)  # over other rows' elements of q
    qc = q.clone()
    got = pkg.kv_attention(q, cache, table, lens, out=shifted)
    assert torch.equal(got, want)
    buf[:, 1:1 + heads * d].view(3, heads, d).copy_(qc)
    assert torch.equal(pkg.kv_attention(q, cache, table, lens, out=q), want)
    with pytest.raises(pkg.HxmiError, match="share"):
        pkg.kv_attention(qc, cache, table, lens, out=torch.empty((1, heads, d), dtype=q.dtype, device=dev).expand(3, -1, -1))


def test_attention_leaves_out_pages_outside_the_cache(pkg, dev):
    """Entries of no block, in the middle, at the end, everywhere; lengths past
    the table; a NaN page behind a request's tokens or behind a row's."""
    heads, kv_heads, d, block, blocks = 4, 2, 64, 16, 12
    cache, (k, v) = filled(pkg, dev, blocks, kv_heads, d, block, 47)
    table = ints(dev, 3, -1, 5, 2 ** 31 - 1, 1, 1, 2, 3, 4, 9, -5, 12, -1, -1, -2 ** 31, 0, 7, 7, 7, 7).view(4, 5)
    lens = ints(dev, 80, 70, 48, 500)
    q = normal((4, heads, d), 49, 1.5).to(dev)
    got = pkg.kv_attention(q, cache, table, lens)
    check_attention(got, q, k, v, block, table, lens, [0, 1, 2, 3, 4], d ** -0.5, blocks)
    assert not got[2].any()
    # block 11 has NaN scales: it lies behind the keys of request 0, and behind rows 0 and 1 of request 1
    cache.k_scale[11] = math.nan
    cache.v_scale[11] = math.nan
    table = ints(dev, 3, 2, 11, 5, 1, 11).view(2, 3)
    lens, cu = ints(dev, 32, 34), [0, 1, 5]
    q = normal((5, heads, d), 50, 1.5).to(dev)
    got = pkg.kv_attention(q, cache, table, lens, cu=ints(dev, *cu))
    assert torch.isfinite(got[:3]).all() and torch.isnan(got[3:]).all()
    check_attention(got[:3], q[:3], k, v, block, table, ints(dev, 32, 32), [0, 1, 3], d ** -0.5, blocks)


def test_attention_of_unlike_scales(pkg, dev):
    """Pages whose V scales lie up to 2^60 apart (zero among them), weights
    that favour the small ones; q from 2^-60 to 2^60 in bf16: held apart from
    the weights, no page's share is lost."""
    heads, kv_heads, d, block, blocks = 16, 1, 64, 16, 24
    cache, (k, v) = filled(pkg, dev, blocks, kv_heads, d, block, 57)
    e = torch.arange(blocks).double()
    factor = torch.where(e % 5 == 4, 0, torch.exp2(((e * 7) % 13 - 6) * 5))
    cache.v_scale.mul_(factor[:, None].float().to(dev))
    v = v * factor.repeat_interleave(block)[:, None, None]
    table = torch.arange(blocks, dtype=torch.int32, device=dev).view(1, blocks)
    lens = ints(dev, blocks * block - 3)
    q = normal((1, heads, d), 58, 2.0, dtype=torch.bfloat16)
    q = (q.double() * torch.exp2(torch.arange(heads).double() * 8 - 60)[None, :, None]).to(torch.bfloat16).to(dev)
    for scale in (2.0 ** -60, 0.125, 2.0 ** 30):
        small = q[:, : (16 if scale < 1e-9 else 8 if scale < 1 else 4)]  # (scores that fp32 holds exactly enough)
        small = small.repeat(1, 16 // small.shape[1], 1)
        got = pkg.kv_attention(small, cache, table, lens, scale=scale)
        check_attention(got, small, k, v, block, table, lens, [0, 1], scale, blocks, scale)


def test_attention_of_many_rows_over_bad_pages_and_unlike_scales(pkg, dev):
    """As above in tiles of 128 rows: missing pages, a NaN page that only the
    last rows see, pages whose V scales lie up to 2^60 apart."""
    heads, kv_heads, d, block, blocks = 10, 1, 128, 16, 40
    cache, (k, v) = filled(pkg, dev, blocks, kv_heads, d, block, 62)
    e = torch.arange(blocks).double()
    factor = torch.where(e % 5 == 4, 0, torch.exp2(((e * 7) % 13 - 6) * 5))
    cache.v_scale.mul_(factor[:, None].float().to(dev))
    v = v * factor.repeat_interleave(block)[:, None, None]
    table = torch.randperm(blocks - 1, generator=gen(63)).to(torch.int32)[:32].view(2, 16)
    table[0, [3, 7]] = torch.tensor([-1, blocks], dtype=torch.int32)
    table[1, :10] = -7
    table[1, 15] = blocks - 1
    cache.k_scale[blocks - 1] = math.nan
    cache.v_scale[blocks - 1] = math.nan
    table, lens, cu = table.to(dev), ints(dev, 250, 250), [0, 200, 440]  # row 240 - 10 of the second sees key 240
    q = normal((440, heads, d), 64, 1.5).to(dev)
    for scale in (d ** -0.5, 2.0 ** -20):
        got = pkg.kv_attention(q, cache, table, lens, cu=ints(dev, *cu), scale=scale)
        nan = torch.isnan(got).flatten(1).any(1).cpu()
        assert not nan[:430].any() and nan[430:].all()
        check_attention(got[:430], q[:430], k, v, block, table, ints(dev, 250, 240), [0, 200, 430], scale, blocks)


def test_attention_past_32_bit_offsets(pkg, dev):
    """A cache of more than 4 GiB of codes each: pages at its start and end."""
    heads, kv_heads, d, block, blocks = 8, 8, 128, 64, 70000
    cache = pkg.KVCache.empty(blocks, kv_heads, d, block, device=dev)
    assert cache.k.numel() > 1 << 32
    pages = [0, blocks - 1, 65536, 32768]
    n = 3 * block + 17
    slots = ints(dev, *(pages[p // block] * block + p % block for p in range(n)), dtype=torch.int64)
    x = normal((2, n, kv_heads, d), 67).to(dev)
    pkg.kv_append(cache, x[0], x[1], slots)
    k, v = pkg.kv_read(cache, slots)
    small = pkg.KVCache.empty(4, kv_heads, d, block, device=dev)
    here = torch.arange(n, device=dev)
    pkg.kv_append(small, x[0], x[1], here)
    ks, vs = pkg.kv_read(small, here)
    assert torch.equal(k, ks) and torch.equal(v, vs)
    q = normal((1, heads, d), 68).to(dev)
    got = pkg.kv_attention(q, cache, ints(dev, *pages).view(1, 4), ints(dev, n))
    want = pkg.kv_attention(q, small, ints(dev, 0, 1, 2, 3).view(1, 4), ints(dev, n))
    assert torch.equal(got, want) and want.abs().max() > 0


def test_attention_of_a_long_context(pkg, dev):
    """One token over 70001 keys: shares of many groups a wave, joined."""
    heads, kv_heads, d, block = 8, 2, 64, 128
    blocks = 70001 // block + 1
    cache, (k, v) = filled(pkg, dev, blocks, kv_heads, d, block, 77)
    table = torch.randperm(blocks, generator=gen(78)).to(torch.int32).view(1, blocks).to(dev)
    q = normal((1, heads, d), 79, 2.0).to(dev)
    lens = ints(dev, 70001)
    got = pkg.kv_attention(q, cache, table, lens)
    check_attention(got, q, k, v, block, table, lens, [0, 1], d ** -0.5, blocks)
    assert all(torch.equal(pkg.kv_attention(q, cache, table, lens), got) for _ in range(5))


# ---- sample --------------------------------------------------------------------------

def sample64(x, u, T=1.0, k=0, p=1.0, m=0.0):
    """One row, from the definition in 64 bits."""
    x = np.asarray(x, dtype=np.float64)
    if np.isnan(x).any() or x.max() == -math.inf:
        return -1
    if not T > 0:
        return int(np.argmax(x))
    with np.errstate(invalid="ignore"):
        w = np.where(x == x.max(), 1.0, np.exp((x - x.max()) / T))
    order = np.lexsort((np.arange(len(x)), -x))
    order = order[:k] if 0 < k < len(x) else order
    if p < 1:
        before = np.concatenate([[0], np.cumsum(w[order])[:-1]])
        order = order[: max(1, np.searchsorted(before, p * math.fsum(w[order]), side="left"))]
    kept = np.sort(order[w[order] >= min(max(m, 0.0), 1.0)])
    cum = np.cumsum(w[kept])
    return int(kept[np.searchsorted(cum, u * cum[-1], side="right")])


def check_sample(pkg, dev, x, u, **kw):
    got = pkg.sample(x.to(dev), u.to(dev), **{n: v.to(dev) if isinstance(v, torch.Tensor) else v for n, v in kw.items()})
    names = dict(temperature="T", top_k="k", top_p="p", min_p="m")
    own = lambda v, r: v[r].item() if isinstance(v, torch.Tensor) else v  # noqa: E731
    f32 = lambda v: v if isinstance(v, int) else float(np.float32(v))  # noqa: E731
    want = [sample64(x[r].double().numpy(), u[r].item(), **{names[n]: f32(own(v, r)) for n, v in kw.items()})
            for r in range(len(x))]
    assert got.dtype == torch.int64 and got.tolist() == want, (kw, [(r, a, b) for r, (a, b) in
                                                                   enumerate(zip(got.tolist(), want)) if a != b][:5])


SETTINGS = [
    {}, dict(temperature=0.0), dict(temperature=0.05), dict(temperature=30.0), dict(top_k=1), dict(top_k=3),
    dict(top_k=50, temperature=0.7), dict(top_p=0.9), dict(top_p=0.5, temperature=1.3), dict(top_p=0.0),
    dict(top_p=1e-6), dict(min_p=0.1), dict(min_p=1.0), dict(min_p=2.0, top_p=0.999), dict(top_k=40, top_p=0.8, min_p=0.05),
    dict(top_k=10 ** 6, top_p=1.0), dict(top_k=-1),
]


@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16, torch.float32])
@pytest.mark.parametrize("vocab", [1, 2, 7, 8, 9, 511, 512, 513, 1000, 8191, 33001])
def test_sample(pkg, dev, dtype, vocab):
    x = normal((6, vocab + 3), vocab, 2.5, dtype=dtype)[:, 1:1 + vocab]  # (rows off the 16-byte grid)
    u = torch.rand(6, generator=gen(vocab))
    for s in SETTINGS:
        check_sample(pkg, dev, x, u, **s)


@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16, torch.float32])
def test_sample_of_masked_and_equal_logits(pkg, dev, dtype):
    """Masks that leave one token, a few or none; equal logits (the lowest
    index first), both zeros; infinities and NaN; u at its ends."""
    V, inf = 1300, math.inf
    low = torch.finfo(dtype).min
    rows = [torch.zeros(V), torch.full((V,), -inf), torch.full((V,), low), torch.full((V,), 3.0)]
    one = torch.full((V,), -inf)
    one[777] = -5.0
    few = torch.full((V,), low)
    few[[5, 600, 1299]] = torch.tensor([1.0, 1.0, 2.0])
    signed = torch.zeros(V)
    signed[::3] = -0.0
    top = torch.randn(V, generator=gen(1))
    top[[9, 1000]] = inf
    nan = torch.randn(V, generator=gen(2))
    nan[1200] = math.nan
    neg_nan = torch.randn(V, generator=gen(3))
    neg_nan[0] = -math.nan
    steps = torch.arange(V).float() // 100  # 100 equal ones each
    x = torch.stack([*rows, one, few, signed, top, nan, neg_nan, steps, -steps]).to(dtype)
    settings = [{}, dict(temperature=0.0), dict(top_k=2), dict(top_k=150, top_p=0.9), dict(top_p=0.5), dict(min_p=0.5),
                dict(min_p=1.0, top_k=3), dict(top_p=0.25, temperature=4.0), dict(top_k=1299), dict(top_k=1300)]
    for s in settings:
        for u in (0.0, 0.3, 0.5, 0.99999994):
            check_sample(pkg, dev, x, torch.full((len(x),), u), **s)


def test_sample_of_a_large_vocabulary(pkg, dev):
    """Vocabularies up to 2^20, flat ones (every token kept), own settings a row."""
    for vocab, dtype, std in ((151936, torch.bfloat16, 2.5), (151937, torch.float32, 0.01), (1 << 20, torch.float16, 1.0)):
        B = 8
        x = normal((B, vocab), 5, std, dtype=dtype)
        g = gen(6)
        u = torch.rand(B, generator=g)
        check_sample(pkg, dev, x, u)
        check_sample(pkg, dev, x, u, temperature=torch.rand(B, generator=g) * 2 - 0.2,
                     top_k=torch.randint(-1, 4000, (B,), generator=g, dtype=torch.int32),
                     top_p=torch.rand(B, generator=g) * 1.2, min_p=torch.rand(B, generator=g) * 0.01)
        check_sample(pkg, dev, x, u, top_p=0.97)


@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16, torch.float32])
def test_sample_at_extreme_temperatures(pkg, dev, dtype):
    """Temperatures so low that the next smaller logit has no weight (below
    1e-9 of the logits too, where their difference from a bound rounds away),
    and so high that all have the same."""
    x = normal((6, 3000), 15, 2.5, dtype=dtype)
    x[2] = (x[2].float() * 4000).clamp(-60000, 60000).to(dtype)
    x[3] = -x[2].abs() - 1
    x[4, 5:] = x[4, 0]
    x[5] = torch.finfo(dtype).min
    x[5, 100:200] = 0
    u = torch.rand(6, generator=gen(16))
    for t in (1e-38, 1e-9, 1e-7, 1e-5, 1e-3, 1e5, 1e10):
        for kw in ({}, dict(top_k=20), dict(top_k=700), dict(top_p=0.7), dict(top_k=900, top_p=0.5), dict(top_k=9, min_p=0.3)):
            check_sample(pkg, dev, x, u, temperature=t, **kw)
    check_sample(pkg, dev, x[:5], u[:5], temperature=torch.full((5,), math.inf), top_k=20)
    check_sample(pkg, dev, x[:5], u[:5], temperature=torch.full((5,), math.inf), top_p=0.4)


@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16, torch.float32])
def test_sample_of_crowded_values(pkg, dev, dtype):
    """More equal (or nearly equal) logits than a 16-bit count or a list holds."""
    V = 140000
    g = gen(17)
    few = torch.randint(0, 3, (V,), generator=g).float()
    mostly = torch.where(torch.rand(V, generator=g) < 0.9, -1.0, torch.randn(V, generator=g))
    near = 1 + torch.rand(V, generator=g) * 2.0 ** -9  # (fp32: within one of its upper 16 bits' values)
    low = torch.full((V,), torch.finfo(dtype).min)
    low[::17] = torch.randn(V)[::17]
    x = torch.stack([torch.ones(V), few, mostly, near, low]).to(dtype)
    u = torch.rand(5, generator=g)
    for kw in ({}, dict(top_k=50), dict(top_k=600), dict(top_k=70001), dict(top_p=0.9), dict(top_k=100000, top_p=0.6),
               dict(top_k=20, top_p=0.6), dict(min_p=0.2, top_p=0.95)):
        check_sample(pkg, dev, x, u, **kw)


def test_sample_of_other_shapes(pkg, dev):
    """Leading dimensions, columns of a wider tensor, other strides, one row repeated, none."""
    x, u = normal((2, 3, 400), 7).to(dev), torch.rand((2, 3), generator=gen(8)).to(dev)
    want = pkg.sample(x.view(6, 400), u.view(6), top_k=20).view(2, 3)
    assert torch.equal(pkg.sample(x, u, top_k=20), want)
    k = torch.full((2, 3), 20, dtype=torch.int32, device=dev)
    assert torch.equal(pkg.sample(x, u, top_k=k), want)
    assert torch.equal(pkg.sample(x.transpose(0, 1), u.t(), top_k=k.t()), want.t())
    assert torch.equal(pkg.sample(x.transpose(1, 2).contiguous().transpose(1, 2), u, top_k=20), want)
    assert pkg.sample(x[0, 0], u[0, 0], top_k=20) == want[0, 0]
    row = x[0, :1].expand(3, 400)
    assert torch.equal(pkg.sample(row, u[0], top_k=20), pkg.sample(row.contiguous(), u[0], top_k=20))
    assert pkg.sample(x[:0], u[:0]).shape == (0, 3)


# ---- forms, streams, refusals --------------------------------------------------------

def serving_calls(pkg, dev):
    """(name, whether the native entry takes it, call giving tensors)"""
    block, heads, d = 16, 2, 64
    cache, _ = filled(pkg, dev, 20, heads, d, block, 87)
    q = normal((3, 8, d), 88).to(dev)
    x, slots = normal((4, heads, d), 89).to(dev), ints(dev, 5, 6, 40, -1, dtype=torch.int64)
    table, lens = torch.arange(12, dtype=torch.int32, device=dev).view(3, 4), ints(dev, 64, 3, 20)
    logits, u = normal((3, 500), 90).to(dev), torch.rand(3, generator=gen(91)).to(dev)

    def appended(k, v, s):
        c = pkg.KVCache(cache.k.clone(), cache.v.clone(), cache.k_scale.clone(), cache.v_scale.clone(), d)
        pkg.kv_append(c, k, v, s)
        return c.k, c.v, c.k_scale, c.v_scale

    def planned(new):
        t = table.clone()
        return (*pkg.kv_plan(lens, new, t, ints(dev, 19, 18), ints(dev, 2), block_size=block, tokens=9), t)

    return [
        ("append", True, lambda: appended(x, x, slots)),
        ("append strided values", False, lambda: appended(x, x.transpose(1, 2).contiguous().transpose(1, 2), slots)),
        ("read", True, lambda: pkg.kv_read(cache, slots, torch.bfloat16)),
        ("read strided slots", False, lambda: pkg.kv_read(cache, slots.repeat_interleave(2)[::2])),
        ("attention", True, lambda: (pkg.kv_attention(q, cache, table, lens),)),
        ("attention ragged out", True, lambda: (pkg.kv_attention(q, cache, table, lens, cu=ints(dev, 0, 2, 2, 3), scale=1,
                                                                 out=torch.zeros_like(q)),)),
        ("attention over q", False, lambda: (lambda c: (pkg.kv_attention(c, cache, table, lens, out=c),))(q.clone())),
        ("plan", True, lambda: planned(ints(dev, 1, -1, 2))),
        ("plan strided", False, lambda: planned(ints(dev, 1, 9, -1, 9, 2)[::2])),
        ("sample", True, lambda: (pkg.sample(logits, u, top_k=9, top_p=0.9),)),
        ("sample own", True, lambda: (pkg.sample(logits, u, min_p=u * 0.1),)),
        ("sample columns", True, lambda: (pkg.sample(logits[:, 7:400], u, temperature=2),)),
        ("sample strided u", False, lambda: (pkg.sample(logits, u.repeat_interleave(2)[::2]),)),
    ]


def test_native_form_equals_python_form(pkg, dev, monkeypatch):
    getattr(pkg.hxmi._ops, "gemm")  # loads the module
    real, taken = pkg.hxmi._ops, []

    class Spy:
        def __getattr__(self, name):
            def f(*args):
                y = getattr(real, name)(*args)
                taken.append(y is not None)
                return y
            return f

    for name, native, call in serving_calls(pkg, dev):
        monkeypatch.setattr(pkg.hxmi, "_ops", Spy())
        taken.clear()
        got = call()
        assert taken[0] == native, name
        monkeypatch.setattr(pkg.hxmi, "_ops", pkg.hxmi._PythonForms())
        want = call()
        assert len(got) == len(want) and all(torch.equal(a, b) for a, b in zip(got, want)), name


def test_calls_run_on_the_current_stream(pkg, dev):
    want = [[t.clone() for t in call()] for _, _, call in serving_calls(pkg, dev)]
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        for (name, _, call), w in zip(serving_calls(pkg, dev), want):
            got = call()
            s.synchronize()
            assert all(torch.equal(a, b) for a, b in zip(got, w)), name


def test_two_streams_share_nothing(pkg, dev):
    """Calls that share their keys out, in flight on two streams at once."""
    cache, _ = filled(pkg, dev, 128, 2, 64, 64, 97)
    table = torch.arange(128, dtype=torch.int32, device=dev).view(1, 128)
    lens = ints(dev, 8000)
    qs = [normal((1, 8, 64), i).to(dev) for i in range(2)]
    want = [pkg.kv_attention(q, cache, table, lens) for q in qs]
    streams = [torch.cuda.Stream() for _ in range(2)]
    torch.cuda.synchronize()
    got = [[], []]
    for _ in range(30):
        for i, s in enumerate(streams):
            with torch.cuda.stream(s):
                got[i].append(pkg.kv_attention(qs[i], cache, table, lens))
    torch.cuda.synchronize()
    assert all(torch.equal(g, w) for gs, w in zip(got, want) for g in gs)


def test_python_forms_refuse(pkg, dev):
    c = pkg.KVCache.empty(4, 2, 64, 16, device=dev)
    x, q = torch.zeros((3, 2, 64), dtype=torch.float16, device=dev), torch.zeros((3, 4, 64), dtype=torch.float16, device=dev)
    s, table, lens = ints(dev, 0, 1, 2, dtype=torch.int64), torch.zeros((3, 2), dtype=torch.int32, device=dev), ints(dev, 1, 1, 1)
    u, logits = torch.zeros(3, device=dev), torch.zeros((3, 50), device=dev)
    hx = pkg
    bad = [
        ("dtype", lambda: hx.kv_append(c, x.float(), x.float(), s)), ("dtype", lambda: hx.kv_append(c, x, x.bfloat16(), s)),
        ("tokens, 2, 64", lambda: hx.kv_append(c, x[:, :1], x[:, :1], s)), ("tokens, 2, 64", lambda: hx.kv_append(c, x, x[:2], s)),
        ("slots", lambda: hx.kv_append(c, x, x, s.int())), ("slots", lambda: hx.kv_append(c, x, x, s[:2])),
        ("KVCache", lambda: hx.kv_append((c.k, c.v), x, x, s)), ("fp16 or bf16", lambda: hx.kv_read(c, s, torch.float32)),
        ("slots", lambda: hx.kv_read(c, s.view(3, 1))),
        ("belong", lambda: hx.kv_read(hx.KVCache(c.k, c.v[:2], c.k_scale, c.v_scale, 64), s)),
        ("belong", lambda: hx.kv_read(hx.KVCache(c.k, c.v, c.k_scale, c.v_scale, 40), s)),
        ("head_dim", lambda: hx.kv_read(hx.KVCache(c.k, c.v, c.k_scale, c.v_scale, 60), s)),
        ("int8", lambda: hx.kv_read(hx.KVCache(c.k.short(), c.v, c.k_scale, c.v_scale, 64), s)),
        ("contiguous", lambda: hx.kv_read(hx.KVCache(c.k.transpose(0, 1).contiguous().transpose(0, 1), c.v, c.k_scale,
                                                     c.v_scale, 64), s)),
        ("fp16 or bf16 q", lambda: hx.kv_attention(q.float(), c, table, lens)),
        ("multiple of 2 heads", lambda: hx.kv_attention(q[:, :3], c, table, lens)),
        ("multiple of 2 heads", lambda: hx.kv_attention(q[..., :32], c, table, lens)),
        ("block_table", lambda: hx.kv_attention(q, c, table.long(), lens)),
        ("block_table", lambda: hx.kv_attention(q, c, table[:2], lens)),
        ("unit stride", lambda: hx.kv_attention(q, c, table.t().contiguous().t(), lens)),
        ("share", lambda: hx.kv_attention(q, c, table[:1].expand(3, 2), lens)),
        ("lens", lambda: hx.kv_attention(q, c, table, lens.long())), ("one row", lambda: hx.kv_attention(q[:2], c, table, lens)),
        ("cu", lambda: hx.kv_attention(q, c, table, lens, cu=lens)), ("scale", lambda: hx.kv_attention(q, c, table, lens, scale=0)),
        ("scale", lambda: hx.kv_attention(q, c, table, lens, scale=1e39)),
        ("out", lambda: hx.kv_attention(q, c, table, lens, out=q.float())),
        ("without blocks", lambda: hx.kv_attention(q, hx.KVCache.empty(0, 2, 64, 16, device=dev), table, lens)),
        ("logits", lambda: hx.sample(logits.double(), u)), ("u must", lambda: hx.sample(logits, u[:2])),
        ("u must", lambda: hx.sample(logits, u.half())), ("top_k", lambda: hx.sample(logits, u, top_k=u)),
        ("top_p", lambda: hx.sample(logits, u, top_p=u[:2])), ("temperature", lambda: hx.sample(logits, u, temperature=-1)),
        ("temperature", lambda: hx.sample(logits, u, temperature=math.nan)), ("top_p", lambda: hx.sample(logits, u, top_p=math.nan)),
        ("vocab", lambda: hx.sample(logits[:, :0], u)),
        ("new", lambda: hx.kv_plan(lens, lens[:2], table, lens, lens[:1], block_size=16, tokens=3)),
        ("free_count", lambda: hx.kv_plan(lens, lens, table, lens, lens, block_size=16, tokens=3)),
        ("block_size", lambda: hx.kv_plan(lens, lens, table, lens, lens[:1], block_size=17, tokens=3)),
        ("tokens", lambda: hx.kv_plan(lens, lens, table, lens, lens[:1], block_size=16, tokens=-3)),
        ("free_blocks", lambda: hx.kv_plan(lens, lens, table, lens.repeat(2)[::2], lens[:1], block_size=16, tokens=3)),
        ("lens", lambda: hx.kv_plan(lens.long(), lens, table, lens, lens[:1], block_size=16, tokens=3)),
        ("4096", lambda: hx.kv_plan(*(torch.zeros(4097, dtype=torch.int32, device=dev),) * 2,
                                    torch.zeros((4097, 1), dtype=torch.int32, device=dev), lens, lens[:1], block_size=16,
                                    tokens=3)),
        ("GPU", lambda: hx.kv_attention(q, c, table.cpu(), lens)),
    ]
    for i, (msg, call) in enumerate(bad):
        with pytest.raises(pkg.HxmiError, match=msg):
            call()
            pytest.fail(f"call {i} ({msg}) was taken")


# ---- together ------------------------------------------------------------------------

class Server:
    """A one-layer decoder with a cache: embeddings, one projection to q, k and
    v, attention over the cache, the output row added, logits, a token."""

    def __init__(self, pkg, dev, dtype, seed):
        self.pkg, self.heads, self.kv, self.d, self.block, self.blocks, self.R = pkg, 4, 2, 64, 16, 18, 3
        H = self.heads * self.d
        n = lambda *sh, i, std=1.0: normal(sh, seed + i, std, dtype=dtype).to(dev)  # noqa: E731
        self.embed, self.wqkv = n(200, H, i=0), n((self.heads + 2 * self.kv) * self.d, H, i=1, std=0.06)
        self.wo, self.lm = n(H, H, i=2, std=0.06), n(200, H, i=3, std=0.15)
        self.cache = pkg.KVCache.empty(self.blocks, self.kv, self.d, self.block, device=dev)
        self.table = torch.full((self.R, 6), -1, dtype=torch.int32, device=dev)
        self.free = torch.arange(self.blocks, dtype=torch.int32, device=dev)
        self.count, self.lens = ints(dev, self.blocks), torch.zeros(self.R, dtype=torch.int32, device=dev)

    def step(self, ids, new, u, rows):
        """Rows `ids` of the requests' new tokens; a token for each request."""
        pkg, H = self.pkg, self.heads * self.d
        p = pkg.kv_plan(self.lens, new, self.table, self.free, self.count, block_size=self.block, tokens=rows)
        x = self.embed[ids]
        qkv = pkg.linear(x, self.wqkv).view(rows, -1, self.d)
        q, k, v = qkv.split([self.heads, self.kv, self.kv], 1)
        pkg.kv_append(self.cache, k, v, p.slots)
        o = torch.zeros_like(x)
        pkg.kv_attention(q, self.cache, self.table, p.lens, cu=p.cu, out=o.view(rows, self.heads, self.d))
        y = x + pkg.linear(o, self.wo)
        last = (p.cu[1:] - 1).clamp(min=0)
        logits = pkg.linear(y[last.long()], self.lm)
        token = pkg.sample(logits, u, temperature=0.9, top_k=40, top_p=0.95)
        self.lens.copy_(p.lens)
        self.count.copy_(p.free_count)
        return dict(token=token, logits=logits, attended=o, q=q, slots=p.slots, cu=p.cu, positions=p.positions)


@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
def test_serving_loop(pkg, dev, dtype):
    """Prompts of three lengths, then tokens one at a time, one request ended
    and another begun in its place: attention against the 64-bit form over what
    the cache holds, tokens against the 64-bit sampling of the logits."""
    s, g = Server(pkg, dev, dtype, 5), gen(99)
    prompts = [19, 1, 40]
    new = list(prompts)
    token = None
    for step in range(30):
        rows = sum(max(n, 0) for n in new) + 2  # (two rows of padding)
        if step in (0, 12):
            ids = torch.randint(0, 200, (rows,), generator=g).to(dev)
        else:
            ids = torch.cat([token[[r for r, n in enumerate(new) if n > 0]], torch.zeros(2, dtype=torch.int64, device=dev)])
        u = torch.rand(3, generator=g)
        out = s.step(ids, ints(dev, *new), u.to(dev), rows)
        token = out["token"].clamp(min=0)
        live = [r for r, n in enumerate(new) if n > 0]
        cu, lens = out["cu"].tolist(), s.lens.tolist()
        assert out["slots"].tolist()[cu[-1]:] == [-1, -1] and not out["attended"][cu[-1]:].any()
        # what the cache holds, in 64 bits
        cells = torch.arange(s.blocks * s.block, device=dev)
        k, v = ((c.cpu().double() * sc.cpu().double().view(s.blocks, s.kv, 1, 1)) for c, sc in
                ((s.cache.k, s.cache.k_scale), (s.cache.v.transpose(-1, -2).reshape(s.cache.k.shape), s.cache.v_scale)))
        k, v = (t.transpose(1, 2).reshape(len(cells), s.kv, s.d) for t in (k, v))
        want, room = attention64(out["q"].cpu(), k, v, s.block, s.table.cpu(), lens, cu, s.d ** -0.5, s.blocks)
        got = out["attended"].view(want.shape).cpu().double()
        off = (got - want).abs() - HALF[dtype] * want.abs() - room
        assert off[:cu[-1]].max() <= 2.0 ** -25, step
        for r in live:
            assert out["token"][r].item() == sample64(out["logits"][r].cpu().double().numpy(), u[r].item(),
                                                      float(np.float32(0.9)), 40, float(np.float32(0.95))), (step, r)
        new = [1, 1, 1]
        if step == 10:
            new = [1, -1, 1]  # the second ends
        if step == 11:
            new = [1, 37, 1]  # another takes its place
    assert s.lens.tolist() == [19 + 29, 37 + 17, 40 + 29]


def test_serving_loop_in_a_graph(pkg, dev):
    """The step captured once and replayed, with eager work and
    synchronisations between: the same tokens, lengths and cache as eager steps."""
    eager, graphed = Server(pkg, dev, torch.float16, 6), Server(pkg, dev, torch.float16, 6)
    prompt, new, u0 = torch.randint(0, 200, (24,), generator=gen(1)).to(dev), ints(dev, 9, 8, 7), torch.full((3,), 0.4, device=dev)
    first = [s.step(prompt, new, u0, 24)["token"] for s in (eager, graphed)]
    assert torch.equal(*first)
    ids, one, u = first[1].clone(), ints(dev, 1, 1, 1), torch.zeros(3, device=dev)
    saved = [t.clone() for t in (graphed.lens, graphed.count, graphed.cache.k, graphed.cache.v, graphed.cache.k_scale,
                                 graphed.cache.v_scale)]
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        graphed.step(ids, one, u, 3)  # warm up
    torch.cuda.current_stream().wait_stream(side)
    for t, w in zip((graphed.lens, graphed.count, graphed.cache.k, graphed.cache.v, graphed.cache.k_scale,
                     graphed.cache.v_scale), saved):
        t.copy_(w)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = graphed.step(ids, one, u, 3)
    token = first[0]
    for i in range(20):
        r = torch.rand(3, generator=gen(i)).to(dev)
        want = eager.step(token, one, r, 3)
        token = want["token"]
        u.copy_(r)
        graph.replay()
        torch.cuda.synchronize()
        for n in ("token", "logits", "attended", "slots"):
            assert torch.equal(out[n], want[n]), (i, n)
        ids.copy_(out["token"])
    assert torch.equal(eager.lens, graphed.lens) and torch.equal(eager.cache.k, graphed.cache.k)
    assert torch.equal(eager.cache.v, graphed.cache.v) and eager.lens.tolist() == [29, 28, 27]


def test_two_captured_attentions_share_no_counters(pkg, dev):
    """Two graphs whose calls share their keys out, replayed in turn and at once."""
    cache, _ = filled(pkg, dev, 64, 2, 64, 64, 107)
    table, lens = torch.arange(64, dtype=torch.int32, device=dev).view(1, 64), ints(dev, 4000)
    qs = [normal((1, 8, 64), 60 + i).to(dev) for i in range(2)]
    want = [pkg.kv_attention(q, cache, table, lens) for q in qs]
    graphs, outs = [], []
    for q in qs:
        graphs.append(torch.cuda.CUDAGraph())
        with torch.cuda.graph(graphs[-1]):
            outs.append(pkg.kv_attention(q, cache, table, lens))
    streams = [torch.cuda.Stream() for _ in qs]
    for i in range(6):
        for o in outs:
            o.fill_(math.nan)
        torch.cuda.synchronize()
        for g, s in zip(graphs, streams):
            with torch.cuda.stream(s if i % 2 else streams[0]):
                g.replay()
        torch.cuda.synchronize()
        assert torch.equal(pkg.kv_attention(qs[0], cache, table, lens), want[0])
        assert all(torch.equal(o, w) for o, w in zip(outs, want)), i
