"""The 4-bit key/value cache on the GPU: rows written and read back, and
attention over it, each against a plain implementation in 64 bits, at the sizes
and masks where they can go wrong."""
import math

import numpy as np
import pytest
import torch

from gpu_util import gen, normal
from kv4_util import SCALES, TOP, numbers, quantised

pytestmark = pytest.mark.gpu

HALF = {torch.float16: 2.0 ** -11, torch.bfloat16: 2.0 ** -8}  # half a step of the type, relative


def ints(dev, *v, dtype=torch.int32):
    return torch.tensor(v, dtype=dtype, device=dev)


# ---- writing and reading -------------------------------------------------------------

APPENDS = [(2, 64, 16, torch.float16), (1, 128, 64, torch.bfloat16), (3, 40, 32, torch.float16), (2, 8, 16, torch.bfloat16),
           (1, 96, 128, torch.float16), (5, 120, 256, torch.bfloat16), (2, 80, 32, torch.float16)]


class Held:
    """What a cache should hold."""

    def __init__(self, cells, heads, d):
        self.k, self.v = (torch.zeros((cells, heads, d), dtype=torch.float64) for _ in range(2))

    def append(self, k, v, slots):
        for t, s in enumerate(slots):
            if 0 <= s < self.k.shape[0]:
                self.k[s], self.v[s] = quantised(k[t])[2], quantised(v[t])[2]

    def check(self, pkg, cache, dtype, name=""):
        k, v = numbers(cache, "k"), numbers(cache, "v")
        assert torch.equal(k, self.k) and torch.equal(v, self.v), name
        every = torch.arange(self.k.shape[0], device=cache.k.device)
        for got, want in zip(pkg.kv_read(cache, every, dtype), (self.k, self.v)):
            assert got.dtype == dtype and torch.equal(got.cpu().double(), want), name


@pytest.mark.parametrize("heads, d, block, dtype", APPENDS)
def test_append_in_pieces_of_every_length(pkg, dev, heads, d, block, dtype):
    """Runs of 1 to 70 rows that begin and end anywhere in blocks, over blocks in any order."""
    blocks, g = 9, gen(7)
    cache, held = pkg.KVCache4.empty(blocks, heads, d, block, device=dev), Held(9 * block, heads, d)
    order = torch.randperm(blocks, generator=g).tolist()
    at = 0
    for n in [1, 1, 2, 15, 1, 16, 17, 3, 31, 33, 40, 64, 70, 5] * 3:
        if at + n > blocks * block:
            at = 0
        slots = [order[p // block] * block + p % block for p in range(at, at + n)]
        at += n
        kv = (torch.randn((n, 2 * heads, d), generator=g) * torch.exp2(torch.randint(-9, 9, (n, 2 * heads, 1), generator=g))).to(dtype)
        k, v = kv[:, :heads], kv[:, heads:]
        x = kv.to(dev)
        pkg.kv_append(cache, x[:, :heads], x[:, heads:], ints(dev, *slots, dtype=torch.int64))
        held.append(k, v, slots)
    held.check(pkg, cache, dtype)
    assert not cache.k[..., d // 2:].any() and not cache.v[..., d:, :].any()


@pytest.mark.parametrize("tokens, heads, d, block, dtype", [
    (300, 4, 64, 16, torch.float16), (2000, 1, 128, 32, torch.bfloat16), (9000, 2, 64, 64, torch.float16), (1, 1, 32, 16, torch.float16),
])
def test_append_of_many_requests(pkg, dev, tokens, heads, d, block, dtype):
    """Rows of many requests in one call: single tokens, prompts, rows without a place; nothing else changes."""
    g = gen(17)
    blocks = tokens // block * 2 + 40
    cache = pkg.KVCache4.empty(blocks, heads, d, block, device=dev)
    for t in (cache.k, cache.v, cache.k_scale, cache.v_scale):
        t.copy_(torch.randint(0, 200, t.shape, generator=g))
    held = Held(blocks * block, heads, d)
    held.k, held.v = numbers(cache, "k"), numbers(cache, "v")
    free, slots = torch.randperm(blocks, generator=g).tolist(), []
    while len(slots) < tokens:
        n = int(torch.randint(1, 90, (1,), generator=g)) if torch.rand(1, generator=g) < 0.3 else 1
        first = int(torch.randint(0, block, (1,), generator=g))
        pages = [free.pop() for _ in range(-(-(first + n) // block))] if len(free) > 20 else []
        if not pages or torch.rand(1, generator=g) < 0.1:
            slots += [[-1, blocks * block, 1 << 40][n % 3]] * n
        else:
            slots += [pages[p // block] * block + p % block for p in range(first, first + n)]
    slots = slots[:tokens]
    k, v = normal((tokens, heads, d), 18, 3.0, dtype=dtype), normal((tokens, heads, d), 19, 0.01, dtype=dtype)
    pkg.kv_append(cache, k.to(dev), v.to(dev), ints(dev, *slots, dtype=torch.int64))
    held.append(k, v, slots)
    held.check(pkg, cache, dtype)
    some = ints(dev, *slots, -5, 3, 2, 1, 1, 1, blocks * block, dtype=torch.int64)
    for got, want in zip(pkg.kv_read(cache, some, dtype), (held.k, held.v)):
        want = torch.cat([want, torch.zeros_like(want[:1])])[[s if 0 <= s < blocks * block else -1 for s in some.tolist()]]
        assert torch.equal(got.cpu().double(), want)


@pytest.mark.parametrize("heads, d, block", [(2, 64, 16), (1, 128, 64), (3, 40, 32)])
def test_append_in_any_order(pkg, dev, heads, d, block):
    """Slots with gaps, backwards and shuffled, many of them of the same pieces in one call."""
    g, cells = gen(27), 6 * block
    for n, order in ((cells, "shuffled"), (cells // 2, "every other"), (cells, "backwards"), (7, "few")):
        slots = {"shuffled": torch.randperm(cells, generator=g), "every other": torch.arange(0, cells, 2),
                 "backwards": torch.arange(cells).flip(0), "few": torch.tensor([3, 1, 14, 15, 0, 9, 40])}[order]
        cache, held = pkg.KVCache4.empty(6, heads, d, block, device=dev), Held(cells, heads, d)
        for step in range(2):  # into an empty cache, then over what is there
            k, v = torch.randn((2, n, heads, d), generator=g).half()
            pkg.kv_append(cache, k.to(dev), v.to(dev), slots.to(dev))
            held.append(k, v, slots.tolist())
            held.check(pkg, cache, torch.float16, (order, step))


@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
def test_append_of_every_border(pkg, dev, dtype):
    """Rows whose quotients are every magnitude, every border of two and the
    16-bit numbers beside them, under every scale; the largest and smallest
    values, infinities and NaN."""
    top = torch.finfo(dtype).max
    edge = torch.tensor([0, .25, .5, .75, 1, 1.25, 1.5, 1.75, 2, 2.5, 3, 3.5, 4, 5, 6], dtype=torch.float64)
    rows = []
    for s in SCALES[1:227]:
        e = (edge * s).to(dtype)
        bits = e.view(torch.int16)
        near = torch.cat([e, (bits + 1).view(dtype), (bits - 1).clamp(min=0).view(dtype)])[:31].clone()
        near[1::2] *= -1
        rows.append(torch.cat([(6 * s).to(dtype).view(1), near.clamp(-(6 * s).to(dtype), (6 * s).to(dtype))]))
        over = ((6 * s).to(dtype).view(torch.int16) + 1).view(dtype).view(1)  # one more than a scale holds
        rows.append(torch.cat([over, near.clamp(-over, over)]))
    x = torch.stack(rows)
    more = torch.zeros((12, 32), dtype=dtype)
    more[0, 3], more[1, :2], more[2, 5], more[3, 1] = math.nan, torch.tensor([math.inf, 1.0]), -math.inf, top
    more[4, 2:4], more[5] = torch.tensor([2.0 ** -18, -2.0 ** -19]), 2.0 ** -19
    more[6, 0], more[7, 0], more[8, 0] = 2.0 ** -24, TOP, -TOP
    more[9, :3], more[10, :2] = torch.tensor([60000.0, -100.0, math.nan]), torch.tensor([-0.0, 2.0 ** -17 * 6])
    x = torch.cat([x, more, -more])[:, None]  # [rows, 1 head, 32]
    n = x.shape[0]
    cache = pkg.KVCache4.empty(n // 16 + 1, 1, 32, 16, device=dev)
    slots = torch.arange(n, device=dev)
    pkg.kv_append(cache, x.to(dev), x.flip(-1).contiguous().to(dev), slots)
    code, byte, value = quantised(x)
    for name, flip in (("k", False), ("v", True)):
        got = numbers(cache, name)[:n]
        want = value.flip(-1) if flip else value
        assert torch.equal(got, want), (name, (got != want).nonzero()[:3], x[(got != want).nonzero()[0, 0]])
        assert torch.equal(getattr(cache, name + "_scale").cpu().transpose(2, 3).flatten(0, 2)[:n], byte[:, 0].to(torch.uint8))
    # within half the distance of the magnitudes around it: 1/6 of the value from 4 to 6, 1/4 of a scale at least
    finite = torch.isfinite(x) & (x.abs().double() <= TOP)
    room = torch.maximum(x.double().abs() / 5, SCALES[byte].repeat_interleave(32, -1) / 4)
    assert ((value - x.double()).abs() <= room)[finite].all()
    for r, dt in ((torch.float16, 0), (torch.bfloat16, 1)):
        assert torch.equal(pkg.kv_read(cache, slots, r)[0].cpu().double(), value)


def test_append_and_read_take_any_view(pkg, dev):
    """Rows of a projection at any offset, other strides, slots of other strides."""
    heads, d, n = 2, 64, 21
    slots = ints(dev, *range(5, 5 + n), dtype=torch.int64)
    buf = normal((n, 1 + 2 * heads * d), 31).to(dev)
    kv = buf[:, 1:].view(n, 2 * heads, d)
    want = pkg.KVCache4.empty(3, heads, d, 16, device=dev)
    pkg.kv_append(want, kv[:, :heads].contiguous(), kv[:, heads:].contiguous(), slots)
    for k, v in ((kv[:, :heads], kv[:, heads:]), (kv[:, :heads].transpose(0, 1).contiguous().transpose(0, 1), kv[:, heads:]),
                 (kv[:, :heads].transpose(1, 2).contiguous().transpose(1, 2), kv[:, heads:])):
        c = pkg.KVCache4.empty(3, heads, d, 16, device=dev)
        pkg.kv_append(c, k, v, slots.repeat_interleave(2)[::2])
        assert all(torch.equal(getattr(c, t), getattr(want, t)) for t in ("k", "v", "k_scale", "v_scale"))
    a, b = pkg.kv_read(want, slots), pkg.kv_read(want, slots.repeat_interleave(2)[::2])
    assert all(torch.equal(x, y) for x, y in zip(a, b))
    one = pkg.KVCache4.empty(3, heads, d, 16, device=dev)
    pkg.kv_append(one, kv[:1, :heads].expand(n, -1, -1), kv[:1, heads:].expand(n, -1, -1), slots)  # one row for all
    r = pkg.kv_read(one, slots)
    assert all(torch.equal(t, t[:1].expand_as(t)) for t in r) and torch.equal(r[0][0], a[0][0])


# ---- attention -----------------------------------------------------------------------

def filled(pkg, dev, blocks, heads, d, block, seed, junk=True):
    """A cache of random numbers, and its values [blocks * block, heads, d] in 64 bits."""
    g = gen(seed)
    cache = pkg.KVCache4.empty(blocks, heads, d, block, device=dev)
    x = [torch.randn((blocks * block, heads, d), generator=g) * (0.3 + torch.rand((blocks * block, heads, 1), generator=g))
         for _ in range(2)]
    pkg.kv_append(cache, *(t.half().to(dev) for t in x), torch.arange(blocks * block, device=dev))
    return cache, [numbers(cache, n) for n in ("k", "v")]


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
            if not len(cells):
                continue
            kh, vh = (x[cells].transpose(0, 1).repeat_interleave(group, 0) for x in (k, v))
            s = (q[t].double()[:, None] @ kh.transpose(1, 2))[:, 0] * scale
            w = s.softmax(-1)
            out[t] = (w[:, None] @ vh)[:, 0]
            # a weight is off by half an fp16 step of itself (2^-12), a score by up to 128 fp32 roundings of
            # its terms (products of fp16 numbers are exact; 2^-24 each of at most the sum of magnitudes) and
            # one of itself, a weight below fp16's normal range by 2^-32 of the largest (kept above 2^7)
            size = (q[t].double().abs()[:, None] @ kh.abs().transpose(1, 2))[:, 0] * scale
            by = 2.0 ** -12 + 130 * 2.0 ** -24 * size.amax(-1, keepdim=True) + 2.0 ** -20
            # (twice: the sum of the weights is off by as much)
            room[t] = 2 * by * (w[:, None] @ vh.abs())[:, 0] + len(cells) * 2.0 ** -31 * (w.amax(-1)[:, None] * vh.abs().amax(1))
    return out, room


def check_attention(got, q, k, v, block, table, lens, cu, scale, blocks, name=""):
    want, room = attention64(q.cpu(), k, v, block, table.cpu(), lens.tolist(), cu, scale, blocks)
    got = got.cpu().double()
    live = ~torch.isnan(want)
    off = (got - want).abs() - HALF[q.dtype] * want.abs() - room * (1 + HALF[q.dtype])
    assert live.any() and off[live].max() <= 2.0 ** -25, (name, float(off[live].max()))


LENS = [0, 1, 2, 15, 16, 17, 31, 63, 64, 65, 100, 127, 128, 129, 255, 257, 300, 511, 513, 600]

SHAPES = [  # heads, kv heads, head dim, block, dtype
    (8, 2, 64, 16, torch.float16), (14, 2, 64, 64, torch.bfloat16), (4, 4, 128, 32, torch.float16),
    (32, 4, 128, 64, torch.bfloat16), (3, 1, 40, 128, torch.float16), (6, 2, 80, 16, torch.bfloat16),
    (40, 1, 96, 256, torch.float16), (1, 1, 8, 16, torch.bfloat16), (5, 5, 120, 32, torch.float16),
    (33, 1, 72, 64, torch.bfloat16), (4, 1, 32, 16, torch.float16),
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
    """Prompts: requests that end inside a tile, an empty one, a prompt without
    a context, a context that ends inside a page; rows of no request."""
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
    assert torch.equal(pkg.kv_attention(q, cache, table, lens, out=shifted), want)
    buf[:, 1:1 + heads * d].view(3, heads, d).copy_(qc)
    assert torch.equal(pkg.kv_attention(q, cache, table, lens, out=q), want)
    with pytest.raises(pkg.HxmiError, match="share"):
        pkg.kv_attention(qc, cache, table, lens, out=torch.empty((1, heads, d), dtype=q.dtype, device=dev).expand(3, -1, -1))


@pytest.mark.parametrize("rows", [1, 130])  # tiles of 16 rows and of 128
def test_attention_leaves_out_pages_outside_the_cache(pkg, dev, rows):
    """Entries of no block, in the middle, at the end, everywhere; lengths past
    the table; bytes that are no numbers where no row looks, and where only
    some rows of a tile do."""
    heads, kv_heads, d, block, blocks = 32, 2, 64, 16, 24
    cache, (k, v) = filled(pkg, dev, blocks, kv_heads, d, block, 47)
    table = ints(dev, 3, -1, 5, 2 ** 31 - 1, 1, 1, 2, 3, 4, 9, -5, 24, -1, -1, -2 ** 31, 0, 7, 7, 7, 7).view(4, 5)
    table = torch.cat([table] * 4, 1)
    lens, cu = ints(dev, 300, 230, 250, 900), [rows * i for i in range(5)]
    q = normal((4 * rows, heads, d), 49, 1.5).to(dev)
    got = pkg.kv_attention(q, cache, table, lens, cu=ints(dev, *cu))
    check_attention(got, q, k, v, block, table, lens, cu, d ** -0.5, blocks)
    # blocks 22 and 23 hold no numbers: one lies behind all keys, of the other the last row alone sees the first token
    for b in (22, 23):
        cache.k_scale[b], cache.v_scale[b], cache.k[b], cache.v[b] = 255, 250, 255, 255
    for name in ("v_scale", "k_scale"):
        table = (torch.arange(20, dtype=torch.int32) % 20).view(1, 20).to(dev)
        table[0, 15], table[0, 16] = 23, 22
        lens = ints(dev, 241)
        q = normal((rows + 1, heads, d), 50, 1.5).to(dev)
        got = pkg.kv_attention(q, cache, table, lens, cu=ints(dev, 0, rows + 1))
        assert torch.isfinite(got[:rows]).all() and torch.isnan(got[rows]).all()
        check_attention(got[:rows], q[:rows], k, v, block, table, ints(dev, 240), [0, rows], d ** -0.5, blocks)
        # a page that is not there, block 0's bytes no numbers
        cache.k_scale[0], cache.v_scale[0] = 255, 255
        table[0, 2] = -1
        table[0, 0] = 1
        got = pkg.kv_attention(q[:rows], cache, table, ints(dev, 240), cu=ints(dev, 0, rows))
        check_attention(got, q[:rows], k, v, block, table, ints(dev, 240), [0, rows], d ** -0.5, blocks)
        if name == "v_scale":  # then with keys that are numbers and values that are none
            for b in (22, 23):
                cache.k_scale[b], cache.k[b] = 100, 0
            cache.k_scale[0], cache.v_scale[0] = 100, 100
            k, v = numbers(cache, "k"), numbers(cache, "v")


@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
def test_attention_at_the_ends_of_its_range(pkg, dev, dtype):
    """Keys and values from 2^-17 to 61440, scores that leave one key, that
    leave all alike, that all lie far below zero; a key 2^20 above many others."""
    heads, kv_heads, d, block, blocks = 16, 1, 64, 16, 24
    n = blocks * block - 3
    g = gen(57)
    x = torch.randn((2, blocks * block, 1, d), generator=g)
    x[0] *= torch.exp2(torch.arange(blocks * block) % 9 - 4.0)[:, None, None]
    x[1] *= torch.exp2(torch.arange(blocks * block) % 27 - 14.0)[:, None, None]
    cache = pkg.KVCache4.empty(blocks, kv_heads, d, block, device=dev)
    pkg.kv_append(cache, *x.half().to(dev), torch.arange(blocks * block, device=dev))
    k, v = numbers(cache, "k"), numbers(cache, "v")
    table, lens = torch.arange(blocks, dtype=torch.int32, device=dev).view(1, blocks), ints(dev, n)
    for std, scale in ((1.0, 0.125), (3.0, 1.0), (2.0 ** -12, 0.125), (1.0, 2.0 ** -30), (30.0, 0.125)):
        q = normal((1, heads, d), 58, std, dtype=dtype).to(dev)
        got = pkg.kv_attention(q, cache, table, lens, scale=scale)
        check_attention(got, q, k, v, block, table, lens, [0, 1], scale, blocks, (std, scale))
    if dtype == torch.bfloat16:  # queries that fp16 does not hold
        for by in (2.0 ** 60, 2.0 ** -60):
            q = (normal((1, heads, d), 59).double() * by).to(dtype).to(dev)
            got = pkg.kv_attention(q, cache, table, lens, scale=0.125 / by)
            check_attention(got, q, k, v, block, table, lens, [0, 1], 0.125 / by, blocks, by)
    # one value of 0 under a weight far above thousands of others, which are all that is left
    y = torch.ones((2, blocks * block, 1, d), dtype=torch.float16)
    y[0] = 0
    y[0, 5], y[1, 5] = 3.0, 0.0
    pkg.kv_append(cache, *y.to(dev), torch.arange(blocks * block, device=dev))
    k, v = numbers(cache, "k"), numbers(cache, "v")
    q = torch.full((1, heads, d), 0.5, dtype=dtype, device=dev)
    got = pkg.kv_attention(q, cache, table, lens, scale=13.86 / 96)  # e^13.86 = 2^20
    check_attention(got, q, k, v, block, table, lens, [0, 1], 13.86 / 96, blocks)
    assert (got > 3e-4).all()


@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
@pytest.mark.parametrize("rows", [1, 130])  # tiles of 16 rows and of 128
def test_attention_of_scores_far_beyond(pkg, dev, dtype, rows):
    """Scores from 2^18 to 2^38, of either sign: the key far above the others is
    what remains, equal ones share, and rows with a few small scores beside such stay as they are."""
    heads, kv_heads, d, block, blocks = 32, 1, 64, 16, 16
    n, g = blocks * block, gen(87)
    table, lens = torch.arange(blocks, dtype=torch.int32, device=dev).view(1, blocks), ints(dev, n)
    v = torch.randn((n, 1, d), generator=g).half()
    for size in (96.0, 6144.0, 61440.0):
        for sign in (1, -1):
            k = torch.full((n, 1, d), sign * size)
            k[::3] *= 2 / 3 if sign > 0 else 1
            if sign < 0:
                k[1::3] *= 2 / 3
                k[2::3] *= 2 / 3
            best = torch.arange(n) % 3 != 0  # the (equal) largest scores' keys
            cache = pkg.KVCache4.empty(blocks, 1, d, block, device=dev)
            pkg.kv_append(cache, k.half().to(dev), v.to(dev), torch.arange(n, device=dev))
            vs = numbers(cache, "v")[:, 0]
            q = (torch.rand((rows, heads, d), generator=g) + 0.5) * torch.exp2(torch.arange(heads).float() % 16 - 1)[:, None]
            q[:, 5] = 2.0 ** -18  # (scores of about one beside the others' of 2^20 and more)
            q = q.to(dtype).to(dev)
            got = pkg.kv_attention(q, cache, table, lens, cu=ints(dev, 0, rows), scale=1.0).cpu().double()
            for i in (0, rows - 1):
                seen = torch.arange(n) <= n - rows + i
                want = vs[best & seen].mean(0)
                far = [h for h in range(heads) if h != 5]
                # the weights are equal and their sum exact to 2^-12; other scores lie 30 and more below
                assert ((got[i, far] - want).abs() <= HALF[dtype] * want.abs() + 2.0 ** -11 * vs.abs().mean(0) + 2.0 ** -25).all(), (size, sign, i)
            check_attention(got[:, 5:6].to(dtype), q[:, 5:6], numbers(cache, "k"), numbers(cache, "v"), block, table, lens,
                            [0, rows], 1.0, blocks, (size, sign))


def test_attention_past_32_bit_offsets(pkg, dev):
    """A cache of more than 4 GiB of codes each: pages at its start and end."""
    heads, kv_heads, d, block, blocks = 8, 8, 128, 64, 140000
    cache = pkg.KVCache4.empty(blocks, kv_heads, d, block, device=dev)
    assert cache.k.numel() > 1 << 32
    pages = [0, blocks - 1, 131072, 65536]
    n = 3 * block + 17
    slots = ints(dev, *(pages[p // block] * block + p % block for p in range(n)), dtype=torch.int64)
    x = normal((2, n, kv_heads, d), 67).to(dev)
    pkg.kv_append(cache, x[0], x[1], slots)
    k, v = pkg.kv_read(cache, slots)
    small = pkg.KVCache4.empty(4, kv_heads, d, block, device=dev)
    here = torch.arange(n, device=dev)
    pkg.kv_append(small, x[0], x[1], here)
    ks, vs = pkg.kv_read(small, here)
    assert torch.equal(k, ks) and torch.equal(v, vs) and k.abs().max() > 0
    for rows in (1, 130):
        q = normal((rows, heads, d), 68).to(dev)
        cu = ints(dev, 0, rows)
        got = pkg.kv_attention(q, cache, ints(dev, *pages).view(1, 4), ints(dev, n), cu=cu)
        want = pkg.kv_attention(q, small, ints(dev, 0, 1, 2, 3).view(1, 4), ints(dev, n), cu=cu)
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


# ---- entries -------------------------------------------------------------------------

def cache4_calls(pkg, dev):
    """(name, whether the native entry takes it, call giving tensors)"""
    block, heads, d = 16, 2, 64
    cache, _ = filled(pkg, dev, 20, heads, d, block, 87)
    q = normal((3, 8, d), 88).to(dev)
    x, slots = normal((4, heads, d), 89).to(dev), ints(dev, 5, 6, 40, -1, dtype=torch.int64)
    table, lens = torch.arange(12, dtype=torch.int32, device=dev).view(3, 4), ints(dev, 64, 3, 20)

    def appended(k, v, s):
        c = pkg.KVCache4(cache.k.clone(), cache.v.clone(), cache.k_scale.clone(), cache.v_scale.clone(), d)
        pkg.kv_append(c, k, v, s)
        return c.k, c.v, c.k_scale, c.v_scale

    return [
        ("append", True, lambda: appended(x, x, slots)),
        ("append strided values", False, lambda: appended(x, x.transpose(1, 2).contiguous().transpose(1, 2), slots)),
        ("read", True, lambda: pkg.kv_read(cache, slots, torch.bfloat16)),
        ("read strided slots", False, lambda: pkg.kv_read(cache, slots.repeat_interleave(2)[::2])),
        ("attention", True, lambda: (pkg.kv_attention(q, cache, table, lens),)),
        ("attention ragged out", True, lambda: (pkg.kv_attention(q, cache, table, lens, cu=ints(dev, 0, 2, 2, 3), scale=1,
                                                                 out=torch.zeros_like(q)),)),
        ("attention over q", False, lambda: (lambda c: (pkg.kv_attention(c, cache, table, lens, out=c),))(q.clone())),
    ]


def test_native_form_equals_python_form(pkg, dev, monkeypatch):
    getattr(pkg.hxmi._ops, "gemm")  # loads the module
    real, taken = pkg.hxmi._ops, []

    class Spy:
        def __getattr__(self, name):
            def f(*args):
                y = getattr(real, name)(*args)
                taken.append((name[:4], y is not None))
                return y
            return f

    for name, native, call in cache4_calls(pkg, dev):
        monkeypatch.setattr(pkg.hxmi, "_ops", Spy())
        taken.clear()
        got = call()
        assert taken[0] == ("kv4_", native), name
        monkeypatch.setattr(pkg.hxmi, "_ops", pkg.hxmi._PythonForms())
        want = call()
        assert len(got) == len(want) and all(torch.equal(a, b) for a, b in zip(got, want)), name


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


def test_python_forms_refuse(pkg, dev):
    c, hx = pkg.KVCache4.empty(4, 2, 64, 16, device=dev), pkg
    of = lambda k=c.k, v=c.v, ks=c.k_scale, vs=c.v_scale, d=64: hx.KVCache4(k, v, ks, vs, d)  # noqa: E731
    x, q = torch.zeros((3, 2, 64), dtype=torch.float16, device=dev), torch.zeros((3, 4, 64), dtype=torch.float16, device=dev)
    s, table, lens = ints(dev, 0, 1, 2, dtype=torch.int64), torch.zeros((3, 2), dtype=torch.int32, device=dev), ints(dev, 1, 1, 1)
    shifted = torch.zeros(c.k_scale.numel() + 4, dtype=torch.uint8, device=dev)[4:].view(c.k_scale.shape)
    bad = [
        ("dtype", lambda: hx.kv_append(c, x.float(), x.float(), s)), ("dtype", lambda: hx.kv_append(c, x, x.bfloat16(), s)),
        ("tokens, 2, 64", lambda: hx.kv_append(c, x[:, :1], x[:, :1], s)), ("slots", lambda: hx.kv_append(c, x, x, s.int())),
        ("KVCache4", lambda: hx.kv_append((c.k, c.v), x, x, s)), ("fp16 or bf16", lambda: hx.kv_read(c, s, torch.float32)),
        ("belong", lambda: hx.kv_read(of(v=c.v[:2]), s)), ("belong", lambda: hx.kv_read(of(d=32), s)),
        ("belong", lambda: hx.kv_read(of(ks=c.k_scale[:, :, :1]), s)), ("head_dim", lambda: hx.kv_read(of(d=60), s)),
        ("uint8", lambda: hx.kv_read(of(k=c.k.to(torch.int8)), s)), ("uint8", lambda: hx.kv_read(of(vs=c.v_scale.float()), s)),
        ("belong", lambda: hx.kv_read(hx.KVCache(c.k, c.v, c.k_scale, c.v_scale, 64), s)),  # (as a cache of 8 bits)
        ("contiguous", lambda: hx.kv_read(of(k=c.k.transpose(0, 1).contiguous().transpose(0, 1)), s)),
        ("16-byte", lambda: hx.kv_read(of(ks=shifted), s)),
        ("block_size", lambda: hx.kv_read(of(k=c.k[:, :, :8].contiguous()), s)),
        ("fp16 or bf16 q", lambda: hx.kv_attention(q.float(), c, table, lens)),
        ("multiple of 2 heads", lambda: hx.kv_attention(q[:, :3], c, table, lens)),
        ("block_table", lambda: hx.kv_attention(q, c, table.long(), lens)),
        ("one row", lambda: hx.kv_attention(q[:2], c, table, lens)), ("scale", lambda: hx.kv_attention(q, c, table, lens, scale=0)),
        ("out", lambda: hx.kv_attention(q, c, table, lens, out=q.float())),
        ("without blocks", lambda: hx.kv_attention(q, hx.KVCache4.empty(0, 2, 64, 16, device=dev), table, lens)),
        ("GPU", lambda: hx.kv_attention(q, c, table.cpu(), lens)),
    ]
    for i, (msg, call) in enumerate(bad):
        with pytest.raises(pkg.HxmiError, match=msg):
            call()
            pytest.fail(f"call {i} ({msg}) was taken")
