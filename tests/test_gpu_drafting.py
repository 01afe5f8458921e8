"""The serving operators together, as a program that drafts tokens uses them:
block tables, rotation with norms in place, a 4-bit cache, attention over it,
verification, and lengths that go back to what was accepted."""
import math

import numpy as np
import pytest
import torch

from gpu_util import gen, normal
from kv4_util import numbers, quantised
from test_gpu_kv4 import attention64
from test_gpu_rope import check as check_rope
from test_gpu_verify import verify64

pytestmark = pytest.mark.gpu

HALF = {torch.float16: 2.0 ** -11, torch.bfloat16: 2.0 ** -8}


class Drafter:
    """A one-layer decoder with norms of queries and keys, positions, and a
    4-bit cache; a step takes each request's accepted token and its drafts."""

    def __init__(self, pkg, dev, dtype, seed, bits=4):
        self.pkg, self.dev, self.heads, self.kv, self.d, self.block, self.blocks, self.R = pkg, dev, 4, 2, 64, 16, 30, 3
        H = self.heads * self.d
        n = lambda *sh, i, std=1.0: normal(sh, seed + i, std, dtype=dtype).to(dev)  # noqa: E731
        self.embed, self.wqkv = n(200, H, i=0), n((self.heads + 2 * self.kv) * self.d, H, i=1, std=0.06)
        self.wo, self.lm = n(H, H, i=2, std=0.06), n(200, H, i=3, std=0.15)
        self.gq, self.gk = n(self.d, i=4, std=0.1) + 1, n(self.d, i=5, std=0.1) + 1
        self.freq, _ = pkg.rope_frequencies(self.d, 1e4, device=dev)
        self.cache = (pkg.KVCache4 if bits == 4 else pkg.KVCache).empty(self.blocks, self.kv, self.d, self.block, device=dev)
        self.table = torch.full((self.R, 8), -1, dtype=torch.int32, device=dev)
        self.free = torch.arange(self.blocks, dtype=torch.int32, device=dev)
        self.count = torch.tensor([self.blocks], dtype=torch.int32, device=dev)
        self.lens = torch.zeros(self.R, dtype=torch.int32, device=dev)

    def step(self, ids, new, u, draw, probs, rows):
        pkg = self.pkg
        p = pkg.kv_plan(self.lens, new, self.table, self.free, self.count, block_size=self.block, tokens=rows)
        x = self.embed[ids]
        qkv = pkg.linear(x, self.wqkv).view(rows, -1, self.d)
        q, k, v = qkv.split([self.heads, self.kv, self.kv], 1)
        raw = qkv.clone()
        pkg.qk_rope(q, k, p.positions, self.freq, q_weight=self.gq, k_weight=self.gk, out=(q, k))
        pkg.kv_append(self.cache, k, v, p.slots)
        o = torch.zeros_like(x)
        pkg.kv_attention(q, self.cache, self.table, p.lens, cu=p.cu, out=o.view(rows, self.heads, self.d))
        logits = pkg.linear(x + pkg.linear(o, self.wo), self.lm)
        # row i's draft is the token that row i + 1 was given
        drafts = torch.cat([ids[1:], ids[:1]])
        got = pkg.verify(logits, drafts, u, draw, cu=p.cu, draft_probs=probs, temperature=0.9, top_k=40, top_p=0.95)
        # the rows past the accepted drafts leave the requests again, their blocks go back
        keep = torch.where(p.lens > self.lens, self.lens + got.counts, p.lens)
        self.lens.copy_(p.lens)
        self.count.copy_(p.free_count)
        pkg.kv_trim(self.lens, keep, self.table, self.free, self.count, block_size=self.block)
        return dict(tokens=got.tokens, counts=got.counts, logits=logits, attended=o, qkv=qkv, raw=raw, slots=p.slots, cu=p.cu,
                    positions=p.positions, drafts=drafts, lens=p.lens)


@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
def test_drafting_loop(pkg, dev, dtype):
    """Prompts of three lengths, each a row of drafts of its own, then one to
    four drafts a step: every operator of every step against its definition."""
    s, g = Drafter(pkg, dev, dtype, 5), gen(99)
    token, new = None, [19, 2, 40]
    for step in range(8):
        rows = sum(new) + 2  # (two rows of padding)
        ids = torch.randint(0, 200, (rows,), generator=g)
        if token is not None:
            at = np.cumsum([0] + new)
            for r in range(3):
                ids[at[r]] = token[r]
        probs = (torch.randn((rows, 200), generator=g) * 1.5).softmax(-1).to(torch.float32) if step % 2 else None
        u, draw = torch.rand(rows, generator=g) * 0.2, torch.rand(3, generator=g)
        before, cells = s.lens.tolist(), {n: numbers(s.cache, n) for n in ("k", "v")}
        out = s.step(ids.to(dev), torch.tensor(new, dtype=torch.int32, device=dev), u.to(dev), draw.to(dev),
                     None if probs is None else probs.to(dev), rows)
        cu, slots = out["cu"].tolist(), out["slots"].tolist()
        assert slots[cu[-1]:] == [-1, -1] and out["lens"].tolist() == [b + n for b, n in zip(before, new)]
        pos = out["positions"]
        assert pos.tolist()[:cu[-1]] == [b + i for b, n in zip(before, new) for i in range(n)]
        H, K = s.heads, s.kv
        for a, b, w in ((0, H, s.gq), (H, H + K, s.gk)):
            check_rope(out["qkv"][:cu[-1], a:b], out["raw"][:cu[-1], a:b], pos[:cu[-1]], s.freq, weight=w)
        for t, slot in enumerate(slots[:cu[-1]]):
            cells["k"][slot] = quantised(out["qkv"][t, H:H + K])[2]
            cells["v"][slot] = quantised(out["qkv"][t, H + K:])[2]
        assert all(torch.equal(numbers(s.cache, n), cells[n]) for n in ("k", "v")), step
        want, room = attention64(out["qkv"][:, :H].cpu(), cells["k"], cells["v"], s.block, s.table.cpu(), out["lens"].tolist(), cu,
                                 s.d ** -0.5, s.blocks)
        got = out["attended"].view(want.shape).cpu().double()
        off = (got - want).abs() - HALF[dtype] * want.abs() - room * (1 + HALF[dtype])
        assert off[:cu[-1]].max() <= 2.0 ** -25, step
        T, P = [float(np.float32(0.9))] * 3, [float(np.float32(0.95))] * 3
        tokens, counts, near = verify64(out["logits"].cpu().double().numpy(), out["drafts"].tolist(), u.tolist(), draw.tolist(), cu,
                                        None if probs is None else probs.double().numpy(), [T, [40] * 3, P, [0.0] * 3])
        assert near == 0 and out["tokens"].tolist() == tokens and out["counts"].tolist() == counts, step
        assert s.lens.tolist() == [b + n for b, n in zip(before, counts)]
        # every block is a request's or free
        held = [s.table[r, :-(-n // s.block)].tolist() for r, n in enumerate(s.lens.tolist())]
        assert sorted(sum(held, []) + s.free[:int(s.count)].tolist()) == list(range(s.blocks))
        token = [tokens[cu[r] + counts[r] - 1] for r in range(3)]
        new = [1 + int(torch.randint(0, 5, (1,), generator=g)) for _ in range(3)]


@pytest.mark.parametrize("requests, width, block, seed", [(1, 4, 16, 0), (70, 5, 32, 1), (2100, 3, 16, 2), (5000, 2, 64, 3)])
def test_trim(pkg, dev, requests, width, block, seed):
    """Lengths taken back by some, all, none and more than there are; a stack short of room."""
    rng = np.random.default_rng(seed)
    i32 = lambda v: torch.tensor(v, dtype=torch.int32, device=dev)  # noqa: E731
    lens = rng.integers(0, width * block + 1, requests)
    keep = np.where(rng.random(requests) < 0.3, lens, rng.integers(-3, width * block + 9, requests))
    table = rng.permutation(requests * (width + 2)).reshape(requests, width + 2)
    held = lambda n: -(-n // block)  # noqa: E731
    want, stack = lens.copy(), [900001, 900002]
    for r in range(requests):
        if 0 <= keep[r] < lens[r]:
            stack += table[r, held(keep[r]):held(lens[r])].tolist()
            want[r] = keep[r]
    for room in (len(stack) + 5, max(len(stack) - 1, 2)):
        a, free, count = i32(lens), torch.full((room,), -7, dtype=torch.int32, device=dev), i32([2])
        free[:2] = i32([900001, 900002])
        t = i32(table)[:, :width]
        pkg.kv_trim(a, i32(keep), t, free, count, block_size=block)
        assert a.tolist() == want.tolist() and count.tolist() == [min(len(stack), room)]
        assert free.tolist() == (stack + [-7] * 5)[:room] and torch.equal(t, i32(table)[:, :width])


def test_trim_refuses(pkg, dev):
    i32 = lambda *v: torch.tensor(v, dtype=torch.int32, device=dev)  # noqa: E731
    lens, table, free, count = i32(5, 6), torch.zeros((2, 3), dtype=torch.int32, device=dev), i32(1, 2, 3), i32(1)
    bad = [
        ("lens", lambda: pkg.kv_trim(lens.long(), lens, table, free, count, block_size=16)),
        ("keep", lambda: pkg.kv_trim(lens, lens[:1].clone(), table, free, count, block_size=16)),
        ("share", lambda: pkg.kv_trim(lens, lens, table, free, count, block_size=16)),
        ("share", lambda: pkg.kv_trim(lens, i32(1, 1), table, free, free[:1], block_size=16)),
        ("block_table", lambda: pkg.kv_trim(lens, i32(1, 1), table[:1], free, count, block_size=16)),
        ("free_blocks", lambda: pkg.kv_trim(lens, i32(1, 1), table, free[::2], count, block_size=16)),
        ("free_count", lambda: pkg.kv_trim(lens, i32(1, 1), table, free, i32(1, 2), block_size=16)),
        ("block_size", lambda: pkg.kv_trim(lens, i32(1, 1), table, free, count, block_size=17)),
        ("GPU", lambda: pkg.kv_trim(lens, i32(1, 1), table.cpu(), free, count, block_size=16)),
    ]
    for i, (msg, call) in enumerate(bad):
        with pytest.raises(pkg.HxmiError, match=msg):
            call()
            pytest.fail(f"call {i} ({msg}) was taken")
    none = i32()
    pkg.kv_trim(none, i32(), table[:0], free, count, block_size=16)
    assert lens.tolist() == [5, 6] and free.tolist() == [1, 2, 3] and count.tolist() == [1]


@pytest.mark.parametrize("bits", [4, 8])
def test_drafting_step_in_a_graph(pkg, dev, bits):
    """The step captured once and replayed, with eager work between: as eager steps."""
    pair = [Drafter(pkg, dev, torch.float16, 6, bits) for _ in range(2)]
    eager, graphed = pair
    g = gen(3)
    prompt = torch.randint(0, 200, (24,), generator=g).to(dev)
    first = torch.tensor([9, 8, 7], dtype=torch.int32, device=dev)
    u, draw = torch.zeros(24, device=dev), torch.full((3,), 0.4, device=dev)
    probs = (torch.randn((24, 200), generator=g)).softmax(-1).to(dev)
    for s in pair:
        s.step(prompt, first, u, draw, probs, 24)
    ids, new, v = prompt[:9].clone(), torch.tensor([3, 3, 3], dtype=torch.int32, device=dev), u[:9].clone()
    q = probs[:9].clone()
    held = [t.clone() for t in (graphed.lens, graphed.count, graphed.table, graphed.free, graphed.cache.k, graphed.cache.v,
                                graphed.cache.k_scale, graphed.cache.v_scale)]
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        graphed.step(ids, new, v, draw, q, 9)  # warm up
    torch.cuda.current_stream().wait_stream(side)
    for t, w in zip((graphed.lens, graphed.count, graphed.table, graphed.free, graphed.cache.k, graphed.cache.v, graphed.cache.k_scale,
                     graphed.cache.v_scale), held):
        t.copy_(w)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = graphed.step(ids, new, v, draw, q, 9)
    for i in range(8):
        ids.copy_(torch.randint(0, 200, (9,), generator=g))
        v.copy_(torch.rand(9, generator=g) * 0.3)
        draw.copy_(torch.rand(3, generator=g))
        q.copy_((torch.randn((9, 200), generator=g)).softmax(-1))
        want = eager.step(ids, new, v, draw, q, 9)
        graph.replay()
        torch.cuda.synchronize()
        for n in ("tokens", "counts", "logits", "attended", "slots", "qkv"):
            assert torch.equal(out[n], want[n]), (i, n)
    assert torch.equal(eager.lens, graphed.lens) and torch.equal(eager.cache.k, graphed.cache.k)
    assert torch.equal(eager.cache.v, graphed.cache.v) and not math.isnan(float(out["logits"].float().sum()))
