"""More operators of a serving step, as measurable cases.

Queries and keys are normalised by head and rotated to their positions
(``qk_rope``), keys and values are written to a cache of 4-bit numbers and read
back (``kv_append`` and ``kv_read`` on a ``KVCache4``), attention runs over it
(``kv_attention``), and drafted tokens are checked against the target's
distribution (``verify``).  ``listed()`` holds the cases, ``draw(rng)`` takes
one more from the same ranges, ``prepare`` makes what a program has in hand
before the call, ``run`` is one pass (in elementary torch operations, or with
``own`` through the library), ``work`` what the pass cannot do without and
``exact`` the same results from the definitions in 64 bits.
"""
import math
import random

import numpy as np
import torch

own = False

DTYPES = {"fp16": torch.float16, "bf16": torch.bfloat16, "fp32": torch.float32}
SIZES = {"fp16": 2, "bf16": 2, "fp32": 4}

# (query heads, key/value heads, head dim)
TINYLLAMA = dict(heads=32, kv_heads=4, dim=64)
QWEN = dict(heads=14, kv_heads=2, dim=64)
WIDE = dict(heads=32, kv_heads=8, dim=128)


def listed():
    return [
        # TinyLlama decoding for a single user: latency
        dict(name="rope_one_user", kind="rope", tokens=1, rotary=64, sections=1, at=1900, theta=1e4, norm="", pairs="halves",
             dtype="fp16", pick=1, **TINYLLAMA),
        # an image and its text: three axes (time, height, width) share the frequencies out
        dict(name="rope_axes_2350", kind="rope", tokens=2350, rotary=64, sections=3, at=4096, theta=1e6, norm="",
             pairs="halves", dtype="bf16", pick=2, **QWEN),
        # prompts of long contexts, norms of queries and keys in the same pass
        dict(name="rope_norm_16384", kind="rope", tokens=16384, rotary=128, sections=1, at=131072, theta=1e6, norm="own",
             pairs="halves", dtype="bf16", pick=3, **WIDE),
        # one token a request into half-filled blocks, read back with the rest of their blocks
        dict(name="append4_decode_128", kind="append", requests=128, new=1, at=3000, kv_heads=8, dim=128, block=64,
             dtype="bf16", pick=4),
        # prompt chunks of ragged lengths that begin and end inside blocks
        dict(name="append4_prompt_8192", kind="append", requests=5, new=2600, at=700, kv_heads=4, dim=64, block=32,
             dtype="fp16", pick=5),
        # TinyLlama decoding for a single user: latency
        dict(name="attend4_one_user", kind="attend", requests=1, context=1900, new=1, block=64, dtype="fp16", pick=6,
             **TINYLLAMA),
        # a full serving batch, contexts up to 8192
        dict(name="attend4_batch_64x8192", kind="attend", requests=64, context=8192, new=1, block=64, dtype="bf16",
             pick=7, **WIDE),
        # drafted tokens to be checked: one to five rows a request, small pages, 7 query heads a key head
        dict(name="attend4_drafts_37", kind="attend", requests=37, context=1500, new=5, block=16, dtype="bf16", pick=8,
             **QWEN),
        # prompt chunks over contexts that are in the cache already
        dict(name="attend4_chunks_3x1024", kind="attend", requests=3, context=8000, new=1024, block=64, dtype="fp16",
             pick=9, **WIDE),
        # one user's four drafted tokens, copied from the prompt: no distribution of their own
        dict(name="verify_one_32000", kind="verify", requests=1, rows=5, ragged=False, vocab=32000, dtype="fp16", drafter="",
             temperature=0.8, top_k=50, top_p=1.0, min_p=0.0, own_settings=False, pick=10),
        # a batch over Qwen2.5's vocabulary, nucleus sampling, a drafting model's distribution
        dict(name="verify_top_p_64", kind="verify", requests=64, rows=5, ragged=True, vocab=151936, dtype="bf16",
             drafter="fp32", temperature=0.9, top_k=0, top_p=0.95, min_p=0.0, own_settings=False, pick=11),
        # logits in 32 bits, every request with its own settings
        dict(name="verify_mixed_48", kind="verify", requests=48, rows=8, ragged=True, vocab=151936, dtype="fp32",
             drafter="bf16", temperature=1.0, top_k=400, top_p=0.9, min_p=0.02, own_settings=True, pick=12),
    ]


def _log_int(rng, lo, hi):
    return min(hi, max(lo, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def _draw(rng):
    kind = rng.choice(["rope", "rope", "append", "append", "attend", "attend", "attend", "verify", "verify"])
    pick = rng.randrange(1 << 30)
    shapes = [(32, 4, 64), (14, 2, 64), (32, 8, 128), (12, 12, 64), (16, 4, 128), (8, 1, 96), (4, 4, 80), (25, 5, 40)]
    if kind == "rope":
        heads, kv_heads, dim = rng.choice(shapes + [(8, 2, 256)])
        rotary = rng.choice([dim, dim, dim, dim // 2, dim // 8 * 2])
        return dict(kind=kind, tokens=_log_int(rng, 1, 16384), heads=heads, kv_heads=kv_heads, dim=dim, rotary=rotary,
                    sections=rng.choice([1, 1, 2, 3]), at=_log_int(rng, 1, 131072), theta=rng.choice([1e4, 1e6]),
                    norm=rng.choice(["", "", "own", "fp32"]), pairs=rng.choice(["halves", "halves", "neighbours"]),
                    dtype=rng.choice(["fp16", "bf16"]), pick=pick)
    if kind == "append":
        shape = rng.choice([(4, 64), (2, 64), (8, 128), (4, 80), (1, 96), (12, 40)])
        new = rng.choice([1, 1, _log_int(rng, 2, 2600)])
        return dict(kind=kind, requests=_log_int(rng, 1, 128 if new == 1 else 6), new=new, at=_log_int(rng, 1, 3000) - 1,
                    kv_heads=shape[0], dim=shape[1], block=rng.choice([16, 32, 64, 128]),
                    dtype=rng.choice(["fp16", "bf16"]), pick=pick)
    if kind == "attend":
        heads, kv_heads, dim = rng.choice(shapes)
        new = rng.choice([1, 1, 1, rng.randint(2, 8), _log_int(rng, 9, 1024)])
        return dict(kind=kind, requests=_log_int(rng, 1, 64 if new < 9 else 3), new=new,
                    context=_log_int(rng, 1, 32768 if new < 9 else 8000), block=rng.choice([16, 32, 64, 128]),
                    dtype=rng.choice(["fp16", "bf16"]), pick=pick, heads=heads, kv_heads=kv_heads, dim=dim)
    return dict(kind=kind, requests=_log_int(rng, 1, 64), rows=rng.randint(1, 8), ragged=rng.random() < 0.6,
                vocab=rng.choice([32000, 151936, _log_int(rng, 300, 151936)]), dtype=rng.choice(["fp16", "bf16", "fp32"]),
                drafter=rng.choice(["", "fp32", "fp32", "bf16", "fp16"]), temperature=round(rng.uniform(0.5, 1.3), 2),
                top_k=rng.choice([0, 0, 1, 50, 400]), top_p=rng.choice([1.0, 1.0, 0.9, 0.95, 0.5]),
                min_p=rng.choice([0.0, 0.0, 0.02, 0.1]), own_settings=rng.random() < 0.5, pick=pick)


def _cost(case):
    w = work(case)
    return w["bytes"] / 4e12 + w["flops"] / 4e14


def draw(rng: random.Random):
    """A case of the same ranges that costs no more than the largest listed one of its kind."""
    case = _draw(rng)
    while _cost(case) > max(_cost(c) for c in listed() if c["kind"] == case["kind"]):
        case = _draw(rng)
    return case


# ---- what a case is made of ----------------------------------------------------------

def _spans(case):
    """(tokens held before the call, new tokens) of each request: fixed by the case, ragged around its figures."""
    rng = random.Random(case["pick"])
    n = case["requests"]
    new = [case["new"] if case["new"] == 1 else rng.randint(max(1, case["new"] // 4), case["new"]) for _ in range(n)]
    if case["kind"] == "append":
        return [rng.randint(case["at"] // 2, case["at"]) for _ in range(n)], new
    held = [max(0, rng.randint(max(1, case["context"] // 2), case["context"]) - k) for k in new]
    held[0] = max(0, case["context"] - new[0])
    return held, new


def _verify_rows(case):
    rng = random.Random(case["pick"])
    return [rng.randint(1, case["rows"]) if case["ragged"] else case["rows"] for _ in range(case["requests"])]


def _padded(dim):
    return -(-dim // 32) * 32


def _tables(held, new, block, gen):
    """A block table over a shuffled pool with some blocks to spare, and the pool's size."""
    counts = [-(-(h + n) // block) for h, n in zip(held, new)]
    width, blocks = max(1, max(counts)), sum(counts) + 8
    ids = torch.randperm(blocks, generator=gen, device="cuda")[:sum(counts)].to(torch.int32).cpu()
    table = torch.full((len(held), width), -1, dtype=torch.int32)
    at = 0
    for r, c in enumerate(counts):
        table[r, :c] = ids[at:at + c]
        at += c
    return table.cuda(), blocks


def _codes(shape, gen):
    """Bytes of two 4-bit numbers each, as values of a normal distribution give them."""
    edge = torch.tensor([0.25, 0.75, 1.25, 1.75, 2.5, 3.5, 5.0], device="cuda")

    def four():
        x = torch.empty(shape, device="cuda").normal_(0, 2.2, generator=gen)
        return torch.bucketize(x.abs(), edge).to(torch.uint8) | (x < 0).to(torch.uint8) << 3

    return four() | four() << 4


def _pool(blocks, case, gen):
    """Keys [blocks, heads, block, bytes of a row] and values [blocks, heads, 16 tokens each, dims, 8 bytes], and the
    scales of 32 dims: keys' and values' [blocks, heads, groups, block]."""
    h, b, d, p = case["kv_heads"], case["block"], case["dim"], _padded(case["dim"])
    k, v = _codes((blocks, h, b, p // 2), gen), _codes((blocks, h, b // 16, p, 8), gen)
    k[..., d // 2:] = 0
    v[..., d:, :] = 0
    scale = lambda: torch.randint(100, 114, (blocks, h, p // 32, b), generator=gen, device="cuda",  # noqa: E731
                                  dtype=torch.int32).to(torch.uint8)
    return dict(k=k, v=v, k_scale=scale(), v_scale=scale(), dim=d)


def _slots(table, block, spans):
    """Slots of the positions [first, last) of each request, as int64 on the GPU."""
    host = table.cpu().to(torch.int64)
    out = []
    for r, (a, b) in enumerate(spans):
        p = torch.arange(a, b)
        out.append(host[r, p // block] * block + p % block)
    return torch.cat(out).cuda()


def _prepare_rope(case, gen):
    T, H, K, D, R = (case[n] for n in ("tokens", "heads", "kv_heads", "dim", "rotary"))
    dtype = DTYPES[case["dtype"]]
    # q and k are views of the rows of one projection, v between them and the next row
    x = torch.empty((T, H + 2 * K, D), device="cuda").normal_(0, 1, generator=gen)
    x = (x * (0.5 + torch.rand((T, H + 2 * K, 1), generator=gen, device="cuda"))).to(dtype)
    n, axes = R // 2, case["sections"]
    inv_freq = case["theta"] ** (-torch.arange(n, dtype=torch.float64, device="cuda") / n)
    axis = None
    if axes > 1:
        axis = (torch.arange(n, device="cuda") * axes // n).to(torch.int32)
        pos = torch.randint(0, case["at"], (axes, T), generator=gen, device="cuda", dtype=torch.int32)
    else:
        # (prompts of several requests: runs that begin anywhere)
        first = torch.randint(0, case["at"], (1 + T // 700,), generator=gen, device="cuda", dtype=torch.int32)
        at = torch.arange(T, device="cuda", dtype=torch.int32)
        pos = first[at // 700] + at % 700
    state = dict(q=x[:, :H], k=x[:, H:H + K], positions=pos, inv_freq=inv_freq, axis=axis, pairs=case["pairs"],
                 q_weight=None, k_weight=None)
    if case["norm"]:
        for name in ("q_weight", "k_weight"):
            w = 1 + 0.2 * torch.empty(D, device="cuda").normal_(0, 1, generator=gen)
            state[name] = w.to(torch.float32 if case["norm"] == "fp32" else dtype)
    return state


def _prepare_verify(case, gen):
    rows, V, R = _verify_rows(case), case["vocab"], case["requests"]
    T = sum(rows)
    x = torch.empty((T, V), device="cuda").normal_(0, 2.5, generator=gen)
    x[:, : max(1, V // 100)] += 3.0 * torch.rand((T, max(1, V // 100)), generator=gen, device="cuda")
    x = x[:, torch.randperm(V, generator=gen, device="cuda")]
    # a drafting model that is near the target, at the same temperature
    y = (x + 0.4 * torch.empty_like(x).normal_(0, 1, generator=gen)) / case["temperature"]
    q = (y - y.amax(-1, keepdim=True)).exp_()
    q /= q.sum(-1, keepdim=True)
    del y
    if case["drafter"]:
        q = q.to(DTYPES[case["drafter"]])
        run_sum = q.double().cumsum(-1)
        target = torch.rand((T, 1), generator=gen, device="cuda") * run_sum[:, -1:]
        drafts = (run_sum <= target).sum(-1).clamp(max=V - 1)
        del run_sum
    else:
        drafts, q = q.argmax(-1), None
    p = {n: case[n] for n in ("temperature", "top_k", "top_p", "min_p")}
    if case["own_settings"]:
        f = torch.rand((4, R), generator=gen, device="cuda")
        p["temperature"] = case["temperature"] * (0.6 + 0.6 * f[0])
        p["temperature"][5::16] = 0.0  # greedy requests
        p["top_k"] = (case["top_k"] * f[1]).to(torch.int32)
        p["top_p"] = 1 - (1 - case["top_p"]) * f[2]
        p["min_p"] = case["min_p"] * f[3]
    logits, cu = x.to(DTYPES[case["dtype"]]), None
    u = torch.rand(T, generator=gen, device="cuda")
    if case["ragged"]:
        cu = torch.tensor([0] + list(np.cumsum(rows)), dtype=torch.int32, device="cuda")
    else:
        fold = lambda t: None if t is None else t.view(R, case["rows"], *t.shape[1:])  # noqa: E731
        logits, drafts, u, q = fold(logits), fold(drafts), fold(u), fold(q)
    return dict(logits=logits, drafts=drafts, u=u, draw=torch.rand(R, generator=gen, device="cuda"), cu=cu,
                draft_probs=q, **p)


def prepare(case, seed):
    gen = torch.Generator(device="cuda").manual_seed(seed)
    kind = case["kind"]
    if kind == "rope":
        return dict(kind=kind, **_prepare_rope(case, gen))
    if kind == "verify":
        return dict(kind=kind, **_prepare_verify(case, gen))
    held, new = _spans(case)
    block = case["block"]
    table, blocks = _tables(held, new, block, gen)
    pool = _pool(blocks, case, gen)
    dtype = DTYPES[case["dtype"]]
    T = sum(new)
    if kind == "append":
        h, d = case["kv_heads"], case["dim"]
        kv = torch.empty((T, 2 * h, d), device="cuda").normal_(0, 1, generator=gen)
        kv *= 0.6 + 0.8 * torch.rand((T, 2 * h, 1), generator=gen, device="cuda")
        kv = kv.to(dtype)  # k and v are views of one projection's rows
        return dict(kind=kind, pool=pool, k=kv[:, :h], v=kv[:, h:],
                    slots=_slots(table, block, [(a, a + n) for a, n in zip(held, new)]),
                    back=_slots(table, block, [(a // block * block, a + n) for a, n in zip(held, new)]))
    q = torch.empty((T, case["heads"], case["dim"]), device="cuda").normal_(0, 1.5, generator=gen).to(dtype)
    lens = torch.tensor([a + n for a, n in zip(held, new)], dtype=torch.int32, device="cuda")
    cu = None
    if case["new"] > 1:
        cu = torch.tensor([0] + list(np.cumsum(new)), dtype=torch.int32, device="cuda")
    return dict(kind=kind, pool=pool, q=q, table=table, lens=lens, cu=cu, most=max(new))


# ---- plain forms ---------------------------------------------------------------------

def rope_plain(x, weight, cos, sin, pairs):
    T, H, D = x.shape
    n = cos.shape[-1]
    y = x.float()
    if weight is not None:
        y = y * torch.rsqrt((y * y).mean(-1, keepdim=True) + 1e-6) * weight.float()
    if pairs == "halves":
        a, b, rest = y[..., :n], y[..., n:2 * n], y[..., 2 * n:]
        parts = [a * cos - b * sin, b * cos + a * sin]
    else:
        a, b, rest = y[..., 0:2 * n:2], y[..., 1:2 * n:2], y[..., 2 * n:]
        parts = [torch.stack([a * cos - b * sin, b * cos + a * sin], -1).view(T, H, 2 * n)]
    return torch.cat(parts + [rest], -1).to(x.dtype)


def qk_rope_plain(s):
    pos = s["positions"].double()
    at = pos[:, None] if s["axis"] is None else pos[s["axis"].long()].T  # [tokens, 1 or pairs]
    angle = at * s["inv_freq"]  # (64 bits: far positions turn thousands of times)
    cos, sin = angle.cos().float()[:, None], angle.sin().float()[:, None]
    return tuple(rope_plain(s[n], s[n + "_weight"], cos, sin, s["pairs"]) for n in ("q", "k"))


VALUES = (0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0)


def scale_value(byte):
    """The number that a scale's byte stands for: the upper bits of a positive fp16 number."""
    return (byte.to(torch.int16) << 7).view(torch.float16).float()


def scale_plain(most):
    """Bytes of the smallest scales that hold `most` as six of them."""
    most = most.clamp(max=61440.0)
    least = (most / 6).to(torch.float16).view(torch.int16) >> 7  # (down to a byte, or up to the next)
    least = (least - 1).clamp(min=0)
    for _ in range(2):
        least = torch.where(scale_value(least) * 6 < most, least + 1, least)
    return least.to(torch.uint8)


def quantise_plain(x):
    """4-bit numbers [..., dims padded to 32] of x [..., dims] and scale bytes [..., groups]."""
    x = x.float()
    x = torch.where(torch.isfinite(x), x, torch.where(x < 0, -61440.0, 61440.0)).clamp(-61440.0, 61440.0)
    x = torch.cat([x, x.new_zeros(*x.shape[:-1], _padded(x.shape[-1]) - x.shape[-1])], -1)
    g = x.view(*x.shape[:-1], -1, 32)
    byte = scale_plain(g.abs().amax(-1))
    s, a = scale_value(byte)[..., None], g.abs()
    # ties go to the even one: borders are above for codes 0, 2, 4, 6 and below for the others
    code = sum((a > m * s if i % 2 == 0 else a >= m * s).to(torch.uint8)
               for i, m in enumerate((0.25, 0.75, 1.25, 1.75, 2.5, 3.5, 5.0)))
    code = torch.where(s > 0, code, 0).to(torch.uint8)
    return (code | (g < 0).to(torch.uint8) << 3).view(x.shape), byte


def append_plain(codes, scale, x, slots, block, keys_last):
    """Rows x [T, heads, dim] into a pool of codes (keys_last: the layout of v), in place."""
    live = ((slots >= 0) & (slots < scale.shape[0] * block)).nonzero()[:, 0]
    slot = slots[live]
    blk, off = slot // block, slot % block
    code, byte = quantise_plain(x[live])
    scale[blk, :, :, off] = byte
    if not keys_last:
        codes[blk, :, off] = code[..., 0::2] | code[..., 1::2] << 4
        return
    # pieces of 16 tokens: their nibbles, the new ones among them
    pieces = codes.permute(0, 2, 1, 3, 4).reshape(-1, codes.shape[1], codes.shape[3], 8)
    piece = slot // 16
    touched = torch.bincount(piece, minlength=pieces.shape[0]).nonzero()[:, 0]
    held = pieces[touched]
    held = torch.stack([held & 15, held >> 4], -1).flatten(-2)
    row = torch.searchsorted(touched, piece)
    held[row, :, :, off % 16] = code
    held = held[..., 0::2] | held[..., 1::2] << 4
    codes[touched // (block // 16), :, touched % (block // 16)] = held


def values_plain(byte, real):
    """The two numbers of each byte, along a new last dimension."""
    table = torch.tensor(VALUES + tuple(-v for v in VALUES), dtype=real, device=byte.device)
    return torch.stack([table[(byte & 15).long()], table[(byte >> 4).long()]], -1)


def read_plain(pool, slots, block, dtype):
    blk, off, d = slots // block, slots % block, pool["dim"]
    k = values_plain(pool["k"][blk, :, off], torch.float32).flatten(-2)
    v = pool["v"][blk, :, off // 16, :, off % 16 // 2]
    v = values_plain(torch.where((off % 2 > 0)[:, None, None], v >> 4, v & 15), torch.float32)[..., 0]
    ks, vs = (scale_value(pool[n][blk, :, :, off]).repeat_interleave(32, -1) for n in ("k_scale", "v_scale"))
    return (k * ks)[..., :d].to(dtype), (v * vs)[..., :d].to(dtype)


def _gathered(pool, table, real):
    """Keys and values [requests, kv heads, width * block, dim] of whole tables, and whether each page is there."""
    ids = table.long()
    there = (ids >= 0) & (ids < pool["k"].shape[0])
    ids = torch.where(there, ids, 0)
    R, W = ids.shape
    H, B, P = pool["k"].shape[1], pool["k"].shape[2], pool["v"].shape[3]
    k = values_plain(pool["k"][ids], real).flatten(-2).permute(0, 2, 1, 3, 4).reshape(R, H, W * B, P)
    v = values_plain(pool["v"][ids], real).flatten(-2).permute(0, 2, 1, 3, 5, 4).reshape(R, H, W * B, P)
    for x, n in ((k, "k_scale"), (v, "v_scale")):
        s = scale_value(pool[n][ids]).to(real).permute(0, 2, 1, 4, 3).reshape(R, H, W * B, P // 32)
        x.view(R, H, W * B, P // 32, 32).mul_(s[..., None])
    return k[..., :pool["dim"]], v[..., :pool["dim"]], there.repeat_interleave(B, 1)


def attend_plain(q, pool, table, lens, cu, most):
    T, H, D = q.shape
    R, Hkv = table.shape[0], pool["k"].shape[1]
    k, v, there = _gathered(pool, table, torch.float32)
    i = torch.arange(most, device=q.device)
    first = torch.arange(R, device=q.device) if cu is None else cu[:-1].long()
    count = torch.ones_like(first) if cu is None else cu[1:].long() - first
    row = torch.where(i < count[:, None], first[:, None] + i, T)  # (T: no such row)
    qp = torch.cat([q.float(), q.new_zeros((1, H, D), dtype=torch.float32)])[row]
    qp = qp.reshape(R, most, Hkv, H // Hkv, D).permute(0, 2, 3, 1, 4).reshape(R, Hkv, -1, D)
    s = torch.matmul(qp, k.transpose(2, 3)).mul_(D ** -0.5).view(R, Hkv, H // Hkv, most, -1)
    last = lens.long()[:, None] - count[:, None] + i  # the last key that row i sees
    j = torch.arange(s.shape[-1], device=q.device)
    seen = (j <= last[..., None]) & (j < lens.long()[:, None, None]) & there[:, None]
    s.masked_fill_(~seen[:, None, None], -math.inf)
    top = s.amax(-1, keepdim=True)
    p = s.sub_(torch.where(top == -math.inf, 0, top)).exp_()
    total = p.sum(-1, keepdim=True)
    o = torch.matmul(p.view(R, Hkv, -1, s.shape[-1]), v).view(R, Hkv, H // Hkv, most, D)
    o = torch.where(total > 0, o / total, 0).permute(0, 3, 1, 2, 4).reshape(R, most, H, D)
    out = q.new_zeros((T + 1, H, D), dtype=torch.float32)
    out[row.reshape(-1)] = o.reshape(-1, H, D)
    return out[:T].to(q.dtype)


def kept_plain(logits, temperature, top_k, top_p, min_p):
    """Probabilities [rows, vocab] (64 bits) of what the settings keep, and whether a row has any."""
    x = logits.double()
    B, V = x.shape
    column = lambda p: (p.double() if isinstance(p, torch.Tensor) else  # noqa: E731
                        torch.full((B,), float(np.float32(p)), dtype=torch.float64, device=x.device))[:, None]
    t, k, p, m = column(temperature), column(top_k), column(top_p), column(min_p)
    xs, order = x.sort(dim=-1, descending=True, stable=True)  # (ties: the lowest index first)
    top = xs[:, :1]
    w = torch.where(xs == top, 0, (xs - top) / torch.where(t > 0, t, 1)).exp_()
    rank = torch.arange(V, device=x.device)
    w = torch.where((k <= 0) | (rank < k), w, 0)
    before = w.cumsum(-1)
    total = before[:, -1:].clone()
    before = torch.cat([torch.zeros_like(total), before[:, :-1]], -1)
    keep = ((p >= 1) | (before < p * total) | (rank == 0)) & (w >= m.clamp(max=1)) & (w > 0)
    keep = torch.where(t > 0, keep, rank == 0)
    kept = torch.zeros_like(x).scatter_(-1, order, torch.where(keep, w, 0))
    bad = torch.isnan(x).any(-1) | (top[:, 0] == -math.inf)
    return kept / kept.sum(-1, keepdim=True), ~bad


def verify_plain(s):
    logits, V, R = s["logits"], s["logits"].shape[-1], s["draw"].shape[0]
    logits = logits.reshape(-1, V)
    T = logits.shape[0]
    t = torch.arange(T, device=logits.device)
    cu = s["cu"].long() if s["cu"] is not None else torch.arange(R + 1, device=t.device) * (T // max(1, R))
    r = (torch.searchsorted(cu, t, right=True) - 1).clamp(max=R - 1)
    per_row = [x[r] if isinstance(x, torch.Tensor) else x for x in
               (s["temperature"], s["top_k"], s["top_p"], s["min_p"])]
    p, good = kept_plain(logits, *per_row)
    d, u = s["drafts"].reshape(-1), s["u"].reshape(-1).double()
    if s["draft_probs"] is None:
        q = torch.zeros_like(p).scatter_(-1, d[:, None], 1.0)
    else:
        q = s["draft_probs"].reshape(T, V).double()
    last = t == cu[1:][r] - 1
    pd, qd = (x.gather(-1, d[:, None])[:, 0] for x in (p, q))
    accept = (pd > u * qd) & good & ~last
    # the first row of each request that is not accepted
    stop = torch.full((R,), T, device=t.device).scatter_reduce_(0, r, torch.where(accept, T, t), "amin")
    row = stop.clamp(max=T - 1)
    left = torch.where(last[row][:, None], p[row], (p[row] - q[row]).clamp(min=0))
    left = torch.where(left.sum(-1, keepdim=True) > 0, left, p[row])
    run_sum = left.cumsum(-1)
    drawn = (run_sum <= s["draw"].double()[:, None] * run_sum[:, -1:]).sum(-1)
    drawn = torch.where(good[row], drawn, -1)
    tokens = torch.where(t < stop[r], d, torch.where(t == stop[r], drawn[r], -1))
    return dict(tokens=tokens.reshape(s["drafts"].shape), counts=(stop - cu[:-1] + 1).int())


def run(state):
    kind, s = state["kind"], state
    if own:
        import __graft_entry__

        hx = __graft_entry__.load_package()
        if kind == "rope":
            return hx.qk_rope(s["q"], s["k"], s["positions"], s["inv_freq"], axis=s["axis"], q_weight=s["q_weight"],
                              k_weight=s["k_weight"], interleaved=s["pairs"] == "neighbours")
        if kind == "verify":
            v = hx.verify(s["logits"], s["drafts"], s["u"], s["draw"], cu=s["cu"], draft_probs=s["draft_probs"],
                          temperature=s["temperature"], top_k=s["top_k"], top_p=s["top_p"], min_p=s["min_p"])
            return dict(tokens=v.tokens, counts=v.counts)
        c = s["pool"]
        cache = hx.KVCache4(c["k"], c["v"], c["k_scale"], c["v_scale"], c["dim"])
        if kind == "append":
            hx.kv_append(cache, s["k"], s["v"], s["slots"])
            return hx.kv_read(cache, s["back"], dtype=s["k"].dtype)
        return hx.kv_attention(s["q"], cache, s["table"], s["lens"], cu=s["cu"])
    if kind == "rope":
        return qk_rope_plain(s)
    if kind == "verify":
        return verify_plain(s)
    c = s["pool"]
    block = c["k"].shape[2]
    if kind == "append":
        append_plain(c["k"], c["k_scale"], s["k"], s["slots"], block, False)
        append_plain(c["v"], c["v_scale"], s["v"], s["slots"], block, True)
        return read_plain(c, s["back"], block, s["k"].dtype)
    return attend_plain(s["q"], c, s["table"], s["lens"], s["cu"], s["most"])


def work(case):
    kind = case["kind"]
    if kind == "rope":
        # rows in and out; an angle's cosine and sine for each pair of a token, a rotation (and a norm) for each value
        n = case["tokens"] * (case["heads"] + case["kv_heads"]) * case["dim"]
        return dict(bytes=4 * n + 4 * case["tokens"] * case["sections"],
                    flops=n * (7 if case["norm"] else 3) + 20 * case["tokens"] * case["rotary"])
    if kind == "verify":
        # every row of logits, and the draft's distribution where a request's token is drawn
        n = sum(_verify_rows(case)) * case["vocab"]
        drafter = SIZES[case["drafter"]] * case["requests"] * case["vocab"] if case["drafter"] else 0
        return dict(bytes=n * SIZES[case["dtype"]] + drafter, flops=4 * n + 4 * case["requests"] * case["vocab"])
    held, new = _spans(case)
    d, h = case["dim"], case["kv_heads"]
    held_bytes = d / 2 + -(-d // 32)  # of a token and head of K or V
    if kind == "append":
        # rows in, their codes out and read back with those of their blocks
        back = sum(a % case["block"] + n for a, n in zip(held, new))
        values = h * d * 2
        return dict(bytes=int(2 * h * (sum(new) * held_bytes + back * held_bytes) + values * 2 * (sum(new) + back)),
                    flops=values * (sum(new) * 4 + back))
    pairs = sum(n * a + n * (n + 1) // 2 for a, n in zip(held, new))
    keys = sum(a + n for a, n in zip(held, new))
    return dict(bytes=int(keys * h * 2 * held_bytes + sum(new) * case["heads"] * d * 4),
                flops=4 * pairs * case["heads"] * d)


# ---- the definitions, in 64 bits -----------------------------------------------------

def _exact_rope(s):
    out = []
    pos = s["positions"].double()
    at = pos[:, None] if s["axis"] is None else torch.stack([pos[a] for a in s["axis"].tolist()], -1)
    turn = torch.exp(1j * (at * s["inv_freq"]))[:, None]  # [tokens, 1, pairs]
    n = turn.shape[-1]
    for name in ("q", "k"):
        x = s[name].double()
        w = s[name + "_weight"]
        if w is not None:
            x = x / (x.pow(2).sum(-1, keepdim=True) / x.shape[-1] + 1e-6).sqrt() * w.double()
        y = x.clone()
        if s["pairs"] == "halves":
            z = torch.complex(x[..., :n], x[..., n:2 * n]) * turn
            y[..., :n], y[..., n:2 * n] = z.real, z.imag
        else:
            z = torch.view_as_complex(x[..., :2 * n].reshape(*x.shape[:2], n, 2).contiguous()) * turn
            y[..., :2 * n] = torch.view_as_real(z).flatten(-2)
        out.append(y)
    return tuple(out)


def _exact_held(pool, name):
    """What a pool holds, [blocks, heads, block, dim]."""
    B, H, G, block = pool[name + "_scale"].shape
    four = pool[name].to(torch.int64)
    four = torch.stack([four % 16, four // 16], -1).flatten(-2)
    if name == "v":
        four = four.transpose(-1, -2).reshape(B, H, block, -1)
    # one sign, two exponent bits and one of mantissa: 0 and 1/2, then (2 + m) / 2 * 2^(e - 1)
    e, m = four // 2 % 4, (four % 2).double()
    number = torch.where(e > 0, torch.ldexp(2 + m, e - 2), m / 2) * torch.where(four >= 8, -1.0, 1.0)
    # five exponent bits and three of mantissa
    byte = pool[name + "_scale"].to(torch.int64)
    e, m = byte // 8, (byte % 8).double()
    scale = torch.where(e > 0, torch.ldexp(8 + m, e - 18), m * 2.0 ** -17)
    return (number * scale.transpose(2, 3).repeat_interleave(32, -1))[..., :pool["dim"]]


def _exact_append(s):
    pool, out = s["pool"], []
    d = pool["dim"]
    slots, back = s["slots"], s["back"]
    value = torch.tensor([0, 0.5, 1, 1.5, 2, 3, 4, 6], dtype=torch.float64, device="cuda")
    # every scale there is, ascending: m * 2^e of four bits, and those below 2^-14
    scales = torch.tensor(sorted({m * 2.0 ** -17 for m in range(8)} |
                                 {(8 + m) * 2.0 ** (e - 17) for e in range(31) for m in range(8)}),
                          dtype=torch.float64, device="cuda")
    scales = scales[scales <= 10240.0]
    for name, x in (("k", s["k"]), ("v", s["v"])):
        cells = _exact_held(pool, name).transpose(1, 2).flatten(0, 1).clone()  # one row a slot
        y = x.double()
        for g in range(-(-d // 32)):
            part = y[..., 32 * g:min(d, 32 * g + 32)]
            scale = scales[torch.searchsorted(scales * 6, part.abs().amax(-1).contiguous())][..., None]
            r = torch.where(scale > 0, part.abs() / scale, 0)  # (a tie is one exactly)
            # among the two numbers beside r the nearer, of two as near the one with the even code
            hi = torch.searchsorted(value, r.contiguous()).clamp(1, 7)
            lo, up, down = hi - 1, value[hi] - r, r - value[hi - 1]
            code = torch.where(up < down, hi, torch.where(up > down, lo, torch.where(hi % 2 == 0, hi, lo)))
            cells[slots, :, 32 * g:min(d, 32 * g + 32)] = torch.sign(part) * value[code] * scale
        out.append(cells[back])
    return tuple(out)


def _exact_attend(s):
    q, pool, lens, table = s["q"], s["pool"], s["lens"].tolist(), s["table"].long()
    T, H, D = q.shape
    group = H // pool["k"].shape[1]
    block = pool["k"].shape[2]
    cu = list(range(T + 1)) if s["cu"] is None else s["cu"].tolist()
    out = torch.zeros((T, H, D), dtype=torch.float64, device=q.device)
    for r, n in enumerate(lens):
        pages = table[r, :-(-n // block)]
        own = dict(dim=D, **{name: pool[name][pages] for name in ("k", "v", "k_scale", "v_scale")})
        k, v = (_exact_held(own, name).transpose(0, 1).flatten(1, 2)[:, :n] for name in ("k", "v"))
        x = q[cu[r]:cu[r + 1]].double().transpose(0, 1)  # [heads, rows, dim]
        rows = x.shape[1]
        hidden = torch.ones((rows, n), dtype=torch.bool, device=q.device).triu(n - rows + 1)
        for h in range(H):
            scores = (x[h] @ k[h // group].T) / math.sqrt(D)
            p = scores.masked_fill_(hidden, -math.inf).softmax(-1)
            out[cu[r]:cu[r + 1], h] = p @ v[h // group]
    return out


def _exact_verify(s):
    V, R = s["logits"].shape[-1], s["draw"].shape[0]
    logits = s["logits"].reshape(-1, V).float().cpu().numpy().astype(np.float64)
    T = logits.shape[0]
    cu = s["cu"].tolist() if s["cu"] is not None else list(range(0, T + 1, T // R))
    q = None if s["draft_probs"] is None else s["draft_probs"].reshape(T, V).float().cpu().numpy().astype(np.float64)
    drafts, u, draw = s["drafts"].reshape(-1).tolist(), s["u"].reshape(-1).tolist(), s["draw"].tolist()
    setting = {n: s[n].tolist() if isinstance(s[n], torch.Tensor) else [float(np.float32(s[n]))] * R
               for n in ("temperature", "top_k", "top_p", "min_p")}

    def target(x, r):
        """(kept tokens in order of their index, their probabilities)"""
        t, k, p, m = (setting[n][r] for n in ("temperature", "top_k", "top_p", "min_p"))
        if t <= 0:
            return np.array([np.argmax(x)]), np.ones(1)
        order = np.argsort(-x, kind="stable")[:int(k) if k > 0 else V]
        w = np.exp((x[order] - x.max()) / t)
        if p < 1:
            cum = np.concatenate([[0.0], np.cumsum(w)[:-1]])
            n = max(1, int(np.searchsorted(cum, p * w.sum(), side="left")))
            order, w = order[:n], w[:n]
        order, w = order[w >= min(m, 1.0)], w[w >= min(m, 1.0)]
        by = np.argsort(order)
        return order[by], w[by] / w.sum()

    tokens, counts = [-1] * T, []
    for r in range(R):
        for i in range(cu[r], cu[r + 1]):
            index, p = target(logits[i], r)
            d, final = drafts[i], i + 1 == cu[r + 1]
            if not final:
                at = int(np.searchsorted(index, d))
                pd = p[at] if at < len(index) and index[at] == d else 0.0
                qd = 1.0 if q is None else q[i, d]
                if pd > u[i] * qd:
                    tokens[i] = d
                    continue
                left = np.where(index == d, 0.0, p) if q is None else np.maximum(p - q[i, index], 0.0)
                p = left if left.sum() > 0 else p
            cum = np.cumsum(p)
            tokens[i] = int(index[np.searchsorted(cum, draw[r] * cum[-1], side="right")])
            counts.append(i + 1 - cu[r])
            break
    return dict(tokens=torch.tensor(tokens, dtype=torch.int64).reshape(s["drafts"].shape),
                counts=torch.tensor(counts, dtype=torch.int32))


def exact(case, seed):
    s = prepare(case, seed)
    return dict(rope=_exact_rope, append=_exact_append, attend=_exact_attend, verify=_exact_verify)[case["kind"]](s)
