"""The operators of a serving step after the prompt, as measurable cases.

A step over a batch of requests takes blocks of an 8-bit key/value cache for
its new tokens (``kv_plan``), writes their keys and values into it
(``kv_append``, read back by ``kv_read``), attends over it (``kv_attention``)
and takes the next token from the logits (``sample``).  ``listed()`` holds the
cases, ``draw(rng)`` takes one more from the same ranges, ``prepare`` makes
what a program has in hand before the call, ``run`` is one pass (in elementary
torch operations, or with ``own`` through the library), ``work`` what the pass
cannot do without and ``exact`` the same results from the definitions in 64
bits.
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
        # one decode step of a small batch: a few requests, most inside their last block
        dict(name="plan_decode_16", kind="plan", requests=16, tokens=16, width=64, block=64, chunk=1, pick=1),
        # a step that mixes decoding requests, prompt chunks and requests that have ended
        dict(name="plan_mixed_1024", kind="plan", requests=1024, tokens=16384, width=512, block=16, chunk=512, pick=2),
        # one token a request into half-filled blocks
        dict(name="append_decode_128", kind="append", requests=128, new=1, at=3000, kv_heads=8, dim=128, block=64,
             dtype="bf16", pick=3),
        # prompt chunks of ragged lengths that begin and end inside blocks
        dict(name="append_prompt_8192", kind="append", requests=5, new=2600, at=700, kv_heads=4, dim=64, block=32,
             dtype="fp16", pick=4),
        # TinyLlama decoding for a single user: latency
        dict(name="attend_one_user", kind="attend", requests=1, context=1900, new=1, block=64, dtype="fp16", pick=5,
             **TINYLLAMA),
        # a full serving batch, contexts up to 8192
        dict(name="attend_batch_64x8192", kind="attend", requests=64, context=8192, new=1, block=64, dtype="bf16",
             pick=6, **WIDE),
        # one very long context, one token
        dict(name="attend_long_131072", kind="attend", requests=1, context=131072, new=1, block=32, dtype="fp16",
             pick=7, **WIDE),
        # drafted tokens to be checked: one to five rows a request, small pages, 7 query heads a key head
        dict(name="attend_drafts_37", kind="attend", requests=37, context=1500, new=5, block=16, dtype="bf16", pick=8,
             **QWEN),
        # prompt chunks over contexts that are in the cache already
        dict(name="attend_chunks_3x1024", kind="attend", requests=3, context=8000, new=1024, block=64, dtype="fp16",
             pick=9, **WIDE),
        # one user, TinyLlama's vocabulary, the usual top-k
        dict(name="sample_one_32000", kind="sample", rows=1, vocab=32000, dtype="fp16", temperature=0.8, top_k=50,
             top_p=1.0, min_p=0.0, per_row=False),
        # a batch over Qwen2.5's vocabulary, nucleus sampling
        dict(name="sample_top_p_64", kind="sample", rows=64, vocab=151936, dtype="bf16", temperature=0.9, top_k=0,
             top_p=0.95, min_p=0.0, per_row=False),
        # the largest batch, logits in 32 bits, every request with its own settings
        dict(name="sample_mixed_256", kind="sample", rows=256, vocab=151936, dtype="fp32", temperature=1.0, top_k=400,
             top_p=0.9, min_p=0.02, per_row=True),
    ]


def _log_int(rng, lo, hi):
    return min(hi, max(lo, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def _draw(rng):
    kind = rng.choice(["plan", "append", "append", "attend", "attend", "attend", "sample", "sample"])
    pick = rng.randrange(1 << 30)
    if kind == "plan":
        requests, chunk = _log_int(rng, 1, 1024), rng.choice([1, 1, 5, 512])
        return dict(kind=kind, requests=requests, chunk=chunk, width=_log_int(rng, 4, 512),
                    tokens=min(16384, max(1, requests * chunk // rng.choice([1, 1, 4]) + rng.randint(0, 7))),
                    block=rng.choice([16, 32, 64, 128]), pick=pick)
    if kind == "append":
        shape = rng.choice([(4, 64), (2, 64), (8, 128), (4, 80), (1, 96), (12, 40)])
        new = rng.choice([1, 1, _log_int(rng, 2, 2600)])
        return dict(kind=kind, requests=_log_int(rng, 1, 128 if new == 1 else 6), new=new, at=_log_int(rng, 1, 3000) - 1,
                    kv_heads=shape[0], dim=shape[1], block=rng.choice([16, 32, 64, 128]),
                    dtype=rng.choice(["fp16", "bf16"]), pick=pick)
    if kind == "attend":
        heads, kv_heads, dim = rng.choice([(32, 4, 64), (14, 2, 64), (32, 8, 128), (12, 12, 64), (16, 4, 128),
                                           (8, 1, 96), (4, 4, 80), (25, 5, 40)])
        new = rng.choice([1, 1, 1, rng.randint(2, 8), _log_int(rng, 9, 1024)])
        return dict(kind=kind, requests=_log_int(rng, 1, 64 if new < 9 else 3), new=new,
                    context=_log_int(rng, 1, 32768 if new < 9 else 8000), block=rng.choice([16, 32, 64, 128]),
                    dtype=rng.choice(["fp16", "bf16"]), pick=pick, heads=heads, kv_heads=kv_heads, dim=dim)
    return dict(kind=kind, rows=_log_int(rng, 1, 256), vocab=rng.choice([32000, 151936, _log_int(rng, 300, 151936)]),
                dtype=rng.choice(["fp16", "bf16", "fp32"]), temperature=round(rng.uniform(0.5, 1.3), 2),
                top_k=rng.choice([0, 1, 20, 50, 400]), top_p=rng.choice([1.0, 1.0, 0.9, 0.95, 0.5]),
                min_p=rng.choice([0.0, 0.0, 0.02, 0.1]), per_row=rng.random() < 0.5)


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
    if case["kind"] == "plan":
        limit = case["width"] * case["block"]
        held = [rng.randint(0, max(0, limit - case["chunk"])) for _ in range(n)]
        # a twentieth has ended, a tenth idles, the others decode or bring a chunk of a prompt
        kinds = [rng.random() for _ in range(n)]
        new = [-1 if k < 0.05 else 0 if k < 0.15 else 1 if k < 0.9 or case["chunk"] == 1 else
               rng.randint(1, case["chunk"]) for k in kinds]
        return held, new
    new = [case["new"] if case["new"] == 1 else rng.randint(max(1, case["new"] // 4), case["new"]) for _ in range(n)]
    if case["kind"] == "append":
        return [rng.randint(case["at"] // 2, case["at"]) for _ in range(n)], new
    held = [max(0, rng.randint(max(1, case["context"] // 2), case["context"]) - k) for k in new]
    held[0] = max(0, case["context"] - new[0])
    return held, new


def _padded(dim):
    return -(-dim // 16) * 16


def _tables(held, new, block, gen):
    """A block table over a shuffled pool with some blocks to spare, and the pool's size."""
    counts = [-(-(h + max(n, 0)) // block) for h, n in zip(held, new)]
    width, blocks = max(1, max(counts)), sum(counts) + 8
    ids = torch.randperm(blocks, generator=gen, device="cuda")[:sum(counts)].to(torch.int32).cpu()
    table = torch.full((len(held), width), -1, dtype=torch.int32)
    at = 0
    for r, c in enumerate(counts):
        table[r, :c] = ids[at:at + c]
        at += c
    return table.cuda(), blocks


def _scale(shape, gen):
    """Block scales as the cache holds them: a spread of amax / 127 in 11 significant bits."""
    s = (0.02 + 0.02 * torch.rand(shape, generator=gen, device="cuda"))
    return (s.view(torch.int32) & ~0x1FFF).view(torch.float32)


def _codes(shape, gen):
    x = torch.empty(shape, dtype=torch.float16, device="cuda").normal_(0, 36, generator=gen)
    return x.round_().clamp_(-127, 127).to(torch.int8)


def _pool(blocks, case, gen):
    h, b, d = case["kv_heads"], case["block"], case["dim"]
    k, v = _codes((blocks, h, b, _padded(d)), gen), _codes((blocks, h, b // 16, _padded(d), 16), gen)
    k[..., d:] = 0
    v[..., d:, :] = 0
    return dict(k=k, v=v, k_scale=_scale((blocks, h), gen), v_scale=_scale((blocks, h), gen), dim=d)


def _slots(table, block, spans):
    """Slots of the positions [first, last) of each request, as int64 on the GPU."""
    host = table.cpu().to(torch.int64)
    out = []
    for r, (a, b) in enumerate(spans):
        p = torch.arange(a, b)
        out.append(host[r, p // block] * block + p % block)
    return torch.cat(out).cuda()


def prepare(case, seed):
    gen = torch.Generator(device="cuda").manual_seed(seed)
    kind = case["kind"]
    if kind == "sample":
        B, V = case["rows"], case["vocab"]
        x = torch.empty((B, V), device="cuda").normal_(0, 2.5, generator=gen)
        x[:, : max(1, V // 100)] += 3.0 * torch.rand((B, max(1, V // 100)), generator=gen, device="cuda")
        x = x.gather(1, torch.randperm(V, generator=gen, device="cuda").expand(B, V)).to(DTYPES[case["dtype"]])
        p = {n: case[n] for n in ("temperature", "top_k", "top_p", "min_p")}
        if case["per_row"]:
            f = torch.rand((4, B), generator=gen, device="cuda")
            p["temperature"] = case["temperature"] * (0.5 + f[0])
            p["temperature"][::16] = 0.0  # greedy requests
            p["top_k"] = (case["top_k"] * f[1]).to(torch.int32)
            p["top_p"] = 1 - (1 - case["top_p"]) * f[2]
            p["min_p"] = case["min_p"] * f[3]
        return dict(kind=kind, logits=x, u=torch.rand(B, generator=gen, device="cuda"), **p)
    held, new = _spans(case)
    block = case["block"]
    if kind == "plan":
        R, W = case["requests"], case["width"]
        blocks = R * W
        counts = torch.tensor([-(-h // block) for h in held], device="cuda")
        ids = torch.randperm(blocks, generator=gen, device="cuda").to(torch.int32)
        col = torch.arange(W, device="cuda")
        first = counts.cumsum(0) - counts
        used = int(counts.sum())
        table = torch.where(col < counts[:, None], ids[(first[:, None] + col).clamp(max=blocks - 1)], -1)
        free = torch.zeros(blocks, dtype=torch.int32, device="cuda")
        # most of the step's needs can be met, the last requests' not always
        spare = min(blocks - used, sum(1 for n in new if n > 0) * (1 + case["chunk"] // (4 * block)))
        free[:spare] = ids[used:used + spare]
        return dict(kind=kind, lens=torch.tensor(held, dtype=torch.int32, device="cuda"),
                    new=torch.tensor(new, dtype=torch.int32, device="cuda"), table=table.to(torch.int32), free=free,
                    free_count=torch.tensor([spare], dtype=torch.int32, device="cuda"), block=block,
                    tokens=case["tokens"])
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

def plan_plain(lens, new, table, free, free_count, block, tokens):
    """Block table and stack in place; slots, positions, cu, lens, free_count."""
    W, F = table.shape[1], free.shape[0]
    held, add, col = lens.long(), new.long().clamp(min=0), torch.arange(W, device=lens.device)
    have = (held + block - 1) // block
    cu = torch.cat([torch.zeros_like(add[:1]), add.cumsum(0)])
    need = torch.where(add > 0, (held + add + block - 1) // block - have, 0)
    fits = (add > 0) & (have + need <= W) & (cu[1:] <= tokens)
    want = torch.where(fits, need, 0)
    back = torch.where(new < 0, have.clamp(max=W), 0)
    avail = free_count.long() + back.sum()
    admitted = fits & ((want == 0) | (want.cumsum(0) <= avail))
    take = torch.where(admitted, want, 0)
    # released blocks go on the stack in request order, taken ones come off its top in request order
    at = free_count.long() + (back.cumsum(0) - back)[:, None] + col
    stack = torch.cat([free, free[:1]])
    stack.scatter_(0, torch.where((col < back[:, None]) & (at < F), at, F).reshape(-1), table.reshape(-1))
    first = take.cumsum(0) - take
    j = col - have[:, None]
    taken = stack[(avail - 1 - first[:, None] - j).clamp(0, F)]
    table.copy_(torch.where((j >= 0) & (j < take[:, None]), taken, table))
    free.copy_(stack[:F])
    t = torch.arange(tokens, device=lens.device)
    r = (torch.searchsorted(cu, t, right=True) - 1).clamp(max=lens.shape[0] - 1)
    pos = held[r] + t - cu[r]
    ok = (t < cu[-1]) & admitted[r]
    pos = torch.where(ok, pos, 0)
    entry = table[r, pos // block].long()
    slots = torch.where(ok & (entry >= 0), entry * block + pos % block, -1)
    after = torch.where(new < 0, 0, torch.where(admitted, held + add, held))
    return slots, pos.int(), cu.int(), after.int(), (avail - take.sum()).int()


def scale_plain(amax):
    """The smallest number of 11 significant bits that is at least amax / 127 (and 2^-100), 0 for 0, NaN for infinity."""
    s = ((amax / 127).view(torch.int32) & ~0x1FFF).view(torch.float32)
    s = torch.where(s * 127 < amax, (s.view(torch.int32) + 0x2000).view(torch.float32), s)
    s = torch.where(amax > 0, s.clamp(min=2.0 ** -100), 0)
    return torch.where(torch.isfinite(amax), s, math.nan)


def append_plain(codes, scale, x, slots, block, keys_last):
    """Rows x [T, heads, dim] into a pool of codes (keys_last: the layout of v), in place."""
    dim = x.shape[-1]
    live = ((slots >= 0) & (slots < scale.shape[0] * block)).nonzero()[:, 0]
    slot, x = slots[live], x[live].float()
    blk, off = slot // block, slot % block
    most = x.abs().amax(-1)
    most = torch.where(torch.isfinite(most), most, math.inf)
    amax = torch.zeros_like(scale).scatter_reduce_(0, blk[:, None].expand_as(most), most, "amax")
    begun = torch.zeros_like(scale).index_fill_(0, blk[off == 0], 1) > 0
    old = torch.where(begun, 0, scale)
    grown = amax > 127 * old
    now = torch.where(grown, scale_plain(amax), old)
    touched = torch.bincount(blk, minlength=scale.shape[0]).nonzero()[:, 0]
    some = (slice(None), slice(None)) + (None,) * (codes.dim() - 2)
    held = codes[touched]
    again = (held.float() * old[touched][some] / now[touched][some]).round().nan_to_num().to(torch.int8)
    codes[touched] = torch.where(grown[touched][some], again, held)
    c = (x / now[blk][..., None]).round().nan_to_num().to(torch.int8)
    if keys_last:
        codes[blk, :, off // 16, :dim, off % 16] = c
    else:
        codes[blk, :, off, :dim] = c
    scale.copy_(now)


def read_plain(pool, slots, block, dtype):
    blk, off, d = slots // block, slots % block, pool["dim"]
    k = pool["k"][blk, :, off, :d].float() * pool["k_scale"][blk][..., None]
    v = pool["v"][blk, :, off // 16, :d, off % 16].float() * pool["v_scale"][blk][..., None]
    top = torch.finfo(dtype).max
    return k.clamp(-top, top).to(dtype), v.clamp(-top, top).to(dtype)


def _gathered(pool, table, real):
    """Keys and values [requests, kv heads, width * block, dim] of whole tables, and whether each page is there."""
    ids = table.long()
    there = (ids >= 0) & (ids < pool["k"].shape[0])
    ids = torch.where(there, ids, 0)
    R, W = ids.shape
    H, B, P = pool["k"].shape[1:]
    k = pool["k"][ids].to(real).mul_(pool["k_scale"][ids].to(real)[..., None, None])
    v = pool["v"][ids].to(real).mul_(pool["v_scale"][ids].to(real)[..., None, None, None])
    k = k.permute(0, 2, 1, 3, 4).reshape(R, H, W * B, P)[..., :pool["dim"]]
    v = v.permute(0, 2, 1, 3, 5, 4).reshape(R, H, W * B, P)[..., :pool["dim"]]
    return k, v, there.repeat_interleave(B, 1)


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


def sample_plain(logits, u, temperature, top_k, top_p, min_p):
    x = logits.double()
    B, V = x.shape
    column = lambda p: (p.double() if isinstance(p, torch.Tensor) else  # noqa: E731
                        torch.full((B,), float(np.float32(p)), dtype=torch.float64, device=x.device))[:, None]
    T, k, p, m = column(temperature), column(top_k), column(top_p), column(min_p)
    xs, order = x.sort(dim=-1, descending=True, stable=True)  # (ties: the lowest index first)
    top = xs[:, :1]
    w = torch.where(xs == top, 0, (xs - top) / torch.where(T > 0, T, 1)).exp()
    rank = torch.arange(V, device=x.device)
    w = torch.where((k <= 0) | (rank < k), w, 0)
    before = w.cumsum(-1)
    total = before[:, -1:].clone()
    before = torch.cat([torch.zeros_like(total), before[:, :-1]], -1)
    keep = ((p >= 1) | (before < p * total) | (rank == 0)) & (w >= m.clamp(max=1)) & (w > 0)
    kept = torch.zeros_like(x).scatter_(-1, order, torch.where(keep, w, 0))
    run_sum = kept.cumsum(-1)
    target = u.double().nan_to_num().clamp(0, 1 - 2.0 ** -24)[:, None] * run_sum[:, -1:]
    token = (run_sum <= target).sum(-1)
    token = torch.where(T[:, 0] > 0, token, order[:, 0])
    return torch.where(torch.isnan(x).any(-1) | (top[:, 0] == -math.inf), -1, token)


def run(state):
    kind = state["kind"]
    if own:
        import __graft_entry__

        hx = __graft_entry__.load_package()
        if kind == "plan":
            p = hx.kv_plan(state["lens"], state["new"], state["table"], state["free"], state["free_count"],
                           block_size=state["block"], tokens=state["tokens"])
            return dict(slots=p.slots, positions=p.positions, cu=p.cu, lens=p.lens, free_count=p.free_count,
                        table=state["table"])
        if kind == "sample":
            return hx.sample(state["logits"], state["u"], temperature=state["temperature"], top_k=state["top_k"],
                             top_p=state["top_p"], min_p=state["min_p"])
        c = state["pool"]
        cache = hx.KVCache(c["k"], c["v"], c["k_scale"], c["v_scale"], c["dim"])
        if kind == "append":
            hx.kv_append(cache, state["k"], state["v"], state["slots"])
            k, v = hx.kv_read(cache, state["back"], dtype=state["k"].dtype)
            return dict(k=k, v=v, k_scale=c["k_scale"], v_scale=c["v_scale"])
        return hx.kv_attention(state["q"], cache, state["table"], state["lens"], cu=state["cu"])
    if kind == "plan":
        slots, positions, cu, lens, count = plan_plain(state["lens"], state["new"], state["table"], state["free"],
                                                       state["free_count"], state["block"], state["tokens"])
        return dict(slots=slots, positions=positions, cu=cu, lens=lens, free_count=count, table=state["table"])
    if kind == "sample":
        return sample_plain(state["logits"], state["u"], state["temperature"], state["top_k"], state["top_p"],
                            state["min_p"])
    c = state["pool"]
    block = c["k"].shape[2]
    if kind == "append":
        append_plain(c["k"], c["k_scale"], state["k"], state["slots"], block, False)
        append_plain(c["v"], c["v_scale"], state["v"], state["slots"], block, True)
        k, v = read_plain(c, state["back"], block, state["k"].dtype)
        return dict(k=k, v=v, k_scale=c["k_scale"], v_scale=c["v_scale"])
    return attend_plain(state["q"], c, state["table"], state["lens"], state["cu"], state["most"])


def work(case):
    kind = case["kind"]
    if kind == "sample":
        n = case["rows"] * case["vocab"]
        return dict(bytes=n * SIZES[case["dtype"]] + case["rows"] * 28, flops=4 * n)
    held, new = _spans(case)
    R, block = case["requests"], case["block"]
    if kind == "plan":
        # lengths and new tokens in, lengths, offsets and what each row gets out, the table's new entries
        rows = min(case["tokens"], sum(max(n, 0) for n in new))
        taken = sum(-(-(h + max(n, 0)) // block) - -(-h // block) for h, n in zip(held, new))
        back = sum(-(-h // block) for h, n in zip(held, new) if n < 0)
        return dict(bytes=16 * R + 12 * case["tokens"] + 8 * (taken + back), flops=10 * R + 4 * rows)
    if kind == "append":
        # rows in, their codes out and read back with those of their blocks, the blocks that were begun read
        values = case["kv_heads"] * case["dim"] * 2
        back = sum(h % block + n for h, n in zip(held, new))
        begun = sum(h % block for h in held)
        return dict(bytes=values * (sum(new) * 3 + begun + back * 3), flops=values * (sum(new) * 4 + back))
    pairs = sum(n * h + n * (n + 1) // 2 for h, n in zip(held, new))
    keys = sum(h + n for h, n in zip(held, new))
    d = case["dim"]
    return dict(bytes=keys * case["kv_heads"] * 2 * d + sum(new) * case["heads"] * d * 4,
                flops=4 * pairs * case["heads"] * d)


# ---- the definitions, in 64 bits -----------------------------------------------------

def _exact_plan(s):
    lens, new, free = s["lens"].tolist(), s["new"].tolist(), s["free"].tolist()
    table, count, block, tokens = s["table"].cpu().numpy().copy(), int(s["free_count"]), s["block"], s["tokens"]
    stack = free[:count]
    held = [-(-n // block) for n in lens]
    for r, n in enumerate(new):
        if n < 0:
            stack += table[r, :held[r]].tolist()
    left, cu, slots, positions, after = len(stack), [0], [-1] * tokens, [0] * tokens, []
    for r, n in enumerate(new):
        cu.append(cu[-1] + max(n, 0))
        after.append(0 if n < 0 else lens[r])
        need = -(-(lens[r] + n) // block) - held[r]
        if n <= 0 or held[r] + need > table.shape[1] or cu[-1] > tokens:
            continue
        left -= need  # (what an earlier request waits for is not given to a later one)
        if need and left < 0:
            continue
        for j in range(need):
            table[r, held[r] + j] = stack.pop()
        after[r] = lens[r] + n
        for i in range(n):
            p = lens[r] + i
            slots[cu[r] + i], positions[cu[r] + i] = int(table[r, p // block]) * block + p % block, p
    one = lambda v, t=torch.int32: torch.tensor(v, dtype=t)  # noqa: E731
    return dict(slots=one(slots, torch.int64), positions=one(positions), cu=one(cu), lens=one(after),
                free_count=one([len(stack)]), table=torch.from_numpy(table))


def _exact_append(s):
    pool, out = s["pool"], {}
    block, d = pool["k"].shape[2], pool["dim"]
    slots, back = s["slots"], s["back"]
    for name, x in (("k", s["k"]), ("v", s["v"])):
        codes = pool[name].double()
        if name == "v":
            codes = codes.transpose(-1, -2).reshape(*pool["k"].shape)
        codes, scale = codes[..., :d].clone(), pool[name + "_scale"].double().clone()
        B, H = scale.shape
        cells = codes.transpose(1, 2).reshape(B * block, H, d)  # one row a slot
        x = x.double()
        a = torch.zeros((B * block, H), dtype=torch.float64, device=x.device)
        a[slots] = x.abs().amax(-1)
        a = a.view(B, block, H).amax(1)
        written = torch.zeros(B * block, dtype=torch.bool, device=x.device)
        written[slots] = True
        scale[written.view(B, block)[:, 0]] = 0
        # the smallest m * 2^e with 2^10 <= m <= 2^11 that is at least a / 127
        least = a / 127
        step = torch.exp2(torch.frexp(least)[1].double() - 11)
        fresh = torch.where(least > 0, torch.ceil(least / step) * step, 0)
        fresh = torch.where((fresh - step) * 127 >= a, fresh - step, fresh)
        now = torch.where(a > 127 * scale, fresh, scale)
        per = lambda t: t.repeat_interleave(block, 0)[..., None]  # noqa: E731
        moved = torch.where(per(a > 127 * scale), torch.round(cells * per(scale) / per(now)), cells)
        moved[slots] = torch.round(x / per(now)[slots]).nan_to_num()
        out[name] = (moved * per(now))[back]
        out[name + "_scale"] = now
    return out


def _exact_attend(s):
    q, pool, lens = s["q"], s["pool"], s["lens"].tolist()
    T, H, D = q.shape
    group = H // pool["k"].shape[1]
    cu = list(range(T + 1)) if s["cu"] is None else s["cu"].tolist()
    out = torch.zeros((T, H, D), dtype=torch.float64, device=q.device)
    for r, n in enumerate(lens):
        k, v, _ = _gathered(pool, s["table"][r:r + 1], torch.float64)
        x = q[cu[r]:cu[r + 1]].double().transpose(0, 1)  # [heads, rows, dim]
        rows = x.shape[1]
        hidden = torch.ones((rows, n), dtype=torch.bool, device=q.device).triu(n - rows + 1)
        for h in range(H):
            scores = (x[h] @ k[0, h // group, :n].T) / math.sqrt(D)
            p = scores.masked_fill_(hidden, -math.inf).softmax(-1)
            out[cu[r]:cu[r + 1], h] = p @ v[0, h // group, :n]
    return out


def _exact_sample(s):
    logits = s["logits"].float().cpu().numpy().astype(np.float64)
    B, V = logits.shape
    row = lambda p, r: float(p[r]) if isinstance(p, torch.Tensor) else float(np.float32(p))  # noqa: E731
    params = {n: s[n].cpu() if isinstance(s[n], torch.Tensor) else s[n] for n in
              ("temperature", "top_k", "top_p", "min_p")}
    u, tokens = s["u"].cpu(), []
    for r in range(B):
        T, k, p, m = (row(params[n], r) for n in ("temperature", "top_k", "top_p", "min_p"))
        x = logits[r]
        if T <= 0:
            tokens.append(int(np.argmax(x)))
            continue
        order = np.argsort(-x, kind="stable")[:int(k) if k > 0 else V]
        w = np.exp((x[order] - x.max()) / T)
        if p < 1:
            cum = np.concatenate([[0.0], np.cumsum(w)[:-1]])
            n = max(1, int(np.searchsorted(cum, p * w.sum(), side="left")))
            order, w = order[:n], w[:n]
        order, w = order[w >= min(m, 1.0)], w[w >= min(m, 1.0)]
        by_index = np.argsort(order)
        cum = np.cumsum(w[by_index])
        tokens.append(int(order[by_index][np.searchsorted(cum, float(u[r]) * cum[-1], side="right")]))
    return torch.tensor(tokens, dtype=torch.int64)


def exact(case, seed):
    s = prepare(case, seed)
    return dict(plan=_exact_plan, append=_exact_append, attend=_exact_attend, sample=_exact_sample)[case["kind"]](s)
