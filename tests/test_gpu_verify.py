"""Verification of drafted tokens on the GPU against the definition in 64 bits:
what is accepted, and what is drawn at the first row that is not, over settings,
types, ragged requests, masked and equal logits."""
import math

import numpy as np
import pytest
import torch

from gpu_util import gen, normal

pytestmark = pytest.mark.gpu


def target64(x, T, k, p, m):
    """Probabilities [vocab] of what the settings keep, or None for a row that gives nothing."""
    x = np.asarray(x, np.float64)
    if np.isnan(x).any() or x.max() == -math.inf:
        return None
    out = np.zeros(len(x))
    if not T > 0:
        out[int(np.argmax(x))] = 1
        return out
    with np.errstate(invalid="ignore"):
        w = np.where(x == x.max(), 1.0, np.exp((x - x.max()) / min(T, 1e28)))
    order = np.argsort(-x, kind="stable")[:k if 0 < k < len(x) else len(x)]
    wo = w[order]
    if p < 1:
        before = np.concatenate([[0.0], np.cumsum(wo)[:-1]])
        keep = before < p * wo.sum()
        keep[0] = True
        order, wo = order[keep], wo[keep]
    order, wo = order[wo >= min(m, 1.0)], wo[wo >= min(m, 1.0)]
    out[order] = wo / wo.sum()
    return out


def verify64(logits, drafts, u, draw, cu, probs, settings):
    """(tokens, counts) of whole lists; `near` counts decisions too close for 64 bits (there should be none)."""
    T, near = len(logits), 0
    tokens, counts = [-1] * T, []
    for r in range(len(draw)):
        n = 0
        for i in range(cu[r], cu[r + 1]):
            n += 1
            final, d = i + 1 == cu[r + 1], drafts[i]
            p = target64(logits[i], *(s[r] for s in settings))
            if p is None:
                break
            inside = not final and 0 <= d < len(p)
            if probs is None:
                q = np.zeros(len(p))
                if inside:
                    q[d] = 1
            else:
                q = np.nan_to_num(np.maximum(np.asarray(probs[i], np.float64), 0), nan=0.0, posinf=math.inf)
            if inside:
                a, b = p[d], float(np.clip(np.nan_to_num(u[i]), 0, 1 - 2.0 ** -24)) * (q[d] if q[d] < math.inf else 1e300)
                near += a != b and abs(a - b) < 1e-12 * max(a, b)
                if a > b:
                    tokens[i] = d
                    continue
            left = p if final else np.maximum(p - q, 0)
            left = left if left.sum() > 0 else p
            cum = np.cumsum(left)
            at = float(np.clip(np.nan_to_num(draw[r]), 0, 1 - 2.0 ** -24)) * cum[-1]
            near += np.abs(cum - at).min() < 1e-13 * cum[-1] and at > 0
            tokens[i] = int(np.searchsorted(cum, at, side="right"))
            break
        counts.append(n)
    return tokens, counts, near


def check(pkg, dev, logits, drafts, u, draw, cu=None, probs=None, name="", **kw):
    """logits etc. on the CPU, flat rows; cu a list (None: equal rows)."""
    R, V = len(draw), logits.shape[-1]
    T = logits.numel() // V
    bounds = cu if cu is not None else [i * (T // R) for i in range(R + 1)]
    settings = []
    for s, neutral in (("temperature", 1.0), ("top_k", 0), ("top_p", 1.0), ("min_p", 0.0)):
        v = kw.get(s, neutral)
        settings.append([float(np.float32(y)) if s != "top_k" else int(y) for y in (v.tolist() if isinstance(v, torch.Tensor) else [v] * R)])
    want = verify64(logits.reshape(T, V).double().numpy(), drafts.reshape(T).tolist(), u.reshape(T).tolist(), draw.tolist(),
                    bounds, None if probs is None else probs.reshape(T, V).double().numpy(), settings)
    assert want[2] == 0, name
    to = lambda t: t.to(dev) if isinstance(t, torch.Tensor) else t  # noqa: E731
    got = pkg.verify(to(logits), to(drafts), to(u), to(draw), cu=None if cu is None else torch.tensor(cu, dtype=torch.int32, device=dev),
                     draft_probs=to(probs), **{n: to(v) for n, v in kw.items()})
    assert got.tokens.shape == drafts.shape and got.counts.dtype == torch.int32
    assert got.tokens.reshape(-1).tolist() == want[0], name
    assert got.counts.tolist() == want[1], name
    return got


def drafted(V, rows, seed, dtype, probs_dtype, std=2.5, noise=0.5):
    """(logits, drafts, u, probs): a draft's distribution near the target's, its tokens drawn from it."""
    g = gen(seed)
    x = torch.randn((rows, V), generator=g) * std
    y = (x + noise * torch.randn((rows, V), generator=g)).softmax(-1)
    d = torch.multinomial(y, 1, generator=g)[:, 0]
    return x.to(dtype), d, torch.rand(rows, generator=g), y.to(probs_dtype)


SETTINGS = [{}, dict(temperature=0.7), dict(top_k=5), dict(top_p=0.8), dict(min_p=0.05), dict(temperature=0.0),
            dict(temperature=1.3, top_k=40, top_p=0.9, min_p=0.01), dict(top_k=1), dict(top_k=600, top_p=0.99)]


@pytest.mark.parametrize("dtype, probs_dtype", [(torch.float16, torch.float32), (torch.bfloat16, torch.bfloat16),
                                                (torch.float32, torch.float16), (torch.float32, torch.float32)])
@pytest.mark.parametrize("vocab", [1, 2, 9, 511, 512, 513, 1000, 8191, 33001])
def test_verify(pkg, dev, dtype, probs_dtype, vocab):
    rows = [3, 1, 0, 5, 2, 4]
    cu = [0] + np.cumsum(rows).tolist()
    T = cu[-1] + 2  # two rows of no request
    logits, drafts, u, probs = drafted(vocab, T, vocab, dtype, probs_dtype)
    draw = torch.rand(len(rows), generator=gen(vocab + 1))
    for i, kw in enumerate(SETTINGS):
        check(pkg, dev, logits, drafts, u, draw, cu, probs, (i, "probs"), **kw)
        check(pkg, dev, logits, drafts, u, draw, cu, None, (i, "certain"), **kw)
    T = 12
    shape = lambda t: t[:T].reshape(4, 3, *t.shape[1:])  # noqa: E731
    got = check(pkg, dev, shape(logits), shape(drafts), shape(u), draw[:4], None, shape(probs), "equal rows", top_k=20)
    assert got.tokens.shape == (4, 3)


@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16, torch.float32])
def test_verify_accepts_and_refuses_all(pkg, dev, dtype):
    """The draft's distribution the target's own: every token that has a weight
    is accepted; one that has none: none is."""
    V, rows = 3000, 8
    x, _, u, _ = drafted(V, rows, 5, dtype, torch.float32)
    q = x.double().softmax(-1)
    d = q.argmax(-1)
    under = (q * (1 - 1e-6)).float()
    got = check(pkg, dev, x.view(2, 4, V), d.view(2, 4), u.view(2, 4), torch.tensor([0.3, 0.9]), None, under.view(2, 4, V), "own")
    assert got.counts.tolist() == [4, 4]
    d[1:3] = torch.tensor([-1, V])  # outside the vocabulary
    got = check(pkg, dev, x.view(2, 4, V), d.view(2, 4), u.view(2, 4), torch.tensor([0.3, 0.9]), None, under.view(2, 4, V), "out")
    assert got.counts.tolist() == [2, 4]
    got = check(pkg, dev, x.view(2, 4, V), d.view(2, 4), torch.zeros(2, 4), torch.tensor([0.3, 0.9]), None, None, "out, certain")
    assert got.counts.tolist() == [2, 4]
    low = x.double().argmin(-1)  # a token that top_k leaves out
    got = check(pkg, dev, x.view(2, 4, V), low.view(2, 4), u.view(2, 4), torch.tensor([0.0, 0.999]), None, None, "low", top_k=10)
    assert got.counts.tolist() == [1, 1]
    # a draft that covers all the target keeps (probabilities that do not sum to 1): drawn from p
    huge = torch.full((2, 4, V), 2.0)
    huge[0, 0, 7], huge[1, 0] = math.inf, math.inf
    got = check(pkg, dev, x.view(2, 4, V), low.view(2, 4), u.view(2, 4), torch.tensor([0.4, 0.6]), None, huge, "covered")
    assert got.counts.tolist() == [1, 1]


@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16, torch.float32])
def test_verify_of_masked_and_equal_logits(pkg, dev, dtype):
    """Equal logits on the threshold (the lowest indices stay), masks, infinities, NaN."""
    V, R, S = 2100, 9, 3
    g = gen(31)
    x = (torch.randn((R * S, V), generator=g) * 2).round() / 2  # many equals
    x[3] = 0.0
    x[4, 100:] = -math.inf
    x[5] = torch.finfo(dtype).min
    x[5, 700] = 1.0
    x[6, 2000] = math.nan
    x[10] = -math.inf
    x[12, 50], x[12, 60] = math.inf, math.inf
    x[20] = 3.0
    x = x.to(dtype)
    q = (x.double().nan_to_num(0, 3, -40) * 0.9).softmax(-1).float()
    q[7, :500], q[8, 3] = math.nan, -5.0
    u, draw = torch.rand(R * S, generator=g) * 0.8, torch.rand(R, generator=g)
    for seed in range(3):
        d = torch.stack([torch.topk(x[i].double().nan_to_num(-1e9), 300)[1][int(torch.randint(0, 300, (1,), generator=g))] for i in range(R * S)])
        for i, kw in enumerate((dict(), dict(top_k=7), dict(top_k=1500), dict(top_p=0.6), dict(top_k=90, top_p=0.7), dict(temperature=0.0),
                                dict(min_p=0.3))):
            shaped = x.view(R, S, V), d.view(R, S), u.view(R, S), draw
            check(pkg, dev, *shaped, None, q.view(R, S, V), (seed, i), **kw)
            check(pkg, dev, *shaped, None, None, (seed, i, "certain"), **kw)


def test_verify_of_a_large_vocabulary_with_own_settings(pkg, dev):
    V, rows = 151936, [1, 4, 5, 2, 3, 5]
    cu = [0] + np.cumsum(rows).tolist()
    g = gen(41)
    own = dict(temperature=torch.tensor([1.0, 0.0, 0.8, 1.2, 0.7, 1.0]), top_k=torch.tensor([0, 0, 50, 400, 5000, 0], dtype=torch.int32),
               top_p=torch.tensor([1.0, 0.9, 0.95, 1.0, 0.9, 0.9]), min_p=torch.tensor([0.0, 0.0, 0.01, 0.0, 0.0, 0.2]))
    for dtype, pt in ((torch.bfloat16, torch.float32), (torch.float32, torch.bfloat16), (torch.float16, torch.float16)):
        logits, drafts, u, probs = drafted(V, cu[-1], 42, dtype, pt, noise=0.3)
        draw = torch.rand(6, generator=g)
        check(pkg, dev, logits, drafts, u, draw, cu, probs, dtype, **own)
        check(pkg, dev, logits, drafts, u, draw, cu, None, dtype, **own)
        check(pkg, dev, logits, drafts, u, draw, cu, probs, dtype)


def test_verify_at_extreme_numbers(pkg, dev):
    """u and draw at and past the ends of [0, 1), NaN among them; temperatures that leave one or all alike."""
    V = 700
    logits, drafts, _, probs = drafted(V, 12, 51, torch.float32, torch.float32)
    u = torch.tensor([0.0, 1.0, -3.0, math.nan, 7.0, 1 - 2.0 ** -24, 0.0, 0.5, 0.5, math.inf, -0.0, 0.2])
    for draw in ([0.0, 1.0, math.nan, -1.0], [1 - 2.0 ** -24, 5.0, 0.0, math.inf]):
        for T in (1e-12, 1e6, 1e30):
            for q in (probs, None):
                check(pkg, dev, logits.view(4, 3, V), drafts.view(4, 3), u.view(4, 3), torch.tensor(draw), None,
                      None if q is None else q.view(4, 3, V), (draw, T), temperature=T)


def test_verify_distribution(pkg, dev):
    """What comes out first is distributed as the target: 20000 drafts of one
    token against its own probabilities (chi-squared, 15 degrees of freedom)."""
    V, n = 16, 20000
    g = gen(61)
    x, y = torch.randn(V, generator=g), torch.randn(V, generator=g)
    p, q = x.double().softmax(-1), y.double().softmax(-1)
    d = torch.multinomial(q.expand(n, V), 1, generator=g)
    drafts = torch.cat([d, torch.zeros_like(d)], 1)
    got = pkg.verify(x.to(dev).expand(n, 2, V), drafts.to(dev), torch.rand((n, 2), generator=g).to(dev), torch.rand(n, generator=g).to(dev),
                     draft_probs=q.float().to(dev).expand(n, 2, V))
    seen = torch.bincount(got.tokens[:, 0].cpu(), minlength=V).double()
    # mean 15, standard deviation 5.5: 60 lies eight of them out (one in 10^6 by chance), and the numbers are fixed
    assert ((seen - n * p) ** 2 / (n * p)).sum() < 60
    assert (got.counts == 2).float().mean() > 0.3


def test_verify_takes_views_and_nothing(pkg, dev):
    V = 600
    logits, drafts, u, probs = drafted(V, 9, 71, torch.bfloat16, torch.float32)
    cu, draw = [0, 4, 9], torch.tensor([0.2, 0.7])
    want = check(pkg, dev, logits, drafts, u, draw, cu, probs)
    c = torch.tensor(cu, dtype=torch.int32, device=dev)
    wide = torch.zeros((9, V + 37), dtype=logits.dtype, device=dev)
    wide[:, 5:5 + V] = logits.to(dev)
    q = torch.zeros((9, 2 * V), device=dev)
    q[:, ::2] = probs.to(dev)
    views = dict(logits=wide[:, 5:5 + V], drafts=drafts.to(dev).repeat_interleave(2)[::2], u=u.to(dev).repeat_interleave(3)[::3],
                 draw=draw.to(dev).repeat_interleave(2)[::2], cu=c.repeat_interleave(2)[::2], draft_probs=q[:, ::2])
    got = pkg.verify(**views)
    assert torch.equal(got.tokens, want.tokens) and torch.equal(got.counts, want.counts)
    turned = logits.t().contiguous().t()
    got = pkg.verify(turned.to(dev), drafts.to(dev), u.to(dev), draw.to(dev), cu=c, draft_probs=probs.to(dev))
    assert torch.equal(got.tokens, want.tokens)
    same = pkg.verify(logits[:1].to(dev).expand(9, V), drafts.to(dev), u.to(dev), draw.to(dev), cu=c)  # one row for all
    again = pkg.verify(logits[:1].to(dev).repeat(9, 1), drafts.to(dev), u.to(dev), draw.to(dev), cu=c)
    assert torch.equal(same.tokens, again.tokens)
    none = pkg.verify(logits.to(dev)[:0], drafts.to(dev)[:0], u.to(dev)[:0], draw.to(dev), cu=torch.zeros_like(c))
    assert none.counts.tolist() == [0, 0] and none.tokens.numel() == 0
    none = pkg.verify(logits.to(dev), drafts.to(dev), u.to(dev), draw.to(dev), cu=torch.zeros_like(c))  # rows of no request
    assert none.counts.tolist() == [0, 0] and none.tokens.tolist() == [-1] * 9
    past = pkg.verify(logits.to(dev), drafts.to(dev), u.to(dev), draw.to(dev), cu=torch.tensor([-3, 4, 999], dtype=torch.int32, device=dev),
                      draft_probs=probs.to(dev))  # bounds past the rows: the rows there are
    assert torch.equal(past.tokens, want.tokens) and torch.equal(past.counts, want.counts)


def verify_calls(pkg, dev):
    V = 900
    logits, drafts, u, probs = (t.to(dev) for t in drafted(V, 8, 81, torch.float16, torch.float32))
    cu, draw = torch.tensor([0, 3, 8], dtype=torch.int32, device=dev), torch.tensor([0.1, 0.6], device=dev)
    k = torch.tensor([4, 70], dtype=torch.int32, device=dev)
    return [
        ("ragged", True, lambda: pkg.verify(logits, drafts, u, draw, cu=cu, draft_probs=probs, top_p=0.9)),
        ("certain", True, lambda: pkg.verify(logits, drafts, u, draw, cu=cu, top_k=k)),
        ("equal rows", True, lambda: pkg.verify(logits.view(2, 4, V), drafts.view(2, 4), u.view(2, 4), draw, temperature=2)),
        ("columns", True, lambda: pkg.verify(logits[:, 3:700], drafts.clamp(max=696), u, draw, cu=cu, draft_probs=probs[:, 3:700])),
        ("strided u", False, lambda: pkg.verify(logits, drafts, u.repeat_interleave(2)[::2], draw, cu=cu)),
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

    for name, native, call in verify_calls(pkg, dev):
        monkeypatch.setattr(pkg.hxmi, "_ops", Spy())
        taken.clear()
        got = call()
        assert taken[0] == native, name
        monkeypatch.setattr(pkg.hxmi, "_ops", pkg.hxmi._PythonForms())
        want = call()
        assert all(torch.equal(a, b) for a, b in zip(got, want)), name


def test_verify_on_two_streams_and_in_graphs(pkg, dev):
    calls = verify_calls(pkg, dev)
    want = [[t.clone() for t in call()] for _, _, call in calls]
    streams = [torch.cuda.Stream() for _ in range(2)]
    torch.cuda.synchronize()
    got = [[], []]
    for _ in range(10):
        for i, s in enumerate(streams):
            with torch.cuda.stream(s):
                got[i].append(calls[i][2]())
    torch.cuda.synchronize()
    assert all(torch.equal(a, b) for i in range(2) for g in got[i] for a, b in zip(g, want[i]))
    graphs, outs = [], []
    for _, _, call in calls[:2]:
        graphs.append(torch.cuda.CUDAGraph())
        with torch.cuda.graph(graphs[-1]):
            outs.append(call())
    for i in range(5):
        for o in outs:
            o.tokens.fill_(-9)
        torch.cuda.synchronize()
        for g, s in zip(graphs, streams):
            with torch.cuda.stream(s if i % 2 else streams[0]):
                g.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for o, w in zip(outs, want) for a, b in zip(o, w)), i
        assert torch.equal(calls[0][2]().tokens, want[0][0])


def test_verify_refuses(pkg, dev):
    x, d, u, draw = torch.zeros((2, 3, 50), device=dev), torch.zeros((2, 3), dtype=torch.int64, device=dev), torch.zeros((2, 3), device=dev), torch.zeros(2, device=dev)
    cu, hx = torch.tensor([0, 3, 6], dtype=torch.int32, device=dev), pkg
    bad = [
        ("logits", lambda: hx.verify(x.double(), d, u, draw)), ("vocab", lambda: hx.verify(x[0], d[0], u[0], draw)),
        ("vocab", lambda: hx.verify(x, d, u, draw, cu=cu)), ("draw", lambda: hx.verify(x, d, u, draw[:1])),
        ("draw", lambda: hx.verify(x, d, u, draw.double())), ("draw", lambda: hx.verify(x, d, u, draw.view(2, 1))),
        ("drafts", lambda: hx.verify(x, d.int(), u, draw)), ("drafts", lambda: hx.verify(x, d[:, :2], u, draw)),
        ("u must", lambda: hx.verify(x, d, u[:, :2], draw)), ("u must", lambda: hx.verify(x, d, u.half(), draw)),
        ("cu", lambda: hx.verify(x.view(6, 50), d.view(6), u.view(6), draw, cu=cu[:2])),
        ("cu", lambda: hx.verify(x.view(6, 50), d.view(6), u.view(6), draw, cu=cu.long())),
        ("draft_probs", lambda: hx.verify(x, d, u, draw, draft_probs=x[:, :2])),
        ("draft_probs", lambda: hx.verify(x, d, u, draw, draft_probs=x.double())),
        ("temperature", lambda: hx.verify(x, d, u, draw, temperature=-1)), ("temperature", lambda: hx.verify(x, d, u, draw, temperature=u)),
        ("top_k", lambda: hx.verify(x, d, u, draw, top_k=draw)), ("top_p", lambda: hx.verify(x, d, u, draw, top_p=math.nan)),
        ("min_p", lambda: hx.verify(x, d, u, draw, min_p=draw[:1])), ("vocab", lambda: hx.verify(x[..., :0], d, u, draw)),
        ("without a request", lambda: hx.verify(x.view(6, 50), d.view(6), u.view(6), draw[:0], cu=cu[:1])),
        ("GPU", lambda: hx.verify(x, d.cpu(), u, draw)),
    ]
    for i, (msg, call) in enumerate(bad):
        with pytest.raises(pkg.HxmiError, match=msg):
            call()
            pytest.fail(f"call {i} ({msg}) was taken")
