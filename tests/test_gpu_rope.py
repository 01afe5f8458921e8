"""qk_rope on the GPU: norms of queries and keys by head and their rotation,
against the definition in 64 bits, over types, layouts, axes, positions and
views."""
import math

import pytest
import torch

from gpu_util import gen, normal

pytestmark = pytest.mark.gpu

HALF = {torch.float16: 2.0 ** -11, torch.bfloat16: 2.0 ** -8}  # half a step of the type, relative


def rope64(x, pos, freq, axis, scale, weight, eps, interleaved):
    """The definition; and what its roundings in 32 bits can move a value by."""
    x, n = x.cpu().double(), freq.numel()
    size = x.abs()
    if weight is not None:
        f = weight.cpu().double() / (x.pow(2).mean(-1, keepdim=True) + eps).sqrt()
        x, size = x * f, size * f.abs()
    pos = pos.cpu().double()
    at = pos[:, None].expand(-1, n) if pos.dim() == 1 else pos[axis.cpu().long() if axis is not None else [0] * n].T
    t = at * freq.cpu().double()
    c, s = scale * t.cos()[:, None], scale * t.sin()[:, None]
    y, room = x.clone(), size.clone()
    a, b = (slice(0, 2 * n, 2), slice(1, 2 * n, 2)) if interleaved else (slice(0, n), slice(n, 2 * n))
    y[..., a] = x[..., a] * c - x[..., b] * s
    y[..., b] = x[..., b] * c + x[..., a] * s
    room[..., a] = room[..., b] = (size[..., a] + size[..., b]) * abs(scale)
    # a product, a sum, a cosine and the norm's factors: some ten roundings of 2^-24; the angle,
    # in 64 bits on both sides, is off by 2^-52 of its turns
    return y, room * (2.0 ** -20 + t.abs().max() * 2.0 ** -50 if n else 2.0 ** -20)


def check(got, x, pos, freq, axis=None, scale=1.0, weight=None, eps=1e-6, interleaved=False, name=""):
    want, room = rope64(x, pos, freq, axis, scale, weight, eps, interleaved)
    assert got.shape == x.shape and got.dtype == x.dtype, name
    # (2^-25: half a step of fp16 below its normal range)
    off = (got.cpu().double() - want).abs() - HALF[x.dtype] * want.abs() * (1 + 2.0 ** -10) - room - 2.0 ** -25
    assert off.max() <= 0, (name, float(off.max()))


def rows(shape, seed, dtype, dev):
    return normal(shape, seed, 1.0, dtype=dtype).to(dev)


SHAPES = [  # tokens, heads, kv heads, head dim, rotary dim, dtype
    (1, 32, 4, 64, 64, torch.float16), (3, 14, 2, 64, 64, torch.bfloat16), (70, 32, 8, 128, 128, torch.float16),
    (1100, 5, 1, 128, 64, torch.bfloat16), (9, 3, 3, 40, 10, torch.float16), (33, 2, 1, 40, 20, torch.bfloat16),
    (17, 4, 2, 80, 32, torch.float16), (5, 8, 2, 256, 256, torch.bfloat16), (6, 1, 1, 256, 2, torch.float16),
    (2, 3, 1, 8, 8, torch.float16), (4, 2, 2, 24, 0, torch.bfloat16), (8, 25, 5, 40, 40, torch.float16),
    (2050, 2, 1, 16, 16, torch.bfloat16), (12, 7, 1, 96, 96, torch.float16), (3, 1, 1, 248, 240, torch.float16),
]


@pytest.mark.parametrize("interleaved", [False, True])
@pytest.mark.parametrize("T, H, K, d, rotary, dtype", SHAPES)
def test_rope(pkg, dev, T, H, K, d, rotary, dtype, interleaved):
    q, k = rows((T, H, d), 1, dtype, dev), rows((T, K, d), 2, dtype, dev)
    pos = torch.randint(0, 9000, (T,), generator=gen(3)).to(dev)
    freq, _ = pkg.rope_frequencies(rotary, 1e4, device=dev)
    w = normal((d,), 4, 0.5, dtype=dtype).to(dev) + 1
    for weights in ((None, None), (w, w.flip(0)), (w.float(), None), (None, w.float()), (w, w.float())):
        a, b = pkg.qk_rope(q, k, pos.int(), freq, q_weight=weights[0], k_weight=weights[1], eps=1e-5, interleaved=interleaved)
        check(a, q, pos, freq, weight=weights[0], eps=1e-5, interleaved=interleaved, name="q")
        check(b, k, pos, freq, weight=weights[1], eps=1e-5, interleaved=interleaved, name="k")
    a, b = pkg.qk_rope(q, None, pos, freq, interleaved=interleaved)
    assert b is None
    check(a, q, pos, freq, interleaved=interleaved)


@pytest.mark.parametrize("interleaved", [False, True])
@pytest.mark.parametrize("T, H, K, d, sections, dtype", [
    (50, 4, 2, 64, (8, 12, 12), torch.float16), (1300, 14, 2, 64, (16, 0, 16), torch.bfloat16),
    (7, 2, 1, 128, (64,), torch.float16), (9, 2, 1, 40, (5, 7, 3), torch.bfloat16),
])
def test_rope_of_several_axes(pkg, dev, T, H, K, d, sections, dtype, interleaved):
    q, k = rows((T, H, d), 11, dtype, dev), rows((T, K, d), 12, dtype, dev)
    pos = torch.randint(0, 5000, (len(sections), T), generator=gen(13), dtype=torch.int32).to(dev)
    freq, axis = pkg.rope_frequencies(2 * sum(sections), 1e6, sections=sections, device=dev)
    assert axis.tolist() == [i for i, n in enumerate(sections) for _ in range(n)]
    order = torch.randperm(len(axis), generator=gen(14)).to(dev)
    for ax in (axis, axis[order]):
        for p in (pos, pos.long(), torch.cat([pos, pos], 1)[:, T // 2:T // 2 + T]):
            a, b = pkg.qk_rope(q, k, p, freq, axis=ax, interleaved=interleaved)
            check(a, q, p, freq, ax, interleaved=interleaved, name="q")
            check(b, k, p, freq, ax, interleaved=interleaved, name="k")
    far = axis.clone()
    far[0], far[-1] = -3, 99  # the nearest axis there is
    near = far.clamp(0, len(sections) - 1)
    got = pkg.qk_rope(q, k, pos, freq, axis=far, interleaved=interleaved)
    want = pkg.qk_rope(q, k, pos, freq, axis=near, interleaved=interleaved)
    assert all(torch.equal(a, b) for a, b in zip(got, want))


def test_rope_at_far_positions(pkg, dev):
    """Angles of 2^31 turns and more, and before the first token; any scale."""
    q, k = rows((8, 3, 64), 21, torch.float16, dev), rows((8, 1, 64), 22, torch.float16, dev)
    pos = torch.tensor([0, -1, -131072, 1 << 20, (1 << 24) + 1, (1 << 31) - 1, -(1 << 31), 1 << 40], device=dev)
    freq, _ = pkg.rope_frequencies(64, 5e5, device=dev)
    for scale in (1.0, 0.5, -1.25, 0.0):
        a, b = pkg.qk_rope(q[:7], k[:7], pos[:7].int() if scale == 0.5 else pos[:7], freq, scale=scale)
        check(a, q[:7], pos[:7], freq, scale=scale, name=scale)
        check(b, k[:7], pos[:7], freq, scale=scale, name=scale)
    a, _ = pkg.qk_rope(q[7:], None, pos[7:], freq * 2.0 ** -12)
    check(a, q[7:], pos[7:], freq * 2.0 ** -12)


def test_rope_of_special_values(pkg, dev):
    """Infinities and NaN stay in their own head; zeros and the largest values."""
    q = rows((3, 4, 64), 31, torch.bfloat16, dev)
    q[0, 1, 5], q[1, 2, 40], q[2, 3] = math.nan, math.inf, 0
    freq, _ = pkg.rope_frequencies(64, device=dev)
    pos, w = torch.arange(3, device=dev) + 7, torch.ones(64, device=dev)
    for weight in (None, w):
        a, _ = pkg.qk_rope(q, None, pos, freq, q_weight=weight)
        bad = (~torch.isfinite(a)).flatten(2).any(-1).tolist()
        assert bad == [[False, True, False, False], [False, False, True, False], [False] * 4]
        assert not a[2, 3].any()
    x = torch.full((1, 1, 64), 65504.0, dtype=torch.float16, device=dev)
    a, _ = pkg.qk_rope(x, None, pos[:1], freq, q_weight=w)  # (mean of squares 2^32)
    check(a, x, pos[:1], freq, weight=w)


def test_rope_of_views_and_into_any_rows(pkg, dev):
    """q and k of one projection at any offset; out in other rows, in place,
    and over elements that are read."""
    T, H, K, d = 37, 6, 2, 64
    freq, _ = pkg.rope_frequencies(48, device=dev)
    pos = torch.arange(T, device=dev, dtype=torch.int32) * 3
    buf = rows((T, 1 + (H + 2 * K) * d), 41, torch.float16, dev)
    for interleaved in (False, True):
        for rotary in (48, 44):  # (whole chunks of pairs, and not)
            f = freq[:rotary // 2].contiguous()
            x = buf.clone()
            qkv = x[:, 1:].view(T, H + 2 * K, d)
            q, k = qkv[:, :H], qkv[:, H:H + K]
            wq, wk = pkg.qk_rope(q, k, pos, f, interleaved=interleaved)
            check(wq, q, pos, f, interleaved=interleaved)
            check(wk, k, pos, f, interleaved=interleaved)
            assert torch.equal(x, buf)
            t = q.transpose(0, 1).contiguous().transpose(0, 1)  # heads first
            assert torch.equal(pkg.qk_rope(t, None, pos, f, interleaved=interleaved)[0], wq)
            t = q.transpose(1, 2).contiguous().transpose(1, 2)  # last stride not 1
            assert torch.equal(pkg.qk_rope(t, k, pos, f, interleaved=interleaved)[0], wq)
            oq = torch.zeros((H, T, d + 3), dtype=q.dtype, device=dev)[..., 3:].transpose(0, 1)
            ok = torch.zeros((T, K, 2 * d), dtype=q.dtype, device=dev)[..., ::2]
            got = pkg.qk_rope(q, k, pos, f, interleaved=interleaved, out=(oq, ok))
            assert got[0] is oq and got[1] is ok and torch.equal(oq, wq) and torch.equal(ok, wk)
            got = pkg.qk_rope(q, k, pos, f, interleaved=interleaved, out=(q, k))  # in place
            assert got[0] is q and torch.equal(q, wq) and torch.equal(k, wk)
            rest = buf[:, 1:].view(T, H + 2 * K, d)[:, H + K:]
            assert torch.equal(qkv[:, H + K:], rest) and torch.equal(x[:, 0], buf[:, 0])  # nothing else
            x.copy_(buf)
            oq = x[:, 9:9 + H * d].view(T, H, d)  # over other elements of q
            assert torch.equal(pkg.qk_rope(q, k, pos, f, interleaved=interleaved, out=(oq, torch.empty_like(wk)))[0], wq)
            x.copy_(buf)
            ok = qkv[:, 1:1 + K]  # k's result over q
            got = pkg.qk_rope(q, k, pos, f, interleaved=interleaved, out=(torch.empty_like(wq), ok))
            assert torch.equal(got[0], wq) and torch.equal(ok, wk)


def test_rope_without_tokens_or_heads(pkg, dev):
    freq, _ = pkg.rope_frequencies(64, device=dev)
    none = torch.zeros(0, dtype=torch.int32, device=dev)
    q, k = (torch.zeros((0, h, 64), dtype=torch.float16, device=dev) for h in (4, 2))
    a, b = pkg.qk_rope(q, k, none, freq)
    assert a.shape == q.shape and b.shape == k.shape
    pkg.qk_rope(q, k, none, freq, out=(q, k))
    x, pos = torch.ones((3, 0, 64), dtype=torch.float16, device=dev), torch.zeros(3, dtype=torch.int32, device=dev)
    z = rows((3, 2, 64), 51, torch.float16, dev)
    a, b = pkg.qk_rope(x, z, pos, freq)
    assert a.shape == x.shape and torch.equal(b, z)  # position 0: as they are


def rope_calls(pkg, dev):
    """(name, whether the native entry takes it, call)"""
    T, H, K, d = 19, 8, 2, 64
    freq, axis = pkg.rope_frequencies(d, sections=(10, 12, 10), device=dev)
    qkv = rows((T, H + 2 * K, d), 61, torch.bfloat16, dev)
    pos = torch.randint(0, 4000, (3, T), generator=gen(62), dtype=torch.int32).to(dev)
    w = normal((d,), 63, dtype=torch.bfloat16).to(dev)

    def place(interleaved=False, **kw):
        x = qkv.clone()
        pkg.qk_rope(x[:, :H], x[:, H:H + K], pos[0], freq, interleaved=interleaved, out=(x[:, :H], x[:, H:H + K]), **kw)
        return (x,)

    q, k = qkv[:, :H], qkv[:, H:H + K]
    return [
        ("plain", True, lambda: pkg.qk_rope(q, k, pos[0], freq)),
        ("norms", True, lambda: pkg.qk_rope(q, k, pos[0], freq, q_weight=w, k_weight=w, scale=1, eps=0)),
        ("axes", True, lambda: pkg.qk_rope(q, k, pos, freq, axis=axis, interleaved=True)),
        ("one axis", True, lambda: pkg.qk_rope(q, k, pos[:1], freq)),
        ("no k", True, lambda: pkg.qk_rope(q, None, pos[0].long(), freq)[:1]),
        ("in place", True, place),
        ("in place, norms", True, lambda: place(q_weight=w)),
        ("mixed weights", False, lambda: pkg.qk_rope(q, k, pos[0], freq, q_weight=w, k_weight=w.float())),
        ("strided positions", False, lambda: pkg.qk_rope(q, k, pos[0].repeat_interleave(2)[::2], freq)),
        ("apart rows of positions", False, lambda: pkg.qk_rope(q[:5], k[:5], pos[:, 2:7], freq, axis=axis)),
        ("other rows", False, lambda: pkg.qk_rope(q, k, pos[0], freq, out=(torch.empty_like(q), torch.empty_like(k)))),
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

    for name, native, call in rope_calls(pkg, dev):
        monkeypatch.setattr(pkg.hxmi, "_ops", Spy())
        taken.clear()
        got = call()
        assert taken[0] == native, name
        monkeypatch.setattr(pkg.hxmi, "_ops", pkg.hxmi._PythonForms())
        want = call()
        assert len(got) == len(want) and all(torch.equal(a, b) for a, b in zip(got, want)), name


def test_rope_on_another_stream_and_in_a_graph(pkg, dev):
    want = [[t.clone() for t in call()] for _, _, call in rope_calls(pkg, dev)]
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        for (name, _, call), w in zip(rope_calls(pkg, dev), want):
            got = call()
            s.synchronize()
            assert all(torch.equal(a, b) for a, b in zip(got, w)), name
    freq, _ = pkg.rope_frequencies(64, device=dev)
    q, k = rows((5, 4, 64), 71, torch.float16, dev), rows((5, 1, 64), 72, torch.float16, dev)
    pos = torch.zeros(5, dtype=torch.int32, device=dev)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = pkg.qk_rope(q, k, pos, freq)
    for i in range(4):
        pos.fill_(1 + 10 * i)
        graph.replay()
        eager = pkg.qk_rope(q, k, pos, freq)
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(out, eager)), i


def test_rope_refuses(pkg, dev):
    q, k = rows((3, 4, 64), 81, torch.float16, dev), rows((3, 2, 64), 82, torch.float16, dev)
    pos, (freq, axis) = torch.zeros(3, dtype=torch.int32, device=dev), pkg.rope_frequencies(64, sections=(16, 16), device=dev)
    w, two = torch.ones(64, device=dev), torch.zeros((2, 3), dtype=torch.int32, device=dev)
    x = rows((3, 6, 64), 83, torch.float16, dev)
    hx = pkg
    bad = [
        ("fp16 or bf16", lambda: hx.qk_rope(q.float(), k.float(), pos, freq)),
        ("fp16 or bf16", lambda: hx.qk_rope(q, k.float(), pos, freq)),
        ("k must", lambda: hx.qk_rope(q, k.bfloat16(), pos, freq)), ("k must", lambda: hx.qk_rope(q, k[:2], pos, freq)),
        ("k must", lambda: hx.qk_rope(q, k[..., :32], pos, freq)),
        ("heads, head_dim", lambda: hx.qk_rope(q.view(3, 256), None, pos, freq)),
        ("multiple of 8", lambda: hx.qk_rope(q[..., :60], None, pos, freq[:30])),
        ("up to 256", lambda: hx.qk_rope(q.view(3, 1, 256).repeat(1, 1, 2), None, pos, freq)),
        ("do not fit", lambda: hx.qk_rope(q[..., :32], None, pos, freq)),
        ("float64", lambda: hx.qk_rope(q, k, pos, freq.float())), ("float64", lambda: hx.qk_rope(q, k, pos, freq.view(2, -1))),
        ("positions", lambda: hx.qk_rope(q, k, pos.float(), freq)), ("positions", lambda: hx.qk_rope(q, k, pos[:2], freq)),
        ("positions", lambda: hx.qk_rope(q, k, pos.view(3, 1), freq)), ("need axis", lambda: hx.qk_rope(q, k, two, freq)),
        ("axis", lambda: hx.qk_rope(q, k, two, freq, axis=axis[:5])), ("axis", lambda: hx.qk_rope(q, k, two, freq, axis=axis.long())),
        ("at least one axis", lambda: hx.qk_rope(q, k, two[:0], freq, axis=axis)),
        ("q_weight", lambda: hx.qk_rope(q, k, pos, freq, q_weight=w[:32])),
        ("k_weight", lambda: hx.qk_rope(q, k, pos, freq, k_weight=w.bfloat16())),
        ("eps", lambda: hx.qk_rope(q, k, pos, freq, eps=-1.0)), ("scale", lambda: hx.qk_rope(q, k, pos, freq, scale=math.nan)),
        ("scale", lambda: hx.qk_rope(q, k, pos, freq, scale=1e39)), ("eps", lambda: hx.qk_rope(q, k, pos, freq, eps=math.inf)),
        ("out's q", lambda: hx.qk_rope(q, k, pos, freq, out=(q.float(), k))),
        ("out's k", lambda: hx.qk_rope(q, k, pos, freq, out=(q, k[:2]))),
        ("no|none", lambda: hx.qk_rope(q, None, pos, freq, out=(q, k))),
        ("for k", lambda: hx.qk_rope(q, k, pos, freq, out=(q, None))),
        ("share", lambda: hx.qk_rope(q, k, pos, freq, out=(q[:1].expand(3, 4, 64), k))),
        ("must not share", lambda: hx.qk_rope(q, k, pos, freq, out=(x[:, :4], x[:, 3:5]))),
        ("GPU", lambda: hx.qk_rope(q, k, pos.cpu(), freq)),
        ("even", lambda: hx.rope_frequencies(7)), ("add up", lambda: hx.rope_frequencies(64, sections=(16, 17))),
    ]
    for i, (msg, call) in enumerate(bad):
        with pytest.raises(pkg.HxmiError, match=msg):
            call()
            pytest.fail(f"call {i} ({msg}) was taken")
