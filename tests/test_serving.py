"""CPU checks of the serving operators' entries (kv_plan, kv_append, kv_read,
kv_attention, sample): what they refuse before any launch, empty calls,
workspace sizes and the cache's layout."""
import pytest
import torch

P = 1 << 12  # aligned, never dereferenced: every call below is refused or has nothing to do


def last(pkg):
    return pkg.load_library().hxmi_last_error().decode()


def plan(pkg, requests=4, width=4, ld=4, capacity=16, tokens=8, block=16, ptr=P, count=P):
    return pkg.load_library().hxmi_kv_plan(ptr, ptr, ptr, ptr, count, ptr, ptr, ptr, ptr, ptr, requests, width, ld,
                                           capacity, tokens, block, None)


@pytest.mark.parametrize("bad, msg", [
    (dict(requests=-1), "negative"), (dict(tokens=-1), "negative"), (dict(block=48), "power of two"),
    (dict(block=8), "power of two"), (dict(block=512), "power of two"), (dict(requests=4097), "4096"),
    (dict(ld=3), "ld_table"), (dict(ptr=None), "null"), (dict(count=None), "null"),
    (dict(tokens=1 << 31), "2^31"), (dict(width=1 << 27, ld=1 << 27, block=16), "2^30"),
])
def test_plan_refuses(pkg, bad, msg):
    assert plan(pkg, **bad) == 1
    assert msg in last(pkg)


def append(pkg, tokens=4, blocks=4, heads=2, d=64, block=16, bf16=0, ptr=P, codes=P, ld=128, hs=64):
    return pkg.load_library().hxmi_kv_append(bf16, ptr, ptr, ptr, codes, codes, P, P, tokens, blocks, heads, d, block,
                                             ld, hs, ld, hs, None)


def read(pkg, tokens=4, blocks=4, heads=2, d=64, block=16, bf16=0, ptr=P, codes=P):
    return pkg.load_library().hxmi_kv_read(bf16, codes, codes, P, P, ptr, ptr, ptr, tokens, blocks, heads, d, block,
                                           None)


@pytest.mark.parametrize("call", [append, read])
@pytest.mark.parametrize("bad, msg", [
    (dict(tokens=-1), "tokens"), (dict(heads=0), "positive"), (dict(d=0), "positive"), (dict(d=68), "multiple of 8"),
    (dict(d=136), "up to 128"), (dict(block=24), "power of two"), (dict(blocks=-1), "positive"),
    (dict(codes=None), "null cache"), (dict(codes=P + 8), "16-byte"), (dict(ptr=None), "null"), (dict(bf16=2), "is_bf16"),
])
def test_cache_calls_refuse(pkg, call, bad, msg):
    assert call(pkg, **bad) == 1
    assert msg in last(pkg)


def test_append_refuses_negative_strides(pkg):
    assert append(pkg, ld=-1) == 1 and "stride" in last(pkg)
    assert append(pkg, hs=-8) == 1 and "stride" in last(pkg)


def attend(pkg, bf16=0, q=P, table=P, lens=P, cu=P, o=P, tokens=8, requests=4, heads=8, kv_heads=2, d=64, block=16,
           blocks=4, width=4, ld=4, ldq=512, hq=64, scale=0.125, ws=None, codes=P):
    return pkg.load_library().hxmi_kv_attention(bf16, q, codes, codes, P, P, table, lens, cu, o, tokens, requests,
                                                heads, kv_heads, d, block, blocks, width, ld, ldq, hq, 512, 64, scale,
                                                ws, 0, None)


@pytest.mark.parametrize("bad, msg", [
    (dict(bf16=3), "is_bf16"), (dict(tokens=-1), "negative"), (dict(requests=-1), "negative"),
    (dict(heads=7), "multiple of kv_heads"), (dict(cu=None), "one row a request"), (dict(scale=0.0), "scale"),
    (dict(scale=-1.0), "scale"), (dict(scale=float("inf")), "scale"), (dict(scale=float("nan")), "scale"),
    (dict(d=72, kv_heads=0), "positive"), (dict(d=132), "multiple of 8"), (dict(block=20), "power of two"),
    (dict(blocks=0), "without blocks"), (dict(q=None), "null"), (dict(lens=None), "null"), (dict(table=None), "null"),
    (dict(ld=3), "ld_table"), (dict(ldq=-1), "stride"), (dict(ws=P + 16), "256-byte"),
    (dict(tokens=1 << 28), "2^31"), (dict(width=1 << 27, ld=1 << 27), "2^30"), (dict(codes=P + 4), "16-byte"),
])
def test_attention_refuses(pkg, bad, msg):
    assert attend(pkg, **bad) == 1
    assert msg in last(pkg)


def sample(pkg, dtype=0, x=P, u=P, t=1.0, k=0, p=1.0, m=0.0, rows=2, vocab=100, ld=100, out=P):
    return pkg.load_library().hxmi_sample(dtype, x, u, None, None, None, None, t, k, p, m, out, rows, vocab, ld, None)


@pytest.mark.parametrize("bad, msg", [
    (dict(dtype=3), "dtype"), (dict(dtype=-1), "dtype"), (dict(rows=-1), "rows"), (dict(vocab=0), "vocab"),
    (dict(vocab=(1 << 20) + 1, ld=1 << 21), "vocab"), (dict(ld=99), "leading dimension"), (dict(x=None), "null"),
    (dict(u=None), "null"), (dict(out=None), "null"), (dict(x=P + 1), "aligned"), (dict(x=P + 2, dtype=2), "aligned"),
    (dict(t=-0.5), "temperature"), (dict(t=float("nan")), "temperature"), (dict(t=float("inf")), "temperature"),
    (dict(p=float("nan")), "top_p"), (dict(m=float("nan")), "min_p"),
])
def test_sample_refuses(pkg, bad, msg):
    assert sample(pkg, **bad) == 1
    assert msg in last(pkg)


def test_empty_calls_do_nothing(pkg):
    assert append(pkg, tokens=0, ptr=None) == 0 and append(pkg, blocks=0, codes=None) == 0
    assert read(pkg, tokens=0, ptr=None) == 0
    assert attend(pkg, tokens=0, q=None) == 0 and attend(pkg, requests=0, lens=None) == 0
    assert sample(pkg, rows=0, x=None, vocab=0) == 0


def test_attention_workspace(pkg):
    """Few rows share the keys out, enough tiles do not; within the counters."""
    need = pkg.load_library().hxmi_kv_attention_workspace_bytes
    assert need(1, 1, 32, 4, 64, 64, 30, 0) > 16384
    assert need(1, 1, 32, 8, 128, 32, 4096, 0) > need(1, 1, 32, 8, 128, 32, 64, 0) > 0
    assert need(1024, 1024, 32, 8, 128, 64, 128, 0) == 0  # 8192 tiles
    assert need(1, 1, 32, 4, 64, 16, 1, 0) == 0  # one page
    assert need(0, 1, 32, 4, 64, 64, 30, 0) == 0 and need(1, 1, 31, 4, 64, 64, 30, 0) == 0
    assert need(1, 1, 32, 4, 64, 63, 30, 0) == 0


def test_cache_layout(pkg):
    c = pkg.KVCache.empty(3, 2, 40, 32, device="cpu")
    assert c.k.shape == (3, 2, 32, 48) and c.v.shape == (3, 2, 2, 48, 16) and c.k.dtype == torch.int8
    assert c.k_scale.shape == (3, 2) and c.k_scale.dtype == torch.float32 and not c.v.any()
    assert (c.blocks, c.kv_heads, c.block_size, c.head_dim) == (3, 2, 32, 40)
    for bad in (dict(block_size=48), dict(head_dim=44), dict(head_dim=136), dict(head_dim=0)):
        with pytest.raises(pkg.HxmiError):
            pkg.KVCache.empty(**{**dict(blocks=1, kv_heads=1, head_dim=64, block_size=16, device="cpu"), **bad})


def test_ops_refuse_cpu_tensors(pkg):
    c = pkg.KVCache.empty(2, 1, 64, 16, device="cpu")
    x, i = torch.zeros(2, 1, 64, dtype=torch.float16), torch.zeros(2, dtype=torch.int32)
    table = torch.zeros(2, 1, dtype=torch.int32)
    for call in (lambda: pkg.kv_append(c, x, x, i.long()), lambda: pkg.kv_read(c, i.long()),
                 lambda: pkg.kv_attention(x, c, table, i), lambda: pkg.sample(x[:, 0], torch.zeros(2)),
                 lambda: pkg.kv_plan(i, i, table, i, i[:1], block_size=16, tokens=2)):
        with pytest.raises(pkg.HxmiError, match="GPU"):
            call()
