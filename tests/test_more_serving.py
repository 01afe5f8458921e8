"""CPU checks of qk_rope's, the 4-bit cache's and verify's entries: what they refuse
before any launch, empty calls, workspace sizes and the cache's layout."""
import pytest
import torch

P = 1 << 12  # aligned, never dereferenced: every call below is refused or has nothing to do


def last(pkg):
    return pkg.load_library().hxmi_last_error().decode()


def rope(pkg, bf16=0, q=P, k=P, qo=P, ko=P, pos=P, pos64=0, freq=P, w32=0, tokens=4, heads=8, kv_heads=2, d=64, rotary=64,
         axes=1, ldp=4, ld=768, hs=64, ldo=768, interleaved=0, eps=1e-6, scale=1.0):
    return pkg.load_library().hxmi_qk_rope(bf16, q, k, qo, ko, pos, pos64, freq, None, None, None, w32, tokens, heads,
                                           kv_heads, d, rotary, axes, ldp, ld, hs, ld, hs, ldo, 64, ldo, 64, interleaved,
                                           eps, scale, None)


@pytest.mark.parametrize("bad, msg", [
    (dict(bf16=2), "flag"), (dict(pos64=-1), "flag"), (dict(w32=3), "flag"), (dict(interleaved=2), "flag"),
    (dict(tokens=-1), "tokens"), (dict(tokens=1 << 31, ldp=1 << 31), "tokens"), (dict(heads=-1), "heads"),
    (dict(heads=1 << 20), "heads"), (dict(d=0), "multiple of 8"), (dict(d=68), "multiple of 8"), (dict(d=264), "up to 256"),
    (dict(rotary=63), "even"), (dict(rotary=66), "at most head_dim"), (dict(rotary=-2), "even"), (dict(axes=0), "axes"),
    (dict(axes=3, ldp=3), "ld_pos"), (dict(eps=-1.0), "eps"), (dict(eps=float("nan")), "eps"),
    (dict(scale=float("inf")), "scale"), (dict(ld=-1), "stride"), (dict(hs=-1), "stride"), (dict(ldo=-1), "stride"),
    (dict(q=None), "null q"), (dict(qo=None), "null q"), (dict(k=None), "null k"), (dict(ko=None), "null k"),
    (dict(pos=None), "null positions"), (dict(freq=None), "null positions"),
])
def test_rope_refuses(pkg, bad, msg):
    assert rope(pkg, **bad) == 1
    assert msg in last(pkg)


def trim(pkg, requests=4, width=4, ld=4, capacity=16, block=16, ptr=P, count=P):
    return pkg.load_library().hxmi_kv_trim(ptr, ptr, ptr, ptr, count, requests, width, ld, capacity, block, None)


@pytest.mark.parametrize("bad, msg", [
    (dict(requests=-1), "negative"), (dict(width=-1), "negative"), (dict(capacity=-1), "negative"), (dict(block=24), "power of two"),
    (dict(ld=3), "ld_table"), (dict(ptr=None), "null"), (dict(count=None), "null"), (dict(capacity=1 << 31), "2^31"),
    (dict(width=1 << 27, ld=1 << 27), "2^30"), (dict(requests=1 << 30, width=4), "2^31"),
])
def test_trim_refuses(pkg, bad, msg):
    assert trim(pkg, **bad) == 1
    assert msg in last(pkg)


def append(pkg, tokens=4, blocks=4, heads=2, d=64, block=16, bf16=0, ptr=P, codes=P, scale=P, ld=128, hs=64):
    return pkg.load_library().hxmi_kv4_append(bf16, ptr, ptr, ptr, codes, codes, scale, scale, tokens, blocks, heads, d,
                                              block, ld, hs, ld, hs, None)


def read(pkg, tokens=4, blocks=4, heads=2, d=64, block=16, bf16=0, ptr=P, codes=P, scale=P):
    return pkg.load_library().hxmi_kv4_read(bf16, codes, codes, scale, scale, ptr, ptr, ptr, tokens, blocks, heads, d,
                                            block, None)


@pytest.mark.parametrize("call", [append, read])
@pytest.mark.parametrize("bad, msg", [
    (dict(tokens=-1), "tokens"), (dict(heads=0), "positive"), (dict(d=0), "positive"), (dict(d=68), "multiple of 8"),
    (dict(d=136), "up to 128"), (dict(block=24), "power of two"), (dict(blocks=-1), "positive"),
    (dict(codes=None), "null cache"), (dict(codes=P + 8), "16-byte"), (dict(scale=P + 4), "16-byte"),
    (dict(scale=None), "null cache"), (dict(ptr=None), "null"), (dict(bf16=2), "is_bf16"),
])
def test_cache_calls_refuse(pkg, call, bad, msg):
    assert call(pkg, **bad) == 1
    assert msg in last(pkg) and "hxmi_kv4_" in last(pkg)


def test_append_refuses_negative_strides(pkg):
    assert append(pkg, ld=-1) == 1 and "stride" in last(pkg)
    assert append(pkg, hs=-8) == 1 and "stride" in last(pkg)


def attend(pkg, bf16=0, q=P, table=P, lens=P, cu=P, o=P, tokens=8, requests=4, heads=8, kv_heads=2, d=64, block=16,
           blocks=4, width=4, ld=4, ldq=512, hq=64, scale=0.125, ws=None, codes=P, scales=P):
    return pkg.load_library().hxmi_kv4_attention(bf16, q, codes, codes, scales, scales, table, lens, cu, o, tokens,
                                                 requests, heads, kv_heads, d, block, blocks, width, ld, ldq, hq, 512, 64,
                                                 scale, ws, 0, None)


@pytest.mark.parametrize("bad, msg", [
    (dict(bf16=3), "is_bf16"), (dict(tokens=-1), "negative"), (dict(requests=-1), "negative"),
    (dict(heads=7), "multiple of kv_heads"), (dict(cu=None), "one row a request"), (dict(scale=0.0), "scale"),
    (dict(scale=float("nan")), "scale"), (dict(d=132), "multiple of 8"), (dict(block=20), "power of two"),
    (dict(blocks=0), "without blocks"), (dict(q=None), "null"), (dict(lens=None), "null"), (dict(table=None), "null"),
    (dict(ld=3), "ld_table"), (dict(ldq=-1), "stride"), (dict(ws=P + 16), "256-byte"), (dict(tokens=1 << 28), "2^31"),
    (dict(width=1 << 27, ld=1 << 27), "2^30"), (dict(codes=P + 4), "16-byte"), (dict(scales=P + 4), "16-byte"),
])
def test_attention_refuses(pkg, bad, msg):
    assert attend(pkg, **bad) == 1
    assert msg in last(pkg) and "hxmi_kv4_attention" in last(pkg)


def verify(pkg, dtype=0, x=P, d=P, u=P, draw=P, cu=P, q=P, q_type=2, t=1.0, k=0, p=1.0, m=0.0, out=P, counts=P, rows=6,
           requests=2, vocab=100, ld=100, ldq=100, ws=P, ws_bytes=1 << 20):
    return pkg.load_library().hxmi_verify(dtype, x, d, u, draw, cu, q, q_type, None, None, None, None, t, k, p, m, out, counts,
                                          rows, requests, vocab, ld, ldq, ws, ws_bytes, None)


@pytest.mark.parametrize("bad, msg", [
    (dict(dtype=3), "dtype"), (dict(q_type=-1), "probs_dtype"), (dict(rows=-1), "rows"), (dict(requests=-1), "requests"),
    (dict(requests=0), "without a request"), (dict(cu=None, rows=5), "same number"), (dict(vocab=0), "vocab"),
    (dict(vocab=(1 << 20) + 1, ld=1 << 21, ldq=1 << 21), "vocab"), (dict(ld=99), "leading dimension"),
    (dict(ldq=99), "draft_probs"), (dict(x=None), "null"), (dict(u=None), "null"), (dict(d=None), "null drafts"),
    (dict(draw=None), "null draw"), (dict(counts=None), "counts"), (dict(out=None), "null"), (dict(x=P + 1), "aligned"),
    (dict(q=P + 2), "aligned"), (dict(t=-0.5), "temperature"), (dict(t=float("nan")), "temperature"),
    (dict(p=float("nan")), "top_p"), (dict(m=float("nan")), "min_p"), (dict(ws=None), "workspace"),
    (dict(ws=P + 16), "workspace"), (dict(ws_bytes=16384), "workspace"),
])
def test_verify_refuses(pkg, bad, msg):
    assert verify(pkg, **bad) == 1
    assert msg in last(pkg)


def test_verify_workspace(pkg):
    need = pkg.load_library().hxmi_verify_workspace_bytes
    assert need(0, 1, 9) == need(-1, 1, 9) == need(1, 0, 9) == need(1, 1, 0) == 0 and need(1, 1, 1) > 16384
    assert need(100, 3, 9) - need(1, 3, 9) == 99 * (need(2, 3, 9) - need(1, 3, 9))
    assert need(7, 3, 152000) - need(7, 2, 152000) == (152000 + 511) // 512 * 8


def test_empty_calls_do_nothing(pkg):
    assert verify(pkg, rows=0, requests=0, x=None, draw=None) == 0 and trim(pkg, requests=0, ptr=None) == 0
    assert rope(pkg, tokens=0, q=None, k=None, pos=None) == 0 and rope(pkg, heads=0, kv_heads=0, q=None, k=None) == 0
    assert append(pkg, tokens=0, ptr=None) == 0 and append(pkg, blocks=0, codes=None, scale=None) == 0
    assert read(pkg, tokens=0, ptr=None) == 0
    assert attend(pkg, tokens=0, q=None) == 0 and attend(pkg, requests=0, lens=None) == 0


def test_attention_workspace(pkg):
    """Few rows share the keys out, enough tiles do not; within the counters."""
    need = pkg.load_library().hxmi_kv4_attention_workspace_bytes
    assert need(1, 1, 32, 4, 64, 64, 30, 0) > 16384
    assert need(1, 1, 32, 8, 128, 32, 4096, 0) > need(1, 1, 32, 8, 128, 32, 64, 0) > 0
    assert need(1024, 1024, 32, 8, 128, 64, 128, 0) == 0  # 8192 tiles
    assert need(1, 1, 32, 4, 64, 16, 1, 0) == 0  # one page
    assert need(0, 1, 32, 4, 64, 64, 30, 0) == 0 and need(1, 1, 31, 4, 64, 64, 30, 0) == 0
    assert need(1, 1, 32, 4, 64, 63, 30, 0) == 0


def test_cache_layout(pkg):
    c = pkg.KVCache4.empty(3, 2, 40, 32, device="cpu")
    assert c.k.shape == (3, 2, 32, 32) and c.v.shape == (3, 2, 2, 64, 8) and c.k.dtype == torch.uint8
    assert c.k_scale.shape == c.v_scale.shape == (3, 2, 2, 32) and c.k_scale.dtype == torch.uint8 and not c.v.any()
    assert (c.blocks, c.kv_heads, c.block_size, c.head_dim) == (3, 2, 32, 40)
    for bad in (dict(block_size=48), dict(head_dim=44), dict(head_dim=136), dict(head_dim=0)):
        with pytest.raises(pkg.HxmiError):
            pkg.KVCache4.empty(**{**dict(blocks=1, kv_heads=1, head_dim=64, block_size=16, device="cpu"), **bad})


def test_rope_frequencies(pkg):
    freq, axis = pkg.rope_frequencies(8, 10000.0, device="cpu")
    assert freq.dtype == torch.float64 and axis is None and torch.allclose(freq, torch.tensor([1, 0.1, 0.01, 0.001]).double())
    freq, axis = pkg.rope_frequencies(12, 1e6, sections=(1, 3, 2), device="cpu")
    assert axis.dtype == torch.int32 and axis.tolist() == [0, 1, 1, 1, 2, 2] and freq.numel() == 6
    assert pkg.rope_frequencies(0, device="cpu")[0].numel() == 0
    for bad in (dict(rotary_dim=9), dict(rotary_dim=-2), dict(rotary_dim=8, sections=(1, 2)), dict(rotary_dim=8, sections=(5, -1))):
        with pytest.raises(pkg.HxmiError):
            pkg.rope_frequencies(**bad, device="cpu")


def test_ops_refuse_cpu_tensors(pkg):
    c = pkg.KVCache4.empty(2, 1, 64, 16, device="cpu")
    x, i = torch.zeros(2, 1, 64, dtype=torch.float16), torch.zeros(2, dtype=torch.int32)
    table, freq = torch.zeros(2, 1, dtype=torch.int32), torch.zeros(32, dtype=torch.float64)
    for call in (lambda: pkg.kv_append(c, x, x, i.long()), lambda: pkg.kv_read(c, i.long()),
                 lambda: pkg.kv_attention(x, c, table, i), lambda: pkg.qk_rope(x, x, i, freq),
                 lambda: pkg.verify(x, torch.zeros(2, 1, dtype=torch.int64), torch.zeros(2, 1), torch.zeros(2))):
        with pytest.raises(pkg.HxmiError, match="GPU"):
            call()
