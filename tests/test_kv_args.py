"""Refusals of smoe_kv_append, smoe_kv_gather and smoe_attn_decode, on the CPU:
every argument check comes before any device call."""
import pytest

from refusals import fake_handle, refused

# 8 pages of 32 slots, 4 heads of 64 bf16: rows of 128 bytes.
CACHE = dict(k=1 << 20, v=1 << 21, k_scales=None, v_scales=None, page_stride=16384, head_stride=4096, slot_stride=128,
             n_pages=8, page_size=32, n_heads=4, head_dim=64, bits=16, reserved=0)
I8 = dict(bits=8, page_stride=8192, head_stride=2048, slot_stride=64, k_scales=1 << 22, v_scales=1 << 23)
TOKENS = dict(table=4096, seq=8192, pos=12288, n_seqs=3, table_width=5, n_tokens=7, reserved=0)


def _c(cache, tokens):
    from streamoe_amd import _abi

    return _abi.KvCacheC(*dict(CACHE, **cache).values()), _abi.KvTokensC(*dict(TOKENS, **tokens).values())


def _append(cache={}, tokens={}, **kw):
    from streamoe_amd import _abi

    c, t = _c(cache, tokens)
    a = dict(h=fake_handle(), cache=c, tokens=t, k=1 << 24, v=1 << 25, x_is_bf16=1, x_stride=256)
    a.update(kw)
    return _abi.load().smoe_kv_append(*a.values())


def _gather(cache={}, tokens={}, **kw):
    from streamoe_amd import _abi

    c, t = _c(cache, tokens)
    a = dict(h=fake_handle(), cache=c, tokens=t, k=1 << 24, v=1 << 25, out_is_bf16=0, out_stride=256)
    a.update(kw)
    return _abi.load().smoe_kv_gather(*a.values())


def _attn(cache={}, tokens={}, **kw):
    from streamoe_amd import _abi

    c, t = _c(cache, tokens)
    a = dict(h=fake_handle(), cache=c, tokens=t, q=1 << 24, q_is_bf16=1, q_stride=1024, n_heads=16, scale=0.1, window=0,
             out=1 << 25, out_is_bf16=0, workspace=1 << 26, workspace_bytes=1 << 26)
    a.update(kw)
    return _abi.load().smoe_attn_decode(*a.values())


SHARED = [
    (dict(k=None), {}, "INVALID_ARG"),
    (dict(v=None), {}, "INVALID_ARG"),
    (dict(n_pages=0), {}, "INVALID_ARG"),
    (dict(page_size=0), {}, "INVALID_ARG"),
    (dict(n_heads=0), {}, "INVALID_ARG"),
    (dict(head_dim=0), {}, "INVALID_ARG"),
    (dict(reserved=1), {}, "INVALID_ARG"),
    (dict(bits=4), {}, "UNSUPPORTED_BITS"),
    (dict(k_scales=1 << 22), {}, "INVALID_ARG"),                         # scales of bf16
    (dict(I8, k_scales=None), {}, "INVALID_ARG"),
    (dict(I8, v_scales=None), {}, "INVALID_ARG"),
    (dict(head_dim=72), {}, "UNSUPPORTED_SHAPE"),
    (dict(head_dim=272, slot_stride=544, head_stride=17408, page_stride=69632), {}, "UNSUPPORTED_SHAPE"),
    (dict(page_size=24), {}, "UNSUPPORTED_SHAPE"),
    (dict(n_heads=257, page_stride=1 << 21), {}, "UNSUPPORTED_SHAPE"),
    (dict(slot_stride=1 << 27), {}, "UNSUPPORTED_SHAPE"),
    (dict(k=(1 << 20) + 8), {}, "MISALIGNED"),
    (dict(v=(1 << 21) + 2), {}, "MISALIGNED"),
    (dict(I8, k_scales=(1 << 22) + 4), {}, "MISALIGNED"),
    (dict(page_stride=16392), {}, "MISALIGNED"),
    (dict(slot_stride=136), {}, "MISALIGNED"),
    (dict(slot_stride=112), {}, "INVALID_ARG"),                          # rows on each other
    (dict(head_stride=4080), {}, "INVALID_ARG"),
    (dict(page_stride=0), {}, "INVALID_ARG"),
    (dict(page_stride=1 << 62), {}, "INVALID_ARG"),
    (dict(v=1 << 20), {}, "INVALID_ARG"),                                # k and v the same
    (dict(v=(1 << 20) + 64), {}, "INVALID_ARG"),
    (dict(v=(1 << 20) + 16384), {}, "INVALID_ARG"),
    (dict(I8, v_scales=1 << 22), {}, "INVALID_ARG"),
    (dict(I8, k_scales=(1 << 20) + 65520), {}, "INVALID_ARG"),           # the last row of k
    ({}, dict(table=None), "INVALID_ARG"),
    ({}, dict(seq=None), "INVALID_ARG"),
    ({}, dict(pos=None), "INVALID_ARG"),
    ({}, dict(n_seqs=0), "INVALID_ARG"),
    ({}, dict(table_width=0), "INVALID_ARG"),
    ({}, dict(n_tokens=0), "INVALID_ARG"),
    ({}, dict(reserved=2), "INVALID_ARG"),
    ({}, dict(n_tokens=16385), "UNSUPPORTED_SHAPE"),
    ({}, dict(table_width=(1 << 25) + 1), "UNSUPPORTED_SHAPE"),
    ({}, dict(pos=12290), "MISALIGNED"),
]


@pytest.mark.parametrize("call", [_append, _gather, _attn])
@pytest.mark.parametrize("cache,tokens,code", SHARED)
def test_shared_refusals(call, cache, tokens, code):
    refused(call(cache, tokens), code)


@pytest.mark.parametrize("call", [_append, _gather, _attn])
def test_null(call):
    refused(call(h=None), "INVALID_ARG")
    refused(_null(call, "cache"), "INVALID_ARG")
    refused(_null(call, "tokens"), "INVALID_ARG")


def _null(call, name):
    from streamoe_amd import _abi

    c, t = _c({}, {})
    c, t = (None, t) if name == "cache" else (c, None)
    lib = _abi.load()
    if call is _append:
        return lib.smoe_kv_append(fake_handle(), c, t, 1 << 24, 1 << 25, 1, 256)
    if call is _gather:
        return lib.smoe_kv_gather(fake_handle(), c, t, 1 << 24, 1 << 25, 1, 256)
    return lib.smoe_attn_decode(fake_handle(), c, t, 1 << 24, 1, 1024, 16, 0.1, 0, 1 << 25, 1, 1 << 26, 1 << 26)


@pytest.mark.parametrize("call", [_append, _gather])
@pytest.mark.parametrize("kw,code", [
    (dict(k=None), "INVALID_ARG"),
    (dict(v=None), "INVALID_ARG"),
    (dict(k=(1 << 24) + 8), "MISALIGNED"),
    (dict(v=(1 << 25) + 4), "MISALIGNED"),
    (dict(k=1 << 20), "INVALID_ARG"),                     # the cache's own rows
    (dict(v=(1 << 21) + 131072 - 16), "INVALID_ARG"),     # its last
])
def test_rows(call, kw, code):
    refused(call(**kw), code)


def test_strides_of_rows():
    refused(_append(x_stride=248), "INVALID_ARG")          # rows on each other
    refused(_append(x_stride=260), "MISALIGNED")
    refused(_gather(out_stride=258), "MISALIGNED")
    refused(_gather(out_stride=1 << 62), "INVALID_ARG")
    refused(_append(x_stride=1 << 59, x_is_bf16=0), "INVALID_ARG")
    refused(_gather(k=4080), "INVALID_ARG")                # the table
    refused(_append(dict(I8), k=(1 << 22) + 16), "INVALID_ARG")   # a scale
    # Outputs that lie on each other: the same rows, and shifted ones.
    refused(_gather(v=1 << 24), "INVALID_ARG")
    refused(_gather(v=(1 << 24) + 512), "INVALID_ARG")
    refused(_gather(v=(1 << 24) + 1024, out_stride=500), "INVALID_ARG")


@pytest.mark.parametrize("kw,code", [
    (dict(q=None), "INVALID_ARG"),
    (dict(out=None), "INVALID_ARG"),
    (dict(workspace=None), "INVALID_ARG"),
    (dict(n_heads=0), "INVALID_ARG"),
    (dict(n_heads=18), "INVALID_ARG"),
    (dict(n_heads=4100, q_stride=1 << 20), "UNSUPPORTED_SHAPE"),
    (dict(q_stride=1000), "INVALID_ARG"),
    (dict(q_stride=1028), "MISALIGNED"),
    (dict(q=(1 << 24) + 8), "MISALIGNED"),
    (dict(out=(1 << 25) + 8), "MISALIGNED"),
    (dict(workspace=(1 << 26) + 128), "MISALIGNED"),
    (dict(workspace_bytes=1 << 16), "WORKSPACE_TOO_SMALL"),
    (dict(out=1 << 24), "INVALID_ARG"),                   # the queries
    (dict(out=(1 << 20) + 4096), "INVALID_ARG"),          # the keys
    (dict(workspace=8192), "INVALID_ARG"),                # seq
    (dict(out=(1 << 26) + 4096), "INVALID_ARG"),          # the workspace
])
def test_attn(kw, code):
    refused(_attn(**kw), code)


def test_workspace_size():
    from streamoe_amd import _abi

    lib, (c, _) = _abi.load(), _c({}, {})
    assert 0 < lib.smoe_attn_decode_workspace_size(c, 16, 7) <= lib.smoe_attn_decode_workspace_size(c, 16, 16384)
    assert lib.smoe_attn_decode_workspace_size(c, 18, 7) == 0
    assert lib.smoe_attn_decode_workspace_size(c, 16, 0) == 0
    assert lib.smoe_attn_decode_workspace_size(c, 16, 16385) == 0
    assert lib.smoe_attn_decode_workspace_size(None, 16, 7) == 0
    assert lib.smoe_attn_decode_workspace_size(_c(dict(head_dim=8), {})[0], 16, 7) == 0
