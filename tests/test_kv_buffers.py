"""The Python calls of the cache, the attention and the sampling hold every
buffer against the call before the library sees it: on the CPU, with stand-ins
for device tensors and a library that only counts its calls."""
import pytest
import torch

import streamoe_amd as sa
from test_serving_buffers import BAD, On, k  # noqa: F401 (a fixture)

I32, BF16, I8, F32 = torch.int32, torch.bfloat16, torch.int8, torch.float32


class Cache4(On):
    """[pages, heads, slots, dim] in any order of the axes."""

    def stride(self, *a):
        return self.meta.stride(*a)


def _cache(dtype=BF16, shape=(6, 2, 32, 64), **kw):
    t = lambda at: Cache4(*shape, dtype=dtype, at=at, **kw)
    s = lambda at: On(*shape[:3], at=at, **{x: y for x, y in kw.items() if x == "dev"}) if dtype is I8 else None
    return sa.KvCache(t(1 << 20), t(1 << 24), s(1 << 26), s(1 << 27))


def _tok(n=5, **kw):
    return [On(3, 4, dtype=I32, **kw), On(n, dtype=I32), On(n, dtype=I32)]


def test_cache_struct():
    c = _cache().c()
    assert (c.page_stride, c.head_stride, c.slot_stride, c.bits) == (2 * 32 * 64 * 2, 32 * 64 * 2, 128, 16)
    c = _cache(I8, step=(4096, 64, 128, 1)).c()  # heads behind slots
    assert (c.page_stride, c.head_stride, c.slot_stride, c.bits) == (4096, 64, 128, 8)
    c = _cache(shape=(1, 1, 32, 64), step=(7, 9, 64, 1)).c()  # strides of axes of one
    assert (c.page_stride, c.head_stride, c.slot_stride) == (0, 0, 128)


@pytest.mark.parametrize("make", [
    lambda: sa.KvCache(Cache4(6, 2, 32, 64, dtype=BF16), Cache4(6, 2, 32, 32, dtype=BF16)),
    lambda: sa.KvCache(Cache4(6, 2, 32, 64, dtype=BF16), Cache4(6, 2, 32, 64, dtype=BF16, dev=1)),
    lambda: sa.KvCache(Cache4(6, 2, 32, 64, dtype=BF16, dev=-1), Cache4(6, 2, 32, 64, dtype=BF16, dev=-1)),
    lambda: sa.KvCache(Cache4(6, 2, 32, 64, dtype=F32), Cache4(6, 2, 32, 64, dtype=F32)),
    lambda: sa.KvCache(Cache4(6, 2, 32, 64, dtype=BF16), Cache4(6, 2, 32, 64, dtype=I8)),
    lambda: sa.KvCache(Cache4(6, 2, 32, 64, dtype=I8), Cache4(6, 2, 32, 64, dtype=I8)),          # no scales
    lambda: sa.KvCache(Cache4(6, 2, 32, 64, dtype=I8), Cache4(6, 2, 32, 64, dtype=I8), On(6, 2, 32), On(6, 2, 16)),
    lambda: sa.KvCache(Cache4(6, 2, 32, 64, dtype=I8), Cache4(6, 2, 32, 64, dtype=I8), On(6, 2, 32), On(6, 2, 32, dev=1)),
    lambda: sa.KvCache(Cache4(6, 2, 32, 64, dtype=BF16), Cache4(6, 2, 32, 64, dtype=BF16), On(6, 2, 32), On(6, 2, 32)),
    lambda: sa.KvCache(Cache4(6, 2, 32, 64, dtype=BF16, step=(4096, 2048, 64, 2)), Cache4(6, 2, 32, 64, dtype=BF16)),
    lambda: sa.KvCache(Cache4(6, 2, 32, 64, dtype=BF16, step=(4096, 64, 128, 1)), Cache4(6, 2, 32, 64, dtype=BF16)),
    lambda: sa.KvCache(Cache4(6, 64, 64, dtype=BF16), Cache4(6, 64, 64, dtype=BF16)),
])
def test_caches_that_are_none(make):
    with pytest.raises(sa.SmoeError):
        make().c()


def _refused(k, call):
    before = k.lib.calls
    assert call() == BAD
    assert k.lib.calls == before


@pytest.mark.parametrize("name", ["kv_append", "kv_gather"])
def test_rows(k, name):  # noqa: F811
    go = lambda tok, a, b, n=5, c=None: getattr(k, name)(c or _cache(), *tok, a, b, n)
    rows = lambda **kw: Cache4(5, 2, 64, **kw)
    assert go(_tok(), rows(), rows()) == 0 and k.lib.calls == 1
    assert go(_tok(), Cache4(5, 128, dtype=BF16), rows(dtype=BF16)) == 0
    assert go(_tok(), rows(step=(500, 64, 1)), rows(step=(500, 64, 1))) == 0
    for a, b in ((rows(), rows(dtype=BF16)), (rows(), rows(step=(500, 64, 1))), (rows(step=(500, 128, 1)), rows()),
                 (rows(step=(128, 64, 2)), rows(step=(128, 64, 2))), (rows(dev=1), rows(dev=1)), (rows(), rows(dev=-1)),
                 (Cache4(4, 2, 64), Cache4(4, 2, 64)), (Cache4(5, 3, 64), Cache4(5, 3, 64)), (Cache4(5, 64), Cache4(5, 64)),
                 (rows(dtype=I8), rows(dtype=I8)), (None, rows()), (rows(), None)):
        _refused(k, lambda: go(_tok(), a, b))
    _refused(k, lambda: go(_tok(4), rows(), rows()))
    _refused(k, lambda: go(_tok(dev=1), rows(), rows()))
    _refused(k, lambda: go([On(12, dtype=I32)] + _tok()[1:], rows(), rows()))
    _refused(k, lambda: go([On(3, 4, dtype=torch.int64)] + _tok()[1:], rows(), rows()))
    _refused(k, lambda: go([On(3, 4, dtype=I32, step=(8, 1))] + _tok()[1:], rows(), rows()))
    _refused(k, lambda: go(_tok(), rows(), rows(), c=_cache(dev=1)))


def test_attn(k):  # noqa: F811
    q = lambda **kw: Cache4(5, 8, 64, **kw)
    ws = On(1 << 16, dtype=torch.uint8)
    go = lambda a=None, o=None, w=ws, tok=None: k.attn_decode(_cache(), *(tok or _tok()), a or q(), 0.1, 0, o or On(5, 8, 64), 8, 5, w)
    assert go() == 0 and k.lib.calls == 1
    assert go(q(dtype=BF16, step=(1024, 64, 1))) == 0
    for a, o in ((q(dev=1), None), (q(step=(512, 128, 1)), None), (Cache4(5, 4, 64), None), (q(dtype=I8), None),
                 (None, On(5, 8, 63)), (None, On(5, 8, 64, dev=1)), (None, On(5, 8, 64, step=(1024, 64, 1))), (None, On(5, 8, 64, dtype=I8))):
        _refused(k, lambda: go(a, o))
    for w in (None, On(64, dtype=torch.uint8, dev=1), On(64, dtype=torch.uint8, step=(2,))):
        _refused(k, lambda: go(w=w))
    _refused(k, lambda: go(tok=_tok(3)))
    _refused(k, lambda: k.attn_decode(_cache(), *_tok(), q(), 0.1, -1, On(5, 8, 64), 8, 5, ws))


def test_sample(k):  # noqa: F811
    one = lambda **kw: On(4, **kw)
    base = dict(logits=On(4, 100), t=one(), k=one(dtype=I32), p=one(), m=one(), u=one(), n=4, V=100, tok=one(dtype=I32), lp=one(),
                ws=On(1 << 16, dtype=torch.uint8))
    go = lambda **kw: k.sample(*dict(base, **kw).values())
    assert go() == 0 and k.lib.calls == 1
    assert go(t=None, k=None, p=None, m=None, lp=None) == 0
    for kw in (dict(logits=On(4, 99)), dict(logits=On(4, 100, dtype=BF16)), dict(logits=None), dict(t=On(3)), dict(k=one()),
               dict(p=one(dev=1)), dict(m=one(dtype=torch.float64)), dict(u=None), dict(u=one(step=(2,))), dict(tok=one()),
               dict(tok=None), dict(lp=On(3)), dict(ws=None), dict(ws=On(64, dtype=torch.uint8, dev=1))):
        _refused(k, lambda: go(**kw))
