"""The Python calls of the serving operators hold every buffer against the
call before the library sees it: on the CPU, with stand-ins for device tensors
and a library that only counts its calls."""
import pytest
import torch

import streamoe_amd as sa

BAD = 1  # SMOE_ERR_INVALID_ARG


class On:
    """A tensor on device `dev`, as far as the calls look."""

    def __init__(self, *shape, dtype=torch.float32, dev=0, step=None, at=1 << 20):
        self.meta = torch.empty(*shape, dtype=dtype, device="meta")
        if step is not None:
            self.meta = self.meta.as_strided(shape, step)
        self.dev, self.at = dev, at
        self.dtype, self.shape = dtype, self.meta.shape

    def get_device(self):
        return self.dev

    def data_ptr(self):
        return self.at

    def detach(self):
        return self

    def __getattr__(self, name):  # numel, element_size, is_contiguous, stride, dim
        return getattr(self.meta, name)

    def __getitem__(self, i):
        t = self.meta[i]
        return On(*t.shape, dtype=self.dtype, dev=self.dev, step=t.stride())


class Library:
    calls = 0

    def __getattr__(self, name):
        def call(*args):
            self.calls += 1
            return 0
        return call


@pytest.fixture
def k(monkeypatch):
    lib = Library()
    monkeypatch.setattr(sa, "_lib", lib)
    k = object.__new__(sa.Kernels)
    k.device, k.h, k.lib = 0, 1, lib
    yield k
    k.h = None


def _refused(k, call):
    before = k.lib.calls
    assert call() == BAD
    assert k.lib.calls == before


# A workspace on the host, on another device, of repeated elements.
WRONG = [dict(dev=-1), dict(dev=1), dict(step=(0,)), dict(step=(2,))]


def test_workspace_of_lora(k):
    b16, i32 = torch.bfloat16, torch.int32
    s = sa.Adapters(On(3, 8, 64, dtype=b16), On(3, 32, 8, dtype=b16), On(3))
    go = lambda ws: k.lora(s, On(5, dtype=i32), On(5, 64), None, On(5, 32), 32, 64, 5, ws)
    assert go(On(1 << 16, dtype=torch.uint8)) == 0 and k.lib.calls == 1
    assert go(On(64, 64)) == 0
    for w in WRONG:
        _refused(k, lambda: go(On(1 << 16, dtype=torch.uint8, **w)))


def test_workspace_of_beam_select(k):
    i32 = torch.int32
    go = lambda ws: k.beam_select(On(8, 100), On(8), None, 0, 2, 4, 100, 4, On(2, 4), On(2, 4, dtype=i32),
                                  On(2, 4, dtype=i32), ws)
    assert go(On(1 << 16, dtype=torch.uint8)) == 0 and k.lib.calls == 1
    for w in WRONG:
        _refused(k, lambda: go(On(1 << 16, dtype=torch.uint8, **w)))


# 64 x 256 codes of 4 bits, groups of 64: 8192 bytes, then 512 and 512.
AT = (0, 8192, 8704)


def _qmm(k, buf, at=AT, out_dim=64, in_dim=256, n=5, **kw):
    w = sa.QuantWeights(buf, *at, kw.get("group", 64), kw.get("bits", 4))
    return k.qmm_i8(w, On(n, in_dim, dtype=torch.int8), On(n), 0, On(n, out_dim), out_dim, in_dim, n)


def test_weights_of_qmm_i8(k):
    u8 = torch.uint8
    assert _qmm(k, On(9216, dtype=u8)) == 0 and k.lib.calls == 1
    assert _qmm(k, On(96, 48, dtype=torch.int16)) == 0           # any type and shape that holds the bytes
    assert _qmm(k, On(9216, dtype=u8), at=(1024, 0, 512)) == 0   # any order
    assert _qmm(k, On(9216, dtype=u8), in_dim=384, out_dim=42, at=(0, 8064, 8568), bits=4) == 0
    for w in WRONG:
        _refused(k, lambda: _qmm(k, On(9216, dtype=u8, **w)))
    _refused(k, lambda: _qmm(k, On(9215, dtype=u8)))                            # the biases end behind it
    _refused(k, lambda: _qmm(k, On(9216, dtype=u8), out_dim=65))
    _refused(k, lambda: _qmm(k, On(9216, dtype=u8), bits=8))                    # the codes do
    _refused(k, lambda: _qmm(k, On(9216, dtype=u8), at=(0, 8706, 8192)))        # the scales do
    _refused(k, lambda: _qmm(k, On(9216, dtype=u8), at=(-16, 8192, 8704)))
    _refused(k, lambda: _qmm(k, On(9216, dtype=u8), group=32))
    _refused(k, lambda: _qmm(k, None))


def test_weights_the_library_refuses_reach_it(k):
    """Widths and groups that do not exist are the library's to name."""
    buf = On(1 << 16, dtype=torch.uint8)
    before = k.lib.calls
    for kw in (dict(bits=5), dict(group=0), dict(group=48), dict(bits=0)):
        assert _qmm(k, buf, **kw) == 0
    assert k.lib.calls == before + 4
