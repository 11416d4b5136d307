"""smoe_qmm_i8's refusals, on the CPU: every argument check comes before any
device call."""
import ctypes as C

import pytest

from refusals import fake_handle, refused


def _call(over=None, **kw):
    from streamoe_amd import _abi

    q = _abi.QWeights(*dict(dict(base=1 << 20, packed_offset=0, scales_offset=1 << 16, biases_offset=1 << 17,
                                 group_size=64, bits=4), **(over or {})).values())
    a = dict(h=fake_handle(), w=C.byref(q), x=1 << 24, x_scales=1 << 25, x_group=0, y=1 << 26, out_dim=100, in_dim=256,
             n_tokens=5)
    a.update(kw)
    return _abi.load().smoe_qmm_i8(*a.values())


@pytest.mark.parametrize("over,kw,code", [
    ({}, dict(h=None), "INVALID_ARG"),
    ({}, dict(w=None), "INVALID_ARG"),
    ({}, dict(x=None), "INVALID_ARG"),
    ({}, dict(x_scales=None), "INVALID_ARG"),
    ({}, dict(y=None), "INVALID_ARG"),
    ({}, dict(out_dim=0), "INVALID_ARG"),
    ({}, dict(in_dim=0), "INVALID_ARG"),
    ({}, dict(n_tokens=0), "INVALID_ARG"),
    (dict(base=None), {}, "INVALID_ARG"),
    (dict(bits=5), {}, "UNSUPPORTED_BITS"),
    (dict(group_size=16), {}, "UNSUPPORTED_GROUP"),
    ({}, dict(x_group=128), "UNSUPPORTED_GROUP"),
    ({}, dict(in_dim=288), "IN_DIM_NOT_MULTIPLE"),
    ({}, dict(in_dim=16448), "UNSUPPORTED_SHAPE"),
    ({}, dict(n_tokens=65535 * 16 + 1), "UNSUPPORTED_SHAPE"),
    ({}, dict(out_dim=(1 << 28) + 1), "UNSUPPORTED_SHAPE"),
    (dict(packed_offset=8), {}, "MISALIGNED"),
    (dict(scales_offset=1), {}, "MISALIGNED"),
    ({}, dict(x=(1 << 24) + 8), "MISALIGNED"),
    ({}, dict(x_scales=(1 << 25) + 2), "MISALIGNED"),
    ({}, dict(y=(1 << 26) + 2), "MISALIGNED"),
])
def test_refusals(over, kw, code):
    refused(_call(over, **kw), code)
