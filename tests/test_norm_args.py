"""smoe_rmsnorm's refusals, on the CPU: every argument check comes before any
device call, so a zeroed block of memory stands in for the handle."""
import ctypes as C

import pytest

from refusals import fake_handle, refused


def _call(**kw):
    from streamoe_amd import _abi

    a = dict(h=fake_handle(), x=4096, x_is_bf16=0, residual=8192, norm_w=None, eps=1e-6, n_tokens=3, hidden=256,
             sum_out=None, out=12288, out_is_bf16=0, out_q=None, out_scales=None, q_group=0)
    a.update(kw)
    return _abi.load().smoe_rmsnorm(*[C.c_float(v) if k == "eps" else v for k, v in a.items()])


@pytest.mark.parametrize("kw,code", [
    (dict(h=None), "INVALID_ARG"),
    (dict(x=None), "INVALID_ARG"),
    (dict(n_tokens=0), "INVALID_ARG"),
    (dict(hidden=0), "INVALID_ARG"),
    (dict(out=None), "INVALID_ARG"),                                  # nothing to write
    (dict(out_q=16384), "INVALID_ARG"),                               # codes without scales
    (dict(out_scales=16384), "INVALID_ARG"),                          # scales without codes
    (dict(out_q=16384, out_scales=32768, q_group=16), "UNSUPPORTED_GROUP"),
    (dict(out_q=16384, out_scales=32768, q_group=64, hidden=96), "IN_DIM_NOT_MULTIPLE"),
    (dict(hidden=16385), "UNSUPPORTED_SHAPE"),
    (dict(n_tokens=1 << 24), "UNSUPPORTED_SHAPE"),
    (dict(x=4100), "MISALIGNED"),
    (dict(residual=8200), "MISALIGNED"),
    (dict(norm_w=8194), "MISALIGNED"),
    (dict(sum_out=8196), "MISALIGNED"),
    (dict(out=12290), "MISALIGNED"),
    (dict(out_q=16385, out_scales=32768), "MISALIGNED"),
    (dict(out_q=16384, out_scales=32772), "MISALIGNED"),
])
def test_refusals(kw, code):
    refused(_call(**kw), code)
