"""smoe_rmsnorm refuses buffers that overlap, but for the in-place pairs of one
type (whose rows each block reads before it writes them). On the CPU: the checks
come before any device call."""
import ctypes as C

import pytest

from refusals import fake_handle, refused

N, H = 4, 256
ROWS = N * H * 4  # bytes of f32 rows


def _call(**kw):
    from streamoe_amd import _abi

    a = dict(h=fake_handle(), x=1 << 20, x_is_bf16=0, residual=2 << 20, norm_w=3 << 20, eps=1e-6, n_tokens=N, hidden=H,
             sum_out=4 << 20, out=5 << 20, out_is_bf16=0, out_q=6 << 20, out_scales=7 << 20, q_group=64)
    a.update(kw)
    return _abi.load().smoe_rmsnorm(*[C.c_float(v) if k == "eps" else v for k, v in a.items()])


@pytest.mark.parametrize("kw", [
    dict(out=1 << 20, out_is_bf16=1),                    # bf16 rows over f32 ones: another row's x
    dict(out=1 << 20, x_is_bf16=1),                      # and the other way round
    dict(sum_out=1 << 20, x_is_bf16=1),
    dict(out=2 << 20, out_is_bf16=1),
    dict(out=(1 << 20) + H * 4),                         # one row further
    dict(sum_out=(2 << 20) - 16),
    dict(out=4 << 20),                                   # two outputs in one place
    dict(out_q=(4 << 20) + ROWS - 16),
    dict(out_q=1 << 20),
    dict(out_q=5 << 20),
    dict(out_scales=2 << 20),
    dict(out_scales=(6 << 20) + N * H - 16),
    dict(out=3 << 20),                                   # the weight
    dict(out_q=(3 << 20) + H * 2 - 16),
])
def test_overlaps_are_refused(kw):
    refused(_call(**kw), "INVALID_ARG")
