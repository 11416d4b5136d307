"""smoe_lora's refusals, on the CPU: every argument check comes before any
device call."""
import ctypes as C

import pytest

from refusals import fake_handle, refused

SET = dict(a=1 << 20, b=1 << 24, a_stride=16 * 256 * 2, b_stride=512 * 16 * 2, scale=4096, ranks=None, n_adapters=3,
           max_rank=16)


def _call(over=None, **kw):
    from streamoe_amd import _abi

    s = _abi.AdaptersC(*dict(SET, **(over or {})).values())
    a = dict(h=fake_handle(), adapters=C.byref(s), ids=8192, x=1 << 26, x_is_bf16=0, base=None, y=1 << 27, out_dim=512,
             in_dim=256, n_tokens=5, workspace=1 << 28, workspace_bytes=1 << 20)
    a.update(kw)
    return _abi.load().smoe_lora(*a.values())


@pytest.mark.parametrize("over,kw,code", [
    ({}, dict(h=None), "INVALID_ARG"),
    ({}, dict(adapters=None), "INVALID_ARG"),
    ({}, dict(ids=None), "INVALID_ARG"),
    ({}, dict(x=None), "INVALID_ARG"),
    ({}, dict(y=None), "INVALID_ARG"),
    ({}, dict(workspace=None), "INVALID_ARG"),
    ({}, dict(out_dim=0), "INVALID_ARG"),
    ({}, dict(in_dim=0), "INVALID_ARG"),
    ({}, dict(n_tokens=0), "INVALID_ARG"),
    (dict(a=None), {}, "INVALID_ARG"),
    (dict(b=None), {}, "INVALID_ARG"),
    (dict(scale=None), {}, "INVALID_ARG"),
    (dict(n_adapters=0), {}, "INVALID_ARG"),
    (dict(max_rank=0), {}, "INVALID_ARG"),
    (dict(a_stride=16 * 256 * 2 - 16), {}, "INVALID_ARG"),
    (dict(b_stride=512 * 16 * 2 - 16), {}, "INVALID_ARG"),
    (dict(max_rank=12), {}, "UNSUPPORTED_SHAPE"),
    (dict(max_rank=136), {}, "UNSUPPORTED_SHAPE"),
    (dict(n_adapters=4097), {}, "UNSUPPORTED_SHAPE"),
    ({}, dict(n_tokens=65537), "UNSUPPORTED_SHAPE"),
    ({}, dict(in_dim=252), "UNSUPPORTED_SHAPE"),
    ({}, dict(in_dim=65544), "UNSUPPORTED_SHAPE"),
    (dict(b_stride=4194304 * 32), dict(out_dim=4194304), "UNSUPPORTED_SHAPE"),
    (dict(a=(1 << 20) + 8), {}, "MISALIGNED"),
    (dict(b=(1 << 24) + 2), {}, "MISALIGNED"),
    (dict(a_stride=16 * 256 * 2 + 2), {}, "MISALIGNED"),
    (dict(scale=4098), {}, "MISALIGNED"),
    (dict(ranks=4098), {}, "MISALIGNED"),
    ({}, dict(x=(1 << 26) + 4), "MISALIGNED"),
    ({}, dict(y=(1 << 27) + 2), "MISALIGNED"),
    ({}, dict(base=(1 << 27) + 2), "MISALIGNED"),
    ({}, dict(workspace=(1 << 28) + 64), "MISALIGNED"),
    ({}, dict(workspace_bytes=100), "WORKSPACE_TOO_SMALL"),
])
def test_refusals(over, kw, code):
    refused(_call(over, **kw), code)


def test_workspace_size():
    from streamoe_amd import _abi

    size = lambda n, **kw: _abi.load().smoe_lora_workspace_size(C.byref(_abi.AdaptersC(*dict(SET, **kw).values())), n)
    assert size(5) > 0 and size(1000) > size(5)
    assert size(0) == 0 and size(5, max_rank=12) == 0 and size(65537) == 0


def test_struct_holds_for_its_own_views():
    """Tensors that change their shape in place leave the set as it was; a
    storage that moves is looked at again."""
    import torch

    import streamoe_amd as sa

    z = lambda *s: torch.zeros(*s, dtype=torch.bfloat16)
    a, b = z(3, 16, 32), z(3, 48, 16)
    s = sa.Adapters(a, b, torch.ones(3))
    a.resize_(3, 8, 16)
    b.transpose_(0, 2)
    c = s.c()
    assert (c.n_adapters, c.max_rank, c.a_stride, c.b_stride) == (3, 16, 1024, 1536)
    a.resize_(300, 16, 32)
    assert s.c().a == a.data_ptr()
    with pytest.raises(sa.SmoeError):
        sa.Adapters(z(3, 16, 32), z(3, 48, 8), torch.ones(3)).c()
