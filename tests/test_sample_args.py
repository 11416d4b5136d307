"""Refusals of smoe_sample, on the CPU: every argument check comes before any
device call."""
import pytest

from refusals import fake_handle, refused


def _sample(**kw):
    from streamoe_amd import _abi

    a = dict(h=fake_handle(), logits=1 << 20, temperature=4096, top_k=8192, top_p=12288, min_p=16384, u=20480, n_rows=5,
             vocab=1000, out_tokens=24576, out_logprobs=28672, workspace=1 << 24, workspace_bytes=1 << 24)
    a.update(kw)
    return _abi.load().smoe_sample(*a.values())


@pytest.mark.parametrize("kw,code", [
    (dict(h=None), "INVALID_ARG"),
    (dict(logits=None), "INVALID_ARG"),
    (dict(u=None), "INVALID_ARG"),
    (dict(out_tokens=None), "INVALID_ARG"),
    (dict(workspace=None), "INVALID_ARG"),
    (dict(n_rows=0), "INVALID_ARG"),
    (dict(vocab=0), "INVALID_ARG"),
    (dict(n_rows=65536), "UNSUPPORTED_SHAPE"),
    (dict(vocab=(1 << 24) + 1), "UNSUPPORTED_SHAPE"),
    (dict(logits=(1 << 20) + 4), "MISALIGNED"),
    (dict(temperature=4098), "MISALIGNED"),
    (dict(top_k=8193), "MISALIGNED"),
    (dict(out_logprobs=28674), "MISALIGNED"),
    (dict(workspace=(1 << 24) + 64), "MISALIGNED"),
    (dict(workspace_bytes=4096), "WORKSPACE_TOO_SMALL"),
    (dict(out_tokens=20480 + 16), "INVALID_ARG"),          # u
    (dict(out_logprobs=24576), "INVALID_ARG"),             # the tokens
    (dict(out_tokens=(1 << 20) + 19996), "INVALID_ARG"),   # the last logit
    (dict(workspace=1 << 20), "INVALID_ARG"),
    (dict(out_logprobs=4096), "INVALID_ARG"),
])
def test_refusals(kw, code):
    refused(_sample(**kw), code)


def test_workspace_size():
    from streamoe_amd import _abi

    lib = _abi.load()
    assert lib.smoe_sample_workspace_size(1, 1) > 0
    assert lib.smoe_sample_workspace_size(64, 151936) >= 64 * 151936 * 8
    assert lib.smoe_sample_workspace_size(0, 10) == 0
    assert lib.smoe_sample_workspace_size(10, 0) == 0
    assert lib.smoe_sample_workspace_size(65536, 10) == 0
    assert lib.smoe_sample_workspace_size(1, (1 << 24) + 1) == 0
