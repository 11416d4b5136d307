"""Refusals of smoe_beam_select and smoe_beam_reorder, on the CPU: every
argument check comes before any device call."""
import ctypes as C

import pytest

from refusals import fake_handle, refused


def _select(**kw):
    from streamoe_amd import _abi

    a = dict(h=fake_handle(), logits=4096, scores=8192, done=None, pad_token=0, n_requests=2, n_beams=4, vocab=100,
             n_picks=8, out_scores=12288, out_rows=16384, out_tokens=20480, workspace=65536, workspace_bytes=1 << 20)
    a.update(kw)
    return _abi.load().smoe_beam_select(*a.values())


@pytest.mark.parametrize("kw,code", [
    (dict(h=None), "INVALID_ARG"),
    (dict(logits=None), "INVALID_ARG"),
    (dict(scores=None), "INVALID_ARG"),
    (dict(out_rows=None), "INVALID_ARG"),
    (dict(workspace=None), "INVALID_ARG"),
    (dict(n_requests=0), "INVALID_ARG"),
    (dict(vocab=0), "INVALID_ARG"),
    (dict(n_beams=17), "UNSUPPORTED_SHAPE"),
    (dict(vocab=(1 << 28) + 1), "UNSUPPORTED_SHAPE"),
    (dict(n_picks=0), "BAD_K"),
    (dict(n_picks=33), "BAD_K"),
    (dict(n_picks=9, vocab=2), "BAD_K"),               # more than there are continuations
    (dict(n_requests=1 << 26), "UNSUPPORTED_SHAPE"),
    (dict(n_requests=262144), "UNSUPPORTED_SHAPE"),
    (dict(done=24576, pad_token=100), "INVALID_ARG"),
    (dict(out_scores=8192), "INVALID_ARG"),            # in place with more picks than beams
    (dict(logits=4100), "MISALIGNED"),
    (dict(workspace=65536 + 16), "MISALIGNED"),
    (dict(workspace_bytes=64), "WORKSPACE_TOO_SMALL"),
])
def test_select_refusals(kw, code):
    refused(_select(**kw), code)


def test_workspace_size():
    from streamoe_amd import _abi

    lib = _abi.load()
    assert lib.smoe_beam_select_workspace_size(2, 4, 151936, 8) > 0
    assert lib.smoe_beam_select_workspace_size(0, 4, 151936, 8) == 0
    assert lib.smoe_beam_select_workspace_size(2, 17, 151936, 8) == 0


def _reorder(each=None, n=None, **kw):
    from streamoe_amd import _abi

    one = dict(src=1 << 20, dst=1 << 21, src_row_stride=1024, dst_row_stride=1024, src_piece_stride=256,
               dst_piece_stride=256, piece_bytes=100, n_pieces=4, reserved=0)
    states = [dict(one, **s) for s in (each if each is not None else [{}])]
    arr = (_abi.BeamStateC * max(1, len(states)))(*[_abi.BeamStateC(*s.values()) for s in states])
    a = dict(h=fake_handle(), states=arr, n_states=len(states) if n is None else n, rows=4096, n_rows=4, src_rows=4)
    a.update(kw)
    return _abi.load().smoe_beam_reorder(*a.values())


@pytest.mark.parametrize("states,kw,code", [
    ([{}], dict(h=None), "INVALID_ARG"),
    ([{}], dict(states=None), "INVALID_ARG"),
    ([{}], dict(n_states=0), "INVALID_ARG"),
    ([{}], dict(rows=None), "INVALID_ARG"),
    ([{}], dict(n_rows=0), "INVALID_ARG"),
    ([{}], dict(src_rows=0), "INVALID_ARG"),
    ([{}], dict(rows=4098), "MISALIGNED"),
    ([dict(src=None)], {}, "INVALID_ARG"),
    ([dict(n_pieces=0)], {}, "INVALID_ARG"),
    ([dict(reserved=1)], {}, "INVALID_ARG"),
    ([dict(dst=1 << 20)], {}, "INVALID_ARG"),                             # in place
    ([dict(dst=(1 << 20) + 3 * 1024 + 3 * 256 + 99)], {}, "INVALID_ARG"),  # last byte of src
    ([dict(dst_row_stride=0)], {}, "INVALID_ARG"),                        # rows of dst on each other
    ([dict(dst_row_stride=800)], {}, "INVALID_ARG"),
    ([dict(dst_piece_stride=99)], {}, "INVALID_ARG"),
    ([dict(src_row_stride=1 << 63)], {}, "INVALID_ARG"),
    ([dict(piece_bytes=1 << 46, dst=1 << 60, n_pieces=1, dst_row_stride=1 << 46)], {}, "UNSUPPORTED_SHAPE"),
    ([dict(n_pieces=1 << 24, piece_bytes=1, src_piece_stride=1, dst_piece_stride=1, dst_row_stride=1 << 24, dst=1 << 60)], {},
     "UNSUPPORTED_SHAPE"),
    ([{}] * 70 + [dict(n_pieces=0)], {}, "INVALID_ARG"),                  # past the first batch of states
])
def test_reorder_refusals(states, kw, code):
    refused(_reorder(states, **kw), code)
