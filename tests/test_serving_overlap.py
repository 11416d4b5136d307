"""smoe_qmm_i8, smoe_lora and smoe_beam_select refuse outputs that overlap what
they read, but for the pairs that the interface allows. On the CPU: the checks
come before any device call."""
import pytest

from refusals import refused
from test_beam_args import _select
from test_lora_args import _call as _lora
from test_qmm_i8_args import _call as _qmm

X, SX, Y = 1 << 24, 1 << 25, 1 << 26


@pytest.mark.parametrize("kw", [
    dict(y=X), dict(y=SX), dict(y=X - 100 * 5 * 4 + 16), dict(y=X + 256 * 5 - 16), dict(y=SX + 16),
    dict(y=1 << 20), dict(y=(1 << 20) + (1 << 16) + 16), dict(y=(1 << 20) + (1 << 17) + 100 * 4 * 2 - 16),
])
def test_qmm_i8(kw):
    refused(_qmm(**kw), "INVALID_ARG")


@pytest.mark.parametrize("kw", [
    dict(y=1 << 26), dict(y=(1 << 26) + 5 * 256 * 4 - 16), dict(y=8192), dict(y=4096), dict(y=1 << 20),
    dict(y=(1 << 20) + 3 * 16 * 256 * 2 - 16), dict(y=1 << 24), dict(y=1 << 28),
    dict(base=(1 << 27) + 512 * 4),                           # another row's place
    dict(base=(1 << 27) - 16),
    dict(workspace=1 << 26), dict(workspace=1 << 24),
    dict(base=(1 << 28) + 256),
])
def test_lora(kw):
    refused(_lora(**kw), "INVALID_ARG")


@pytest.mark.parametrize("kw", [
    dict(out_scores=4096), dict(out_rows=4096 + 3200 - 4), dict(out_tokens=8192), dict(out_rows=8192 + 28),
    dict(out_rows=12288), dict(out_tokens=16384 + 60), dict(out_scores=20480 - 60),
    dict(out_scores=8192 + 4, n_picks=4),                     # in place, but shifted
    dict(done=16384), dict(workspace=4096), dict(workspace=8192 - 256), dict(out_scores=65536),
])
def test_beam_select(kw):
    refused(_select(**kw), "INVALID_ARG")
