"""smoe_qmm_i8's largest sizes together, on the CPU: outputs that no launch has
blocks for are refused before any device call."""
import pytest

from refusals import refused
from test_qmm_i8_args import _call


@pytest.mark.parametrize("n,out_dim", [(65535 * 16, 1 << 28), (65535 * 16, 1 << 26), (1 << 19, 1 << 27)])
def test_more_blocks_than_a_launch_holds(n, out_dim):
    # 128 x 128 outputs a block, fewer than 2^24 blocks
    assert (n + 127) // 128 * ((out_dim + 127) // 128) >= 1 << 24
    refused(_call(dict(scales_offset=1 << 40, biases_offset=1 << 41), n_tokens=n, out_dim=out_dim), "UNSUPPORTED_SHAPE")
