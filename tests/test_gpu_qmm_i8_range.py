"""smoe_qmm_i8 with scales per group far from one, against 64-bit arithmetic:
every kernel, scales so large that a group's sum times its scale leaves f32's
range while the outputs do not, and scales down to 2^-101. The bound is that of
test_gpu_qmm_i8.py, (2 g + 24) u M; products by powers of two round nothing."""
import numpy as np
import pytest

from test_gpu_qmm_i8 import U, _run, _rows, _want, _weights

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("bits,G", [(4, 64), (3, 32), (8, 128)])
@pytest.mark.parametrize("n,O,K", [
    (8, 200, 512),       # few rows
    (45, 2563, 512),     # two column tiles a block
    (11, 17000, 640),    # few rows of many columns
    (130, 4100, 4096),   # 64 x 64 tiles, shares of the steps
    (400, 4100, 512),    # .. one share
    (500, 7001, 2048),   # 128 x 128 tiles, two shares
    (1000, 6404, 1152),  # .. one
])
def test_scales_of_any_size(kernels, n, O, K, bits, G):
    rng = np.random.default_rng(n + K + bits)
    W = _weights(rng, O, K, bits, G)
    x, sx = _rows(rng, n, K, G)
    rows = np.arange(n) % 3
    sx[rows == 0] *= np.float32(2.0 ** (-94 - 1))    # 2^-101 .. 2^-93
    sx[rows == 2] *= np.float32(2.0 ** (117 - bits))  # up to 4e33, 8e33, 2.5e32
    sx = np.maximum(sx, np.float32(2.0 ** -101))
    y = _run(kernels, W, bits, G, x, sx, G, O).astype(np.float64)
    want, M = _want(*W[2:], x, sx, G, bits)
    assert np.max(M) < 2.0 ** 127
    assert np.all(np.isfinite(y))
    bound = (2 * (K // G) + 24) * U * M + 2.0 ** -126
    assert np.all(np.abs(y - want) <= bound), float(np.max(np.abs(y - want) / bound))


def test_the_largest_scale(kernels):
    """Codes of one group, weights so small that the output has room."""
    import torch

    rng = np.random.default_rng(9)
    top = np.finfo(np.float32).max
    for n, O in ((8, 200), (200, 4100), (11, 17000)):
        W = _weights(rng, O, 512, 4, 64)
        s = W[0][W[1][1]:W[1][1] + W[3].size * 2].view(torch.bfloat16)
        s *= 2.0 ** -24
        b = W[0][W[1][2]:].view(torch.bfloat16)
        b *= 2.0 ** -24
        f = lambda v: v.double().cpu().numpy().reshape(O, -1)
        x, sx = _rows(rng, n, 512, 64)
        x[:, 64:] = 0
        sx[:, 0] = top
        y = _run(kernels, W, 4, 64, x, sx, 64, O)
        want, M = _want(W[2], f(s), f(b), x, sx, 64, 4)
        assert np.all(np.abs(y - want) <= 40 * U * M)
