"""smoe_qmm_i8 of more than 16 rows and a vocabulary of columns, at row counts on
both sides of its tiles. Bound as in test_gpu_qmm_i8.py."""
import numpy as np
import pytest

from test_gpu_qmm_i8 import U, _rows, _run, _want, _weights

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("bits,G,xg", [(4, 64, 0), (8, 128, 128), (3, 32, 32)])
def test_rows_of_a_batch(kernels, bits, G, xg):
    O, K = 50003, 1024
    rng = np.random.default_rng(bits)
    W = _weights(rng, O, K, bits, G)
    x, sx = _rows(rng, 192, K, xg)
    want, M = _want(*W[2:], x, sx, G, bits)
    for n in (17, 64, 65, 128, 130, 192):
        y = _run(kernels, W, bits, G, x[:n], sx[:n], xg, O)
        assert np.all(np.abs(y - want[:n]) <= (2 * (K // G) + 24) * U * M[:n] + 1e-30), n
