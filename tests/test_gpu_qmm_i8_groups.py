"""smoe_qmm_i8 of few rows and many columns at every count of groups modulo
eight (the rows' sums are formed eight groups at a time). Bound as in
test_gpu_qmm_i8.py; repeated calls give the same bits."""
import numpy as np
import pytest

from test_gpu_qmm_i8 import U, _rows, _run, _want, _weights

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("bits", [4, 3, 8])
@pytest.mark.parametrize("G", [32, 64, 128])
@pytest.mark.parametrize("grouped", [False, True])
def test_counts_of_groups(kernels, bits, G, grouped):
    rng = np.random.default_rng(bits + G)
    n, O, xg = 11, 16500, G if grouped else 0
    for g in (2, 3, 4, 5, 6, 7, 8, 10, 15, 23, 31):
        K = g * G
        W = _weights(rng, O, K, bits, G)
        x, sx = _rows(rng, n, K, xg)
        want, M = _want(*W[2:], x, sx, G, bits)
        y = _run(kernels, W, bits, G, x, sx, xg, O)
        assert np.all(np.abs(y - want) <= (2 * g + 24) * U * M + 1e-30), g
        for _ in range(2):
            assert np.array_equal(y, _run(kernels, W, bits, G, x, sx, xg, O)), g
