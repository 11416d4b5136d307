"""smoe_beam_select where rows hold the same logits: their log-sum-exps are the
same number, wherever a row lies in memory, so equal scores tie and the lower
row comes first. Nothing is off: rows and tokens are compared for equality, and
so are the scores of requests that are copies of one another."""
import numpy as np
import pytest

from test_gpu_beam import _run, _want

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("V", [3, 5, 101, 1023, 4095, 4097, 4098, 5003, 12291, 30001, 151937])
@pytest.mark.parametrize("R,W,P", [(1, 4, 8), (3, 5, 10), (40, 3, 7)])
def test_copies_of_a_row(kernels, R, W, P, V):
    rng = np.random.default_rng(V + R)
    l = np.repeat((rng.standard_normal((R, 1, V)) * 2.5).astype(np.float32), W, 1).reshape(R * W, V)
    sc = np.repeat(-rng.random(R).astype(np.float32), W)
    _, rows, tok = _run(kernels, l, sc, None, 0, R, W, V, P)
    _, wr, wt = _want(l, sc, None, 0, R, W, V, P)
    assert np.array_equal(rows, wr) and np.array_equal(tok, wt)


@pytest.mark.parametrize("V", [7, 4099, 20002, 70001])
def test_copies_of_a_request(kernels, V):
    rng = np.random.default_rng(V)
    R, W, P = 37, 3, 6
    one = (rng.standard_normal((W, V)) * 2.5).astype(np.float32)
    sc = -rng.random(W).astype(np.float32)
    v, rows, tok = _run(kernels, np.tile(one, (R, 1)), np.tile(sc, R), None, 0, R, W, V, P)
    assert np.array_equal(v, np.tile(v[:1], (R, 1))) and np.array_equal(tok, np.tile(tok[:1], (R, 1)))
    assert np.array_equal(rows, rows[:1] + W * np.arange(R)[:, None])
