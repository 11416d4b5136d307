"""smoe_qmm_i8 against 64-bit arithmetic.

Bound per output, u = 2^-24: a group's sums of codes are exact integers below
2^24 (128 * 255 * 128), so each is one f32; sx s, the bias's sum (b + 128 s and
its product) and the two additions round by u each. With g = in_dim / group and
M = sum_g |sx| (|s| |S_g| + (|b| + 256 |s|) |X_g|) (the 256 only for 8-bit
codes, which enter less 128: S_g = sum (q - 128) x), the 2 g additions and the
joining of up to eight shares round by at most (2 g + 16) u M, the terms
themselves by 4 u M: |y - y64| <= (2 g + 24) u M."""
import numpy as np
import pytest

pytestmark = pytest.mark.gpu

U = 2.0 ** -24


def _weights(rng, O, K, bits, G):
    """(device buffer, offsets, codes, scales, biases)."""
    import torch

    from helpers import gen_quant_matrix
    import oracle

    codes, s, b = gen_quant_matrix(rng, O, K, G, bits)
    raw = codes.view(np.uint8).reshape(O, -1)
    if bits == 8:
        q = raw.astype(np.int64)
    elif bits == 4:
        q = np.stack([raw & 15, raw >> 4], 2).reshape(O, K).astype(np.int64)
    else:
        p = raw.reshape(O, K // 8, 3).astype(np.int64)
        p = p[..., 0] | p[..., 1] << 8 | p[..., 2] << 16
        q = np.stack([p >> (3 * i) & 7 for i in range(8)], 2).reshape(O, K)
    at_s = (raw.size + 15) // 16 * 16
    at_b = at_s + s.size * 2 + 2  # two bytes off: scales and biases of any 2-byte address
    buf = np.zeros(at_b + b.size * 2, np.uint8)
    buf[:raw.size] = raw.ravel()
    buf[at_s:at_s + s.size * 2] = s.view(np.uint8).ravel()
    buf[at_b:] = b.view(np.uint8).ravel()
    f = lambda v: oracle.bf16_to_f32(v).astype(np.float64).reshape(O, K // G)
    return torch.from_numpy(buf).cuda(), (0, at_s, at_b), q, f(s), f(b)


def _rows(rng, n, K, xg):
    return rng.integers(-128, 128, (n, K)).astype(np.int8), (np.abs(rng.standard_normal((n, K // (xg or K)))) * .01 +
                                                             1e-3).astype(np.float32)


def _want(q, s, b, x, sx, G, bits):
    n, K = x.shape
    O, g = s.shape
    xs = x.astype(np.float64).reshape(n, g, G)
    sc = np.broadcast_to(sx.astype(np.float64), (n, g)) if sx.shape[1] == 1 else sx.astype(np.float64)
    y, M = np.zeros((n, O)), np.zeros((n, O))
    off = 128 if bits == 8 else 0
    for i in range(g):
        w = (q[:, i * G:(i + 1) * G] - off).astype(np.float64)
        S, X = xs[:, i] @ w.T, xs[:, i].sum(1, keepdims=True)
        y += sc[:, i:i + 1] * (s[:, i] * S + (b[:, i] + off * s[:, i]) * X)
        M += np.abs(sc[:, i:i + 1]) * (np.abs(s[:, i] * S) + (np.abs(b[:, i]) + 2 * off * np.abs(s[:, i])) * np.abs(X))
    return y, M


def _run(kernels, W, bits, G, x, sx, xg, O):
    import torch

    import streamoe_amd as sa

    n, K = x.shape
    y = torch.full((n + 1, O), 7.0, device="cuda")
    qw = sa.QuantWeights(W[0], *W[1], G, bits)
    assert kernels.qmm_i8(qw, torch.from_numpy(x).cuda(), torch.from_numpy(sx).cuda(), xg, y, O, K, n) == 0
    kernels.sync()
    assert torch.all(y[n] == 7)
    return y[:n].cpu().numpy()


def _check(kernels, n, O, K, bits, G, xg, seed=0):
    rng = np.random.default_rng(seed + n + O + K)
    W = _weights(rng, O, K, bits, G)
    x, sx = _rows(rng, n, K, xg)
    y = _run(kernels, W, bits, G, x, sx, xg, O)
    want, M = _want(*W[2:], x, sx, G, bits)
    bound = (2 * (K // G) + 24) * U * M + 1e-30
    assert np.all(np.abs(y - want) <= bound), float(np.max(np.abs(y - want) / bound))


@pytest.mark.parametrize("bits", [4, 3, 8])
@pytest.mark.parametrize("G", [32, 64, 128])
@pytest.mark.parametrize("grouped", [False, True])
def test_every_layout(kernels, bits, G, grouped):
    for n, O, K in [(1, 1, G), (2, 17, 3 * G), (16, 64, 640), (17, 130, 1024), (5, 333, 7 * 128)]:
        _check(kernels, n, O, K, bits, G, G if grouped else 0)


@pytest.mark.parametrize("n,O,K,bits,G,xg", [
    (1, 4096, 2048, 4, 64, 0), (4, 4096, 2048, 4, 64, 64), (3, 640, 2560, 3, 128, 0), (15, 2560, 640, 8, 32, 32),
    (33, 2048, 512, 4, 64, 64), (64, 1030, 7168, 4, 128, 128), (65, 300, 2048, 8, 64, 0), (100, 2048, 2048, 3, 32, 32),
    (129, 4100, 1024, 4, 64, 0), (257, 512, 4096, 4, 32, 0), (513, 520, 1088, 4, 64, 64), (1000, 1000, 2048, 8, 128, 128),
    (16, 20000, 2048, 4, 64, 0), (2, 50, 16384, 4, 64, 64), (40, 70, 16384, 8, 32, 0), (300, 24, 16384, 3, 128, 0),
])
def test_sizes(kernels, n, O, K, bits, G, xg):
    _check(kernels, n, O, K, bits, G, xg)


@pytest.mark.parametrize("bits,G,grouped", [(4, 64, False), (3, 64, True), (8, 128, False), (4, 32, True), (8, 32, False),
                                            (3, 128, True)])
@pytest.mark.parametrize("n,O,steps", [
    (31, 2090, 5),     # two row tiles a block
    (45, 2563, 4),     # two column tiles a block
    (64, 2600, 11),    # four tiles a block
    (100, 2560, 3),    # four tiles a block, four waves
    (130, 4100, 33),   # 64 x 64 tiles, four shares of the steps
    (129, 4096, 8),    # .. or fewer where the groups do not divide
    (390, 4100, 17),   # .. two shares
    (400, 4100, 4),    # .. one
    (500, 7001, 17),   # 128 x 128 tiles, two shares
    (1000, 6404, 9),   # .. one
])
def test_every_kernel(kernels, n, O, steps, bits, G, grouped):
    """Sizes that every kernel and tile takes, the last step short of 128 inputs
    where the group allows."""
    K = steps * 128 - (128 - G)
    _check(kernels, n, O, K, bits, G, G if grouped else 0)


@pytest.mark.parametrize("bits", [4, 3, 8])
@pytest.mark.parametrize("G", [32, 64, 128])
@pytest.mark.parametrize("grouped", [False, True])
def test_many_columns(kernels, bits, G, grouped):
    """Vocabulary-wide outputs of few rows; groups that end inside a round of
    loads, odd counts of groups."""
    for n, O, K in [(1, 16385, 3 * G), (16, 20007, 640), (9, 33000, 9 * G), (5, 16400, 1152), (7, 17000, G),
                    (2, 16399, 2 * G)]:
        _check(kernels, n, O, K, bits, G, G if grouped else 0)


@pytest.mark.parametrize("n,O,K,bits,G,xg", [
    (3, 16500, 8192, 4, 64, 0), (16, 16500, 7168, 8, 128, 128), (13, 16500, 7168, 3, 32, 32), (4, 16500, 8192, 8, 64, 64),
])
def test_many_columns_of_long_rows(kernels, n, O, K, bits, G, xg):
    """Rows that take most of a CU's LDS, or do not fit it."""
    _check(kernels, n, O, K, bits, G, xg)


def test_largest_codes(kernels):
    """The extreme codes of both sides in whole groups: the integer sums' range."""
    rng = np.random.default_rng(3)
    for bits, G in [(4, 64), (8, 128), (3, 32)]:
        W = list(_weights(rng, 40, 4 * G, bits, G))
        W[0][:W[1][1]] = 255
        W[2][:] = 2 ** bits - 1
        for v in (-128, 127):
            x = np.full((20, 4 * G), v, np.int8)
            sx = np.ones((20, 4), np.float32)
            y = _run(kernels, W, bits, G, x, sx, G, 40)
            want, M = _want(*W[2:], x, sx, G, bits)
            assert np.all(np.abs(y - want) <= 32 * U * M)


def test_nan_and_infinite_scales_stay_in_their_row(kernels):
    rng = np.random.default_rng(4)
    for n, O in ((8, 200), (200, 200), (11, 17000)):
        W = _weights(rng, O, 512, 4, 64)
        for xg in (0, 64):
            x, sx = _rows(rng, n, 512, xg)
            clean = _run(kernels, W, 4, 64, x, sx, xg, O)
            sx[3, -1] = np.nan
            sx[5, 0] = np.inf
            y = _run(kernels, W, 4, 64, x, sx, xg, O)
            assert np.all(np.isnan(y[3])) and not np.any(np.isfinite(y[5]))
            keep = [i for i in range(n) if i not in (3, 5)]
            assert np.array_equal(y[keep], clean[keep])


def test_misfit_tensors_are_refused(kernels):
    import torch

    import streamoe_amd as sa

    W = _weights(np.random.default_rng(5), 64, 256, 4, 64)
    qw = sa.QuantWeights(W[0], *W[1], 64, 4)
    x = torch.zeros(4, 256, dtype=torch.int8, device="cuda")
    sx, y = torch.ones(4, 4, device="cuda"), torch.empty(4, 64, device="cuda")
    assert kernels.qmm_i8(qw, x, sx, 64, y, 64, 256, 4) == 0
    assert kernels.qmm_i8(qw, x, sx, 64, y, 64, 256, 5) == 1
    assert kernels.qmm_i8(qw, x.float(), sx, 64, y, 64, 256, 4) == 1
    assert kernels.qmm_i8(qw, x, sx[:2], 64, y, 64, 256, 4) == 1
    assert kernels.qmm_i8(qw, x, sx, 64, y.t(), 64, 256, 4) == 1
    assert kernels.qmm_i8(qw, x, sx, 32, y, 64, 256, 2) == 5  # UNSUPPORTED_GROUP
    kernels.sync()


def test_graph_replays(kernels):
    import torch

    import streamoe_amd as sa

    W = _weights(np.random.default_rng(6), 300, 1024, 4, 64)
    qw = sa.QuantWeights(W[0], *W[1], 64, 4)
    for n in (3, 90):
        x = torch.zeros(n, 1024, dtype=torch.int8, device="cuda")
        sx, y = torch.rand(n, device="cuda"), torch.empty(n, 300, device="cuda")
        call = lambda: sa.check(kernels.qmm_i8(qw, x, sx, 0, y, 300, 1024, n), "qmm_i8")
        graph = sa.capture_graph(kernels, call)
        for _ in range(3):
            x.random_(-127, 128)
            graph.replay()
            torch.cuda.synchronize()
            got = y.clone()
            call()
            kernels.sync()
            assert torch.equal(got, y)
