"""smoe_sample where top-k asks for more than a mask leaves (or just as many): all
of it is kept, whatever the other filters are. Rows have one answer, by the distance
that tests/test_sample_borders.py derives."""
import numpy as np
import pytest

from test_gpu_sample import U, _run, want_of
from test_sample_borders import _token

pytestmark = pytest.mark.gpu

KEEP = {"all": (1.0, 0.0), "top_p": (0.9, 0.0), "min_p": (1.0, 0.02), "both": (0.97, 0.01)}


@pytest.mark.parametrize("V", [460, 3001, 20011, 151936])
@pytest.mark.parametrize("mask", ["-inf", "nan"])
@pytest.mark.parametrize("share", [0.001, 0.3, 0.95])
@pytest.mark.parametrize("top", ["one", "inf", "flat"])
@pytest.mark.parametrize("keep", list(KEEP))
def test_top_k_of_more_than_is_left(kernels, V, mask, share, top, keep):
    rng = np.random.default_rng(V + int(share * 1000))
    n = 6
    l = (rng.standard_normal((n, V)) * (0.1 if top == "flat" else 2.5)).astype(np.float32)
    l[rng.random((n, V)) > share] = float(mask)
    l[:, V // 3] = 1.0
    if top == "inf":
        l[:, [5, V - 2]] = np.inf
    left = (~np.isnan(l) & (l > -np.inf)).sum(1)
    k = [V - 1, max(449, left[1]), max(449, left[2] + 1), max(449, left[3] - 1), 449, V - 1]
    p, m = (np.full(n, x, np.float32) for x in KEEP[keep])
    t, u = np.array([1.0, 0.5, 2.0, 1.0, 1.0, 50.0], np.float32), rng.random(n).astype(np.float32)
    tok, lp = _run(kernels, l, t, k, p, m, u, V)
    kernels.sync()
    for i in range(n):
        want, near, room = _token(l[i], t[i], k[i], p[i], m[i], u[i])
        if top == "inf":  # equal masses: exact on both sides
            near = 1.0
        assert near > room, i
        assert tok[i] == want, (i, tok[i], want)
        share_of = want_of(l[i], t[i], k[i], p[i], m[i], u[i])[1]
        # Of two f64 sums, rounded; a kept sum is off by V 2^-s of the largest at most.
        assert abs(lp[i] - share_of) <= U * abs(share_of) + 2.0 ** -25, i


def test_the_same_captured(kernels):
    import torch

    import streamoe_amd as sa

    rng = np.random.default_rng(3)
    V, n = 5003, 5
    l = torch.tensor(rng.standard_normal((n, V)) * 2, dtype=torch.float32, device="cuda")
    l[:, 1000:] = -float("inf")
    k = torch.full((n,), 2000, dtype=torch.int32, device="cuda")
    u = torch.tensor(rng.random(n), dtype=torch.float32, device="cuda")
    tok, lp = torch.zeros(n, dtype=torch.int32, device="cuda"), torch.zeros(n, device="cuda")
    ws = torch.empty(kernels.sample_workspace_size(n, V), dtype=torch.uint8, device="cuda")

    def call():
        assert kernels.sample(l, None, k, None, None, u, n, V, tok, lp, ws) == 0

    graph = sa.capture_graph(kernels, call)
    for _ in range(4):
        u.uniform_(0, 0.999)
        tok.fill_(-5)
        ws.fill_(255)
        graph.replay()
        torch.cuda.synchronize()
        got = tok.cpu().numpy().copy()
        for i in range(n):
            want, near, room = _token(l[i].cpu().numpy(), np.float32(1), 2000, np.float32(1), np.float32(0), np.float32(u[i].item()))
            assert near <= room or got[i] == want
        tok.fill_(-5)
        call()
        kernels.sync()
        assert np.array_equal(got, tok.cpu().numpy())
