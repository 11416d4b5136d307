"""smoe_rmsnorm against 64-bit arithmetic.

Bounds, in units of u = 2^-24 (f32's rounding): r is one addition, off by at
most u |r|. The sum of squares adds up to hidden / 256 + 8 terms in a chain
(a thread's values, then the wave and the block), each rounding by u, with the
squares of rounded r: relative (hidden / 256 + 12) u; the root halves it, the
mean's division, the root and the reciprocal add 3 u, and y = r inv w three
more with r's own. So |y - y64| <= (hidden / 512 + 14) u |y64| and 2^-8 |y| more
where y is bf16, plus the smallest normal float. A code is y 127 / top with two
more roundings of a value up to 127, rounded to an integer: the value it stands
for is off by at most (0.5 + 127 (hidden / 256 + 40) u) scales."""
import numpy as np
import pytest

pytestmark = pytest.mark.gpu

U = 2.0 ** -24


def _run(kernels, n, H, xb, wb, out, q, res=True, seed=0, alias=False, fix=None):
    import torch

    g = torch.Generator(device="cuda").manual_seed(seed)
    x = torch.randn(n, H, generator=g, device="cuda")
    r = torch.randn(n, H, generator=g, device="cuda") * 3 if res else None
    if fix:
        fix(x, r)
    x = x.to(torch.bfloat16) if xb else x
    w = (1 + 0.1 * torch.randn(H, generator=g, device="cuda")).to(torch.bfloat16) if wb else None
    x64 = x.double().cpu().numpy()
    r64 = x64 + (r.double().cpu().numpy() if res else 0)
    y = None if out is None else torch.full((n, H), 7.0, device="cuda", dtype=getattr(torch, out))
    s = torch.full((n, H), 7.0, device="cuda")
    if alias:  # in place: the residual becomes the sum, x the norm
        s, y = r, x
    codes = sc = None
    if q is not None:
        codes = torch.full((n, H), 99, dtype=torch.int8, device="cuda")
        sc = torch.full((n, H // (q or H)), 7.0, device="cuda")
    assert kernels.rmsnorm(x, r, w, 1e-6, n, H, s, y, codes, sc, q or 0) == 0
    kernels.sync()
    with np.errstate(all="ignore"):
        y64 = r64 / np.sqrt((r64 ** 2).sum(1, keepdims=True) / H + 1e-6)
        if wb:
            y64 = y64 * w.double().cpu().numpy()
    c = lambda t: None if t is None else t.double().cpu().numpy()
    return r64, y64, c(s), c(y), c(codes), c(sc)


def _check(n, H, out, q, r64, y64, s, y, codes, sc):
    tiny = 2.0 ** -126
    assert np.all(np.abs(s - r64) <= U * np.abs(r64) + tiny)
    rel = (H / 512 + 14) * U
    if y is not None:
        assert np.all(np.abs(y - y64) <= (rel + (2.0 ** -8 if out == "bfloat16" else 0)) * np.abs(y64) + tiny)
    if q is not None:
        G = q or H
        v = y64.reshape(n, H // G, G)
        top = np.abs(v).max(2)
        assert np.all(np.abs(sc - top / 127) <= (rel + 3 * U) * top / 127 + tiny)
        got = codes.reshape(n, H // G, G)
        assert np.all(np.abs(got) <= 127)
        assert np.all(np.abs(got * sc[:, :, None] - v) <= (0.5 + 127 * (H / 256 + 40) * U) * sc[:, :, None] + tiny)


@pytest.mark.parametrize("n,H,xb,wb,out,q", [
    (1, 1, False, True, "float32", None),
    (1, 1, True, True, "bfloat16", 0),
    (3, 7, True, True, "float32", 0),
    (2, 32, False, True, None, 32),
    (5, 96, True, False, "bfloat16", 32),
    (1, 2048, False, True, "float32", None),
    (4, 2056, False, True, "bfloat16", 0),
    (17, 2560, True, True, "bfloat16", 64),
    (3, 4096, False, True, "float32", 128),
    (2, 4097, False, True, "float32", 0),
    (33, 7168, True, True, "bfloat16", 128),
    (2, 16384, True, True, "float32", 0),
    (2, 16383, False, True, "bfloat16", 0),
    (1000, 640, False, True, None, 64),
])
def test_rmsnorm(kernels, n, H, xb, wb, out, q):
    _check(n, H, out, q, *_run(kernels, n, H, xb, wb, out, q, seed=n + H))


def test_without_residual(kernels):
    _check(5, 2048, "float32", 64, *_run(kernels, 5, 2048, False, True, "float32", 64, res=False))


@pytest.mark.parametrize("H", [513, 2048, 16384])
def test_in_place(kernels, H):
    _check(6, H, "float32", 0, *_run(kernels, 6, H, False, True, "float32", 0, alias=True))


def test_zero_rows_and_tiny_groups(kernels):
    def fix(x, r):
        x[0] = 0
        r[0] = 0                      # a row of zeros
        x[1, :64] = 0
        r[1, :64] = 0                 # a group of zeros in an ordinary row
        x[2, 64:128] = 1e-37
        r[2, 64:128] = 0              # below the codes' range

    r64, y64, s, y, codes, sc = _run(kernels, 3, 256, False, False, "float32", 64, fix=fix)
    _check(3, 256, "float32", None, r64, y64, s, y, codes, sc)
    assert np.all(y[0] == 0) and np.all(codes[0] == 0) and np.all(sc[0] == 0)
    assert np.all(codes[1, :64] == 0) and sc[1, 0] == 0 and np.all(sc[1, 1:] > 0)
    assert np.all(codes[2, 64:128] == 0) and sc[2, 1] == 0 and np.all(y[2, 64:128] != 0)


def test_nan_and_infinity_stay_in_their_row(kernels):
    def fix(x, r):
        x[1, 70] = float("nan")
        x[2, 3] = float("inf")

    r64, y64, s, y, codes, sc = _run(kernels, 4, 192, False, True, "float32", 64, fix=fix)
    assert np.all(np.isnan(y[1])) and np.all(np.isnan(sc[1])) and np.all(codes[1] == 0)
    assert np.isnan(y[2, 3]) and np.all(np.delete(y[2], 3) == 0)  # x / inf, as the definition gives
    assert np.isnan(sc[2, 0]) and np.all(sc[2, 1:] == 0) and np.all(codes[2] == 0)
    keep = [0, 3]
    _check(2, 192, "float32", 64, *(t[keep] for t in (r64, y64, s, y, codes, sc)))


def test_rows_behind_the_last_stay(kernels):
    import torch

    x = torch.randn(4, 2048, device="cuda")
    out = torch.full((4, 2048), 5.0, device="cuda")
    q = torch.full((4, 2048), 5, dtype=torch.int8, device="cuda")
    sc = torch.full((4, 32), 5.0, device="cuda")
    assert kernels.rmsnorm(x, None, None, 1e-6, 3, 2048, None, out, q, sc, 64) == 0
    kernels.sync()
    assert torch.all(out[3] == 5) and torch.all(q[3] == 5) and torch.all(sc[3] == 5)


def test_misfit_tensors_are_refused(kernels):
    import torch

    x = torch.randn(8, 256, device="cuda")
    out = torch.empty(8, 256, device="cuda")
    bad = 1  # SMOE_ERR_INVALID_ARG
    assert kernels.rmsnorm(x.t(), None, None, 1e-6, 8, 256, None, out) == bad       # not dense
    assert kernels.rmsnorm(x, None, None, 1e-6, 9, 256, None, out) == bad           # too few rows
    assert kernels.rmsnorm(x.cpu(), None, None, 1e-6, 8, 256, None, out) == bad     # host memory
    assert kernels.rmsnorm(x, x.double(), None, 1e-6, 8, 256, None, out) == bad     # f64
    assert kernels.rmsnorm(x, None, None, 1e-6, 8, 256, None, None) == bad          # nothing to write


def test_graph_replays(kernels):
    import torch

    import streamoe_amd as sa

    x = torch.randn(6, 2560, device="cuda")
    r = torch.randn(6, 2560, device="cuda")
    w = torch.ones(2560, device="cuda").to(torch.bfloat16)
    s, y = torch.empty_like(x), torch.empty_like(x)
    q = torch.empty(6, 2560, dtype=torch.int8, device="cuda")
    sc = torch.empty(6, 40, device="cuda")
    call = lambda: sa.check(kernels.rmsnorm(x, r, w, 1e-6, 6, 2560, s, y, q, sc, 64), "rmsnorm")
    graph = sa.capture_graph(kernels, call)
    for i in range(3):
        x.normal_()
        graph.replay()
        torch.cuda.synchronize()
        got = [t.clone() for t in (s, y, q, sc)]
        call()
        kernels.sync()
        assert all(torch.equal(a, b) for a, b in zip(got, (s, y, q, sc)))
