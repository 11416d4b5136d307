"""The 8-bit rows of smoe_rmsnorm against their own definition, bit by bit:
scale = max|y| / 127 and code = y / scale rounded to nearest even, both
quotients f32's, with y the f32 row that the same call writes. Nothing is off:
a quotient rounded once is one number, and so is its nearest integer."""
import numpy as np
import pytest

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("n,H,xb,q", [(700, 4096, False, 64), (300, 7168, True, 128), (900, 2048, False, 0),
                                      (400, 2560, True, 32), (500, 1023, False, 0), (60, 16384, False, 0)])
def test_codes_are_the_rounded_quotients(kernels, n, H, xb, q):
    import torch

    g = torch.Generator(device="cuda").manual_seed(n + H)
    x = torch.randn(n, H, generator=g, device="cuda")
    x = x.to(torch.bfloat16) if xb else x
    w = (1 + 0.1 * torch.randn(H, generator=g, device="cuda")).to(torch.bfloat16)
    y = torch.empty(n, H, device="cuda")
    codes = torch.empty(n, H, dtype=torch.int8, device="cuda")
    sc = torch.empty(n, H // (q or H), device="cuda")
    assert kernels.rmsnorm(x, None, w, 1e-6, n, H, None, y, codes, sc, q) == 0
    kernels.sync()
    v = y.cpu().numpy().reshape(n, -1, q or H)
    s = np.abs(v).max(2) / np.float32(127)
    assert np.array_equal(sc.cpu().numpy(), s)
    want = np.rint(v / s[:, :, None])
    assert v.dtype == s.dtype == np.float32
    assert np.array_equal(codes.cpu().numpy().reshape(v.shape), want)
