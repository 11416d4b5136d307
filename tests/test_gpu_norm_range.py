"""smoe_rmsnorm over the range of f32, against 64-bit arithmetic.

u = 2^-24. The sum is over the rounded r, each off by u: with the root that is
u at most in 1 / rms, which then rounds by u; r itself and the two products
round by u each: |y - y64| <= 6 u |y64| and a little (u^2), whatever the row's
length. Where rms lies above 2^126, 1 / rms is a subnormal f32, off by up to
2^-150 of at least 2^-128, which is 4 u: 10 u in all."""
import numpy as np
import pytest

pytestmark = pytest.mark.gpu

U = 2.0 ** -24


@pytest.mark.parametrize("H", [96, 1023, 4096, 16384])
@pytest.mark.parametrize("size,eps", [(1e-30, 0.0), (1e-21, 0.0), (1.0, 1e-6), (1e17, 1e-6), (1e20, 1e-6), (2e37, 1e-6)])
def test_rows_of_any_size(kernels, H, size, eps):
    import torch

    g = torch.Generator(device="cuda").manual_seed(H)
    x = torch.randn(5, H, generator=g, device="cuda") * size
    r = torch.randn(5, H, generator=g, device="cuda") * size
    y, s = torch.empty(5, H, device="cuda"), torch.empty(5, H, device="cuda")
    q, sc = torch.empty(5, H, dtype=torch.int8, device="cuda"), torch.empty(5, 1, device="cuda")
    assert kernels.rmsnorm(x, r, None, eps, 5, H, s, y, q, sc) == 0
    kernels.sync()
    r64 = x.double() + r.double()
    want = r64 / ((r64 ** 2).mean(1, keepdim=True) + eps).sqrt()
    off = (y.double() - want).abs().cpu().numpy()
    assert torch.all(torch.isfinite(s))
    assert np.all(off <= 10 * U * want.abs().cpu().numpy() + 2.0 ** -126)
    assert torch.all((q.double() * sc.double() - want).abs() <= 0.501 * sc.double() + 2.0 ** -126)


def test_zero_rows_without_eps(kernels):
    import torch

    x = torch.zeros(2, 64, device="cuda")
    x[1] = 3
    y = torch.empty(2, 64, device="cuda")
    assert kernels.rmsnorm(x, None, None, 0.0, 2, 64, None, y) == 0
    kernels.sync()
    assert torch.all(torch.isnan(y[0])) and torch.all(y[1] == 1)
