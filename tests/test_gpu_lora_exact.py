"""smoe_lora keeps f32: one input of a row and one column of an output's B are
not zero, so y[o] = scale B[o, j] A[j, k] x[k] has no sums to round, only the
products. u = 2^-24: A x enters as three exact parts of x, of which each
addition is off by at most an f32 step (2 u), the scale's product by u, and the
second product again by three steps: 13 u, held to 16 u |y|. Rows with f32's
largest numbers among them."""
import numpy as np
import pytest

pytestmark = pytest.mark.gpu

U = 2.0 ** -24


@pytest.mark.parametrize("n,K,O,N,r", [
    (5, 64, 100, 3, 8), (16, 512, 260, 4, 32), (40, 512, 300, 9, 64),     # both products in one launch
    (40, 4096, 300, 9, 16), (9, 2048, 64, 4, 128),                        # two launches, items by wave
    (200, 2048, 520, 12, 40), (300, 264, 100, 2, 128),                    # .. by block
    (1500, 256, 132, 7, 24), (70, 96, 64, 1100, 8),                       # with a plan
])
def test_single_products(kernels, n, K, O, N, r):
    import torch

    import streamoe_amd as sa

    g = torch.Generator(device="cuda").manual_seed(n + K)
    rn = lambda *s: torch.randn(*s, generator=g, device="cuda")
    ri = lambda hi, *s: torch.randint(0, hi, s, generator=g, device="cuda")
    x = torch.zeros(n, K, device="cuda")
    at = ri(K, n)
    val = rn(n) + 2.0
    val[n // 2] = torch.finfo(torch.float32).max
    x[torch.arange(n, device="cuda"), at] = val
    a = (rn(N, r, K) * 2.0 ** -6).to(torch.bfloat16)
    b = torch.zeros(N, O, r, dtype=torch.bfloat16, device="cuda")
    col = ri(r, N, O)
    b.scatter_(2, col[:, :, None], rn(N, O, 1).clamp(-4, 4).to(torch.bfloat16))
    scale = rn(N).clamp(-4, 4)
    ids = ri(N, n).to(torch.int32)
    y = torch.empty(n, O, device="cuda")
    s = sa.Adapters(a, b, scale)
    ws = torch.empty(kernels.lora_workspace_size(s, n), dtype=torch.uint8, device="cuda")
    assert kernels.lora(s, ids, x, None, y, O, K, n, ws) == 0
    kernels.sync()
    i = ids.long()
    low = a[i, :, at].double() * val.double()[:, None]                       # [n, r]
    want = scale[i].double()[:, None] * low.gather(1, col[i]) * b[i].gather(2, col[i][:, :, None])[:, :, 0].double()
    assert want.abs().max() < torch.finfo(torch.float32).max
    off = ((y.double() - want).abs() / (U * want.abs() + 2.0 ** -149)).cpu().numpy()
    assert np.all(off <= 16), float(np.max(off))
