"""The serving operators where element and byte offsets pass 32 bits: mostly
zeros, checked at the far end against 64-bit arithmetic with the bounds of the
operators' own tests."""
import numpy as np
import pytest

pytestmark = pytest.mark.gpu

U = 2.0 ** -24
BF = 2.0 ** -8  # half of bf16's eps 2^-7: the most a rounding to it is off


@pytest.fixture(autouse=True)
def _room():
    import torch

    torch.cuda.empty_cache()
    if torch.cuda.mem_get_info()[0] < 60 << 30:
        pytest.skip("needs 60 GiB of free device memory")
    yield
    torch.cuda.empty_cache()


def test_norm(kernels):
    import torch

    n, H = 263000, 16384  # 4.31e9 values
    x = torch.zeros(n, H, dtype=torch.bfloat16, device="cuda")
    x[-2:] = torch.randn(2, H, device="cuda").to(torch.bfloat16)
    out, q = torch.empty_like(x), torch.empty(n, H, dtype=torch.int8, device="cuda")
    sc = torch.empty(n, H // 128, device="cuda")
    assert kernels.rmsnorm(x, None, None, 1e-6, n, H, None, None, q, sc, 128) == 0
    assert kernels.rmsnorm(x, None, None, 1e-6, n, H, None, out) == 0
    kernels.sync()
    s = x[-2:].double()
    y = s / torch.sqrt((s ** 2).mean(1, keepdim=True) + 1e-6)
    assert torch.all((out[-2:].double() - y).abs() <= (BF + (H / 256 + 40) * U * (1 + BF)) * y.abs() + 1e-30)
    deq = q[-2:].double().view(2, -1, 128) * sc[-2:].double()[..., None]
    top = y.abs().view(2, -1, 128).amax(-1, keepdim=True)
    assert torch.all((deq - y.view(2, -1, 128)).abs() <= top * (0.5 / 127 + (H / 256 + 50) * U))
    assert not out[-3].any() and not q[:-2:1000].any()


@pytest.mark.parametrize("n,O,K", [(17200, 250000, 64), (3, 2200000, 4096), (40, 2200000, 4096), (2, 600000, 16384)])
def test_qmm_i8(kernels, n, O, K):
    import torch

    import streamoe_amd as sa

    G, last = 64, 48
    codes = torch.zeros(O, K // 2, dtype=torch.uint8, device="cuda")
    s = torch.zeros(O, K // G, dtype=torch.bfloat16, device="cuda")
    b = torch.zeros_like(s)
    codes[-last:] = torch.randint(0, 256, (last, K // 2), dtype=torch.uint8, device="cuda")
    s[-last:], b[-last:] = (torch.randn(last, K // G, device="cuda").to(torch.bfloat16) for _ in range(2))
    # One buffer: the codes, then scales and biases.
    parts = [codes.view(-1), s.view(torch.uint8).view(-1), b.view(torch.uint8).view(-1)]
    at = [0, parts[0].numel(), parts[0].numel() + parts[1].numel()]
    w = torch.cat(parts)
    x = torch.randint(-127, 128, (n, K), dtype=torch.int8, device="cuda")
    sx = torch.rand(n, device="cuda") + 0.5
    y = torch.full((n, O), 7.0, device="cuda")
    assert kernels.qmm_i8(sa.QuantWeights(w, *at, G, 4), x, sx, 0, y, O, K, n) == 0
    kernels.sync()
    c = codes[-last:].long()
    q = torch.stack((c & 15, c >> 4), -1).view(last, K).double()
    per = lambda t: t[-last:].double().repeat_interleave(G, 1)
    m = min(n, 32)
    x64 = x[-m:].double() * sx[-m:, None].double()
    want = (x64[:, None] * (q * per(s) + per(b))[None]).sum(-1)
    mag = (x64.abs()[:, None] * (q * per(s).abs() + per(b).abs())[None]).sum(-1)
    assert torch.all((y[-m:, -last:].double() - want).abs() <= (2 * (K // G) + 24) * U * mag)
    assert not y[-1, :-last].any() and not y[0, : O - last].any()


def test_lora(kernels):
    import torch

    import streamoe_amd as sa

    n, K, O, r = 65536, 64, 66000, 8  # 4.33e9 outputs; adapters 4 GiB apart
    a = torch.zeros(3, 1 << 31, dtype=torch.bfloat16, device="cuda")[:, : r * K].view(3, r, K)
    b = torch.zeros(3, 1 << 31, dtype=torch.bfloat16, device="cuda")[:, : O * r].view(3, O, r)
    a[2], b[2] = torch.randn(r, K, device="cuda").to(a.dtype), torch.randn(O, r, device="cuda").to(b.dtype)
    s = sa.Adapters(a, b, torch.ones(3, device="cuda"))
    ids = torch.full((n,), -1, dtype=torch.int32, device="cuda")
    ids[-20:] = 2
    x = torch.randn(n, K, device="cuda")
    y = torch.ones(n, O, device="cuda")
    ws = torch.empty(kernels.lora_workspace_size(s, n), dtype=torch.uint8, device="cuda")
    assert kernels.lora(s, ids, x, y, y, O, K, n, ws) == 0
    kernels.sync()
    A, B, X = (t.double().cpu() for t in (a[2], b[2], x[-20:]))
    want, mag = 1 + X @ A.T @ B.T, X.abs() @ A.abs().T @ B.abs().T
    got = y[-20:].double().cpu()
    assert torch.all((got - want).abs() <= (2.0 ** -15 + (K + r + 60) * U) * mag + 2 * U * (1 + want.abs()))
    assert torch.all(y[-21] == 1) and torch.all(y[:: 997][:-1] == 1)


def test_beams(kernels):
    import torch

    R, W, V = 1800, 4, 600000  # 4.32e9 logits
    l = torch.zeros(R * W, V, device="cuda")
    l[-1, -1], l[-3, V // 2], l[-3, -2] = 9.0, 8.0, 9.0
    sc = torch.zeros(R * W, device="cuda")
    v, rows, tok = torch.empty(R, W, device="cuda"), *(torch.empty(R, W, dtype=torch.int32, device="cuda") for _ in range(2))
    ws = torch.empty(kernels.beam_select_workspace_size(R, W, V, W), dtype=torch.uint8, device="cuda")
    assert kernels.beam_select(l, sc, None, 0, R, W, V, W, v, rows, tok, ws) == 0
    kernels.sync()
    top = R * W
    # The larger of two rows with one 9 each is the one without the 8.
    assert rows[-1].tolist()[:3] == [top - 1, top - 3, top - 3] and tok[-1].tolist()[:3] == [V - 1, V - 2, V // 2]
    assert torch.equal(tok[:-1].cpu(), torch.arange(W, dtype=torch.int32).expand(R - 1, W))
    assert torch.equal(rows[:-1].cpu(), (torch.arange(R - 1, dtype=torch.int32) * W)[:, None].expand(R - 1, W))
    want = -np.log(V)
    assert abs(float(v[0, 0]) - want) <= (36 + 2 * 200) * U - U * want


def test_reorder(kernels):
    import torch

    import streamoe_amd as sa

    room, used = (1 << 30) + 4096, (1 << 30) + 16
    src = torch.zeros(5, room, dtype=torch.uint8, device="cuda")
    for i in range(5):
        src[i, -8192:].random_(0, 256)
        src[i, :4096].random_(0, 256)
    dst = torch.full((5, room), 9, dtype=torch.uint8, device="cuda")
    rows = torch.tensor([4, 0, 4, 1, 3], dtype=torch.int32, device="cuda")
    assert kernels.beam_reorder([sa.BeamState(src, dst, used)], rows) == 0
    kernels.sync()
    for i, r in enumerate(rows.tolist()):
        assert torch.equal(dst[i, :used], src[r, :used]) and torch.all(dst[i, used:] == 9)
