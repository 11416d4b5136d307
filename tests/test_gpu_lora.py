"""smoe_lora against 64-bit arithmetic.

Bound per output, u = 2^-24, with |.| element by element and s = |scale|:
u_j = A_j x has exact bf16 x bf16 products of x's pair (off by 2^-16 |x|, none
for bf16 x) and f32 sums of in_dim terms, at most (in_dim + 16) u of
m_j = |A_j| |x|: e_j <= (2^-16 + (in_dim + 40) u) m_j (the shares' sum and the
scale's product within the 40). The second product adds 2^-16 + (rank + 8) u of
sum |B_oj| s m_j, and base one rounding: in all
    (2^-15 + (in_dim + rank + 60) u) s |B| |A| |x| + 2 u (|base| + |y|) + tiny."""
import numpy as np
import pytest

pytestmark = pytest.mark.gpu

U = 2.0 ** -24


def _case(n, K, O, N, r, seed=0, xb=False, ranks=None, ids=None, base=True):
    import torch

    g = torch.Generator(device="cuda").manual_seed(seed)
    rn = lambda *s: torch.randn(*s, generator=g, device="cuda")
    x = rn(n, K)
    x = x.to(torch.bfloat16) if xb else x
    a, b = (rn(N, r, K) * 0.05).to(torch.bfloat16), (rn(N, O, r) * 0.05).to(torch.bfloat16)
    scale = rn(N)
    if ids is None:
        ids = torch.randint(-1, N, (n,), generator=g, device="cuda", dtype=torch.int32)
    else:
        ids = torch.tensor(ids, dtype=torch.int32, device="cuda")
    rk = None if ranks is None else torch.tensor(ranks, dtype=torch.int32, device="cuda")
    return x, a, b, scale, ids, rk, rn(n, O) if base else None


def _want(x, a, b, scale, ids, rk, base, O):
    x64, n = x.double(), x.shape[0]
    import torch

    y = torch.zeros(n, O, dtype=torch.float64, device="cuda") if base is None else base.double()
    mag = torch.zeros_like(y)
    for t, i in enumerate(ids.tolist()):
        if i < 0 or i >= a.shape[0]:
            continue
        r = a.shape[1] if rk is None else int(rk[i])
        A, B, s = a[i, :r].double(), b[i, :, :r].double(), scale[i].double()
        y[t] += s * (B @ (A @ x64[t]))
        mag[t] = s.abs() * (B.abs() @ (A.abs() @ x64[t].abs()))
    return y.cpu().numpy(), mag.cpu().numpy()


def _run(kernels, x, a, b, scale, ids, rk, base, inplace=False):
    import torch

    import streamoe_amd as sa

    n, K, O = x.shape[0], x.shape[1], b.shape[1]
    s = sa.Adapters(a, b, scale, rk)
    # The workspace's contents do not matter: all NaN here.
    ws = torch.full(((kernels.lora_workspace_size(s, n) + 3) // 4,), float("nan"), device="cuda")
    y = base.clone() if inplace else torch.full((n + 1, O), 7.0, device="cuda")
    assert kernels.lora(s, ids, x, y if inplace else base, y, O, K, n, ws) == 0
    kernels.sync()
    if not inplace:
        assert torch.all(y[n] == 7)
    return y[:n]


def _check(kernels, case, **kw):
    x, a, b, scale, ids, rk, base = case
    y = _run(kernels, *case, **kw).double().cpu().numpy()
    want, mag = _want(*case, b.shape[1])
    K, r = x.shape[1], a.shape[1]
    b64 = 0 if base is None else np.abs(base.double().cpu().numpy())
    bound = (2.0 ** -15 + (K + r + 60) * U) * mag + 2 * U * (b64 + np.abs(want)) + 1e-30
    assert np.all(np.abs(y - want) <= bound), float(np.max(np.abs(y - want) / bound))


@pytest.mark.parametrize("n,K,O,N,r", [
    (1, 8, 1, 1, 8), (1, 2048, 2048, 3, 16), (2, 40, 7, 2, 8), (8, 2048, 512, 4, 16), (16, 264, 260, 1, 24),
    (17, 512, 513, 1, 32), (33, 1032, 256, 40, 64), (64, 256, 4096, 5, 40), (65, 256, 300, 5, 40),
    (200, 4096, 1028, 40, 64), (257, 128, 130, 7, 128), (1000, 2048, 256, 3, 32), (1025, 64, 64, 1100, 8),
    (5000, 64, 100, 50, 16),
])
@pytest.mark.parametrize("xb", [False, True])
def test_lora(kernels, n, K, O, N, r, xb):
    _check(kernels, _case(n, K, O, N, r, seed=n + K, xb=xb))


@pytest.mark.parametrize("n,K,O,N,r", [
    (8, 4096, 260, 4, 16), (64, 2048, 300, 64, 64), (5, 2048, 513, 3, 128), (33, 8192, 64, 2, 8), (40, 512, 5000, 37, 24),
])
@pytest.mark.parametrize("xb", [False, True])
def test_few_rows_of_much_work(kernels, n, K, O, N, r, xb):
    _check(kernels, _case(n, K, O, N, r, seed=n + K, xb=xb))
    case = _case(n, K, O, N, r, seed=n, xb=xb, ranks=[(5 * i) % (r + 1) for i in range(N)])
    _check(kernels, case, inplace=True)


@pytest.mark.parametrize("n", [3, 70, 300])
def test_ranks_of_their_own_and_garbage_behind_them(kernels, n):
    ranks = [0, 1, 7, 8, 16, 31, 32, 33, 40]
    x, a, b, scale, ids, rk, base = _case(n, 320, 200, len(ranks), 40, seed=n, ranks=ranks)
    for i, r in enumerate(ranks):
        a[i, r:] = float("nan")
        b[i, :, r:] = float("inf")
    _check(kernels, (x, a, b, scale, ids, rk, base))


def test_no_base_in_place_and_rows_without_adapter(kernels):
    import torch

    case = _case(100, 256, 129, 4, 16, base=False)
    y = _run(kernels, *case)
    assert torch.all(y[case[4] == -1] == 0)
    _check(kernels, case)
    case = _case(100, 256, 128, 4, 16)
    _check(kernels, case, inplace=True)
    case = _case(37, 256, 128, 4, 16, ids=[-1] * 37)
    assert torch.equal(_run(kernels, *case), case[6])
    assert torch.equal(_run(kernels, *case, inplace=True), case[6])


@pytest.mark.parametrize("n", [1, 16, 17, 64, 100, 513])
def test_one_adapter_for_all_and_one_each(kernels, n):
    _check(kernels, _case(n, 512, 256, 3, 16, ids=[2] * n))
    _check(kernels, _case(n, 64, 72, n, 8, ids=list(range(n))[::-1]))


def test_a_rows_bits_do_not_depend_on_the_others(kernels):
    import torch

    x, a, b, scale, ids, rk, base = _case(64, 1024, 512, 5, 32)
    y = _run(kernels, x, a, b, scale, ids, rk, base)
    p = torch.randperm(64, device="cuda")
    z = _run(kernels, x[p].contiguous(), a, b, scale, ids[p].contiguous(), rk, base[p].contiguous())
    assert torch.equal(y[p], z)
    other = ids.clone()
    other[1:] = 4 - ids[1:].clamp(min=0)
    assert torch.equal(_run(kernels, x, a, b, scale, other, rk, base)[0], y[0])


def test_nan_and_infinity_stay_in_their_row(kernels):
    import torch

    case = _case(20, 256, 64, 1, 16, ids=[0] * 20)
    clean = _run(kernels, *case)
    case[0][3, 5] = float("nan")
    case[0][7, 9] = float("inf")
    y = _run(kernels, *case)
    assert torch.all(torch.isnan(y[3])) and torch.all(torch.isnan(y[7]))
    keep = [i for i in range(20) if i not in (3, 7)]
    assert torch.equal(y[keep], clean[keep])


@pytest.mark.parametrize("n", [4, 300])
def test_bad_ids_and_ranks_are_reported(kernels, n):
    import torch

    import streamoe_amd as sa

    ids = [0, 5, -2, 1] + [0] * (n - 4)
    case = _case(n, 64, 64, 5, 8, ids=ids)
    with pytest.raises(sa.SmoeError, match="INVALID_ARG"):
        _run(kernels, *case)
    kernels.sync()
    x, a, b, scale, i, rk, base = case
    y = torch.empty(n, 64, device="cuda")
    s = sa.Adapters(a, b, scale)
    ws = torch.empty(kernels.lora_workspace_size(s, n), dtype=torch.uint8, device="cuda")
    assert kernels.lora(s, i, x, base, y, 64, 64, n, ws) == 0
    with pytest.raises(sa.SmoeError):
        kernels.sync()
    assert torch.equal(y[1:3], base[1:3]) and not torch.equal(y[3], base[3])
    good = [v if -1 <= v < 5 else -1 for v in ids]
    assert torch.equal(y, _run(kernels, x, a, b, scale, torch.tensor(good, dtype=torch.int32, device="cuda"), rk, base))
    for bad in (-1, 9):
        with pytest.raises(sa.SmoeError):
            _run(kernels, *_case(n, 64, 64, 2, 8, ranks=[bad, 8], ids=[1] * n))
    kernels.sync()


def test_adapters_that_lie_apart(kernels):
    import torch

    x, a, b, scale, ids, rk, base = _case(30, 128, 96, 4, 16)
    big_a = torch.zeros(4, 40, 128, dtype=torch.bfloat16, device="cuda")
    big_b = torch.zeros(4, 100, 16, dtype=torch.bfloat16, device="cuda")
    big_a[:, 8:24] = a
    big_b[:, 2:98] = b
    y = _run(kernels, x, a, b, scale, ids, rk, base)
    z = _run(kernels, x, big_a[:, 8:24], big_b[:, 2:98], scale, ids, rk, base)
    assert torch.equal(y, z)


def test_misfit_tensors_are_refused(kernels):
    import torch

    import streamoe_amd as sa

    x, a, b, scale, ids, rk, base = _case(6, 64, 32, 2, 8)
    s = sa.Adapters(a, b, scale)
    ws = torch.empty(kernels.lora_workspace_size(s, 6), dtype=torch.uint8, device="cuda")
    y = torch.empty(6, 32, device="cuda")
    assert kernels.lora(s, ids, x, base, y, 32, 64, 7, ws) == 1            # too few rows
    assert kernels.lora(s, ids.long(), x, base, y, 32, 64, 6, ws) == 1
    assert kernels.lora(s, ids, x, base, y, 64, 64, 3, ws) == 1            # not the adapters' out_dim
    assert kernels.lora(s, ids, x.t(), base, y, 32, 64, 6, ws) == 1
    assert kernels.lora(s, ids, x, base, y, 32, 64, 6, ws[:16]) == 9       # WORKSPACE_TOO_SMALL
    for bad in (sa.Adapters(a.float(), b, scale), sa.Adapters(a, b[:1], scale), sa.Adapters(a, b, scale[:1]),
                sa.Adapters(a.transpose(1, 2), b, scale), sa.Adapters(a, b, scale, ids.long())):
        with pytest.raises(sa.SmoeError):
            kernels.lora(bad, ids, x, base, y, 32, 64, 6, ws)


def test_graph_replays(kernels):
    import torch

    import streamoe_amd as sa

    for n in (8, 150):
        x, a, b, scale, ids, rk, base = _case(n, 512, 320, 6, 16)
        s = sa.Adapters(a, b, scale)
        ws = torch.empty(kernels.lora_workspace_size(s, n), dtype=torch.uint8, device="cuda")
        y = torch.empty(n, 320, device="cuda")
        call = lambda: sa.check(kernels.lora(s, ids, x, base, y, 320, 512, n, ws), "lora")
        graph = sa.capture_graph(kernels, call)
        for _ in range(3):
            x.normal_()
            ids.copy_(torch.randint(-1, 6, (n,), device="cuda", dtype=torch.int32))
            graph.replay()
            torch.cuda.synchronize()
            got = y.clone()
            call()
            kernels.sync()
            assert torch.equal(got, y)
