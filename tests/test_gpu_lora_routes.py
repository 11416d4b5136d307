"""smoe_lora's promises on each way its rows find their adapter: both products
in one launch, items found by waves, by blocks, and by the plan of many rows or
many adapters. Bounds as in test_gpu_lora.py."""
import pytest

from test_gpu_lora import _case, _check, _run

pytestmark = pytest.mark.gpu

# rows, inputs, outputs, adapters, rank
ROUTES = [
    pytest.param(20, 64, 100, 9, 40, id="one"),
    pytest.param(20, 4096, 100, 9, 40, id="wave"),
    pytest.param(40, 4096, 36, 1100, 8, id="wave-many-adapters"),
    pytest.param(300, 128, 100, 9, 40, id="block"),
    pytest.param(1024, 64, 40, 9, 40, id="block-most-rows"),
    pytest.param(300, 64, 36, 1022, 8, id="block-most-adapters"),
    pytest.param(1500, 128, 100, 9, 40, id="plan"),
    pytest.param(70, 64, 36, 1100, 8, id="plan-many-adapters"),
    pytest.param(70, 64, 36, 4096, 8, id="plan-most-adapters"),
]


@pytest.mark.parametrize("n,K,O,N,r", ROUTES)
def test_ranks_and_garbage_behind_them(kernels, n, K, O, N, r):
    import torch

    ranks = [(3 * i) % (r + 1) for i in range(N)]
    case = _case(n, K, O, N, r, seed=n, ranks=ranks)
    j = torch.arange(r, device="cuda")
    case[1][(j[None, :] >= case[5][:, None])] = float("nan")
    case[2].masked_fill_((j[None, :] >= case[5][:, None])[:, None, :], float("inf"))
    _check(kernels, case)
    _check(kernels, case, inplace=True)


@pytest.mark.parametrize("n,K,O,N,r", ROUTES)
def test_bad_ids_and_ranks_are_reported(kernels, n, K, O, N, r):
    import torch

    import streamoe_amd as sa

    x, a, b, scale, ids, rk, base = _case(n, K, O, N, r, seed=n, ranks=[r] * N)
    good = ids.clone()
    good[3] = good[n - 1] = -1
    want = _run(kernels, x, a, b, scale, good, rk, base)
    s = sa.Adapters(a, b, scale, rk)
    ws = torch.empty(kernels.lora_workspace_size(s, n), dtype=torch.uint8, device="cuda")
    for low, high in ((-2, N), (-(1 << 31), (1 << 31) - 1)):
        ids = good.clone()
        ids[3], ids[n - 1] = low, high
        y = torch.empty(n, O, device="cuda")
        assert kernels.lora(s, ids, x, base, y, O, K, n, ws) == 0
        with pytest.raises(sa.SmoeError, match="INVALID_ARG"):
            kernels.sync()
        assert torch.equal(y, want)
        kernels.sync()
    for bad, taken in ((-1, 0), (r + 1, r), ((1 << 31) - 1, r)):
        rk[N - 1] = bad
        y = torch.empty(n, O, device="cuda")
        assert kernels.lora(s, good, x, base, y, O, K, n, ws) == 0
        with pytest.raises(sa.SmoeError, match="INVALID_ARG"):
            kernels.sync()
        rk[N - 1] = taken
        assert torch.equal(y, _run(kernels, x, a, b, scale, good, rk, base))


@pytest.mark.parametrize("n,K,O,N,r", ROUTES)
@pytest.mark.parametrize("xb", [False, True])
def test_a_rows_bits_do_not_depend_on_the_others(kernels, n, K, O, N, r, xb):
    import torch

    x, a, b, scale, ids, rk, base = _case(n, K, O, N, r, seed=n, xb=xb)
    y = _run(kernels, x, a, b, scale, ids, rk, base)
    p = torch.randperm(n, device="cuda")
    assert torch.equal(y[p], _run(kernels, x[p].contiguous(), a, b, scale, ids[p].contiguous(), rk, base[p].contiguous()))
    other = torch.full_like(ids, int(ids[0]))
    other[1::2] = N - 1
    assert torch.equal(_run(kernels, x, a, b, scale, other, rk, base)[0], y[0])


@pytest.mark.parametrize("n,K,O,N,r", ROUTES)
def test_nan_and_infinity_stay_in_their_row(kernels, n, K, O, N, r):
    import torch

    case = _case(n, K, O, N, r, seed=n)
    case[4].fill_(1)
    clean = _run(kernels, *case)
    case[0][2, K - 1] = float("nan")
    case[0][n - 2, 1] = float("-inf")
    y = _run(kernels, *case)
    bad = torch.zeros(n, dtype=torch.bool, device="cuda")
    bad[2] = bad[n - 2] = True
    assert torch.all(torch.isnan(y[bad])) and torch.equal(y[~bad], clean[~bad])


@pytest.mark.parametrize("n,K,O,N,r", ROUTES)
def test_replays_with_other_ids(kernels, n, K, O, N, r):
    import torch

    import streamoe_amd as sa

    x, a, b, scale, ids, rk, base = _case(n, K, O, N, r, seed=n, ranks=[r] * N)
    s = sa.Adapters(a, b, scale, rk)
    ws = torch.empty(kernels.lora_workspace_size(s, n), dtype=torch.uint8, device="cuda")
    y = torch.empty(n, O, device="cuda")
    call = lambda: sa.check(kernels.lora(s, ids, x, base, y, O, K, n, ws), "lora")
    graph = sa.capture_graph(kernels, call)
    for k in range(3):
        ids.copy_(torch.randint(-1, N, (n,), device="cuda", dtype=torch.int32) if k != 1 else torch.full_like(ids, 1))
        rk.copy_(torch.randint(0, r + 1, (N,), device="cuda", dtype=torch.int32))
        x.normal_()
        graph.replay()
        torch.cuda.synchronize()
        got = y.clone()
        call()
        kernels.sync()
        assert torch.equal(got, y)
    _check(kernels, (x, a, b, scale, ids, rk, base))
