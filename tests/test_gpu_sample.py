"""smoe_sample against the definition in 64 bits on the host.

Masses are held to 2^-s, s = 62 - bits of vocab, so a sum is off by up to
vocab 2^-s <= 2^-26 of the largest mass at 2^18 tokens; a border or a number u
that lies within that of a running sum may fall to either side. The generated
rows have none that near (asserted); rows of ties, where sums are whole
multiples of equal masses, are exact on both sides."""
import numpy as np
import pytest

pytestmark = pytest.mark.gpu

U = 2.0 ** -24


def want_of(l, t, k, p, m, u):
    """(token, log of its share, distance of the nearest border) by the definition."""
    l = np.asarray(l, np.float64)
    order = np.lexsort((np.arange(len(l)), np.where(np.isnan(l), np.inf, -l)))
    order = order[~np.isnan(l[order]) & (l[order] > -np.inf)]
    if not len(order):
        return -1, np.nan, 1.0
    if t == 0:
        return order[0], 0.0, 1.0
    top = l[order[0]]
    if top == np.inf:
        e = (l[order] == np.inf).astype(np.float64)
    else:
        e = np.exp((l[order] - top) / np.float64(t))
    n = len(order) if k <= 0 else min(k, len(order))
    near = 1.0
    keep = n
    if p < 1:
        cum = np.cumsum(e[:n])
        before = cum - e[:n]
        target = np.float64(p) * cum[-1]
        keep = max(1, int((before < target).sum()))
        if p > 0:
            near = min(near, np.abs(before[1:] - target).min() if n > 1 else 1.0)
    keep = min(keep, int((e >= m).sum()))
    near = min(near, np.abs(e - m)[e > 0].min() if 0 < m < 1 else 1.0)
    by = np.argsort(order[:keep])
    cum = np.cumsum(e[:keep][by])
    at = min(int((cum <= np.float64(u) * cum[-1]).sum()), keep - 1)
    near = min(near, np.abs(cum[:-1] - u * cum[-1]).min() if keep > 1 else 1.0)
    return order[:keep][by][at], np.log(e[:keep][by][at] / cum[-1]), near


def _run(kernels, l, t, k, p, m, u, V, logprobs=True):
    import torch

    n = len(u)
    d = lambda a, ty: None if a is None else torch.tensor(np.asarray(a), dtype=ty, device="cuda")
    lg = l if isinstance(l, torch.Tensor) else d(l, torch.float32)
    tok = torch.full((n + 1,), 77, dtype=torch.int32, device="cuda")
    lp = torch.full((n + 1,), 7.0, device="cuda")
    ws = torch.randint(0, 256, (kernels.sample_workspace_size(n, V),), dtype=torch.uint8, device="cuda")
    status = kernels.sample(lg, d(t, torch.float32), d(k, torch.int32), d(p, torch.float32), d(m, torch.float32),
                            d(u, torch.float32), n, V, tok, lp if logprobs else None, ws)
    assert status == 0
    torch.cuda.synchronize()
    assert int(tok[n]) == 77 and float(lp[n]) == 7
    return tok[:n].cpu().numpy(), lp[:n].double().cpu().numpy()


def _check(kernels, l, t, k, p, m, u, apart=1e-7):
    f = lambda a: np.asarray(a, np.float32)
    l, t, p, m, u = f(l), f(t), f(p), f(m), f(u)
    tok, lp = _run(kernels, l, t, k, p, m, u, l.shape[1])
    kernels.sync()
    for i in range(len(u)):
        a, b, near = want_of(l[i], t[i], k[i], p[i], m[i], u[i])
        if apart is not None:
            assert near > apart, (i, near)
        assert tok[i] == a, (i, tok[i], a, t[i], k[i], p[i], m[i], u[i])
        # The logarithm of two f64 sums, rounded; the kept sum by 2^-26.
        if a >= 0:
            assert abs(lp[i] - b) <= U * abs(b) + 2.0 ** -25, (i, lp[i], b)


# Seeds whose rows have no border within 1e-7 of a running sum.
@pytest.mark.parametrize("V", [1, 2, 3, 31, 1000, 1024, 1025, 5003, 50000, 151936, 262145])
@pytest.mark.parametrize("sigma", [0.3, 2.5, 20.0])
def test_filters(kernels, V, sigma):
    rng = np.random.default_rng(V + int(sigma * 10))
    n = 12
    l = rng.standard_normal((n, V)) * sigma
    l[rng.random((n, V)) < 0.1] = -np.inf
    l[:, V // 2] = 0.25
    t = [1.0, 0.7, 0.0, 1.3, 1.0, 0.2, 3.0, 1.0, 1.0, 0.9, 1.0, 5.0]
    k = [0, 50, 0, 1000, 1, 0, -3, 7, V, 20, 0, 300]
    p = [1.0, 0.9, 0.5, 1.0, 0.9, 0.95, 1.5, 0.3, 1.0, 0.99, 0.0, 0.5]
    m = [0.0, 0.0, 0.1, 0.05, 0.0, 0.0, 0.0, 0.3, 0.02, 0.1, 0.0, 0.0]
    u = rng.random(n).astype(np.float32)
    _check(kernels, l, t, k, p, m, u, apart=None if V <= 3 else 1e-9)


@pytest.mark.parametrize("n", [1, 2, 33, 200, 1100])
def test_batches(kernels, n):
    rng = np.random.default_rng(n)
    l = rng.standard_normal((n, 3001)) * 3
    k = rng.choice([0, 1, 40, 2000], n)
    p = rng.choice([1.0, 0.9, 0.4], n)
    _check(kernels, l, rng.choice([0.0, 0.6, 1.0, 1.7], n), k, p, rng.choice([0.0, 0.01], n), rng.random(n), apart=1e-10)


def test_defaults(kernels):
    """Nothing given: the plain distribution; no logarithms asked for."""
    rng = np.random.default_rng(4)
    l = (rng.standard_normal((5, 2000)) * 2).astype(np.float32)
    u = rng.random(5).astype(np.float32)
    tok, _ = _run(kernels, l, None, None, None, None, u, 2000, logprobs=False)
    for i in range(5):
        assert tok[i] == want_of(l[i], 1.0, 0, 1.0, 0.0, u[i])[0]


def test_numbers_u_walk_through_the_tokens(kernels):
    """Equal logits: u = (i + 0.5) / n gives the i-th kept token, in token order."""
    V = 3000
    l = np.full((1, V), -1.5, np.float32)
    l[0, ::3] = 2.0  # 1000 tokens tie at the top
    for k, kept in ((0, 1000), (10, 10), (999, 999), (1000, 1000)):
        for i in (0, 1, kept // 2, kept - 1):
            u = (i + 0.5) / kept
            tok, lp = _run(kernels, l, [0.01], [k], [1.0], [0.0], [u], V)
            assert tok[0] == 3 * i, (k, i)
            assert abs(lp[0] + np.log(kept)) <= 2 * U * 7
    # Half of the ties' mass, exactly. 0.001 as f32 is 0.001 + 4.7e-11: a
    # thousand of it is more than one token's mass.
    for p, kept in ((0.5, 500), (0.25, 250), (0.001, 2), (0.0, 1)):
        tok, _ = _run(kernels, l, [0.01], [0], [p], [0.0], [1 - 2.0 ** -24], V)
        assert tok[0] == 3 * (kept - 1), (p, tok)


@pytest.mark.parametrize("kind", ["equal", "zeros", "masked_most", "lowest", "inf", "two_inf", "steps", "huge", "tiny"])
def test_rows_of_all_kinds(kernels, kind):
    rng = np.random.default_rng(11)
    V, n = 20011, 6
    l = (rng.standard_normal((n, V)) * 2.5).astype(np.float32)
    if kind == "equal":
        l[:] = 3.25
    elif kind == "zeros":        # of both signs: one value
        l = rng.choice(np.array([0.0, -0.0], np.float32), (n, V))
    elif kind == "masked_most":
        l[rng.random(l.shape) < 0.999] = -np.inf
    elif kind == "lowest":       # a mask of the type's lowest value
        l[rng.random(l.shape) < 0.9] = np.finfo(np.float32).min
    elif kind == "inf":
        l[:, 777] = np.inf
    elif kind == "two_inf":
        l[:, [777, 19000]] = np.inf
        l[:, 5] = np.nan
    elif kind == "steps":        # ties everywhere
        l = np.round(l)
    elif kind == "huge":
        l *= np.float32(1e37)
    elif kind == "tiny":
        l *= np.float32(1e-42)
    t = [1.0, 0.5, 1.0, 2.0, 0.0, 1.0]
    k = [0, 100, 0, 5000, 3, 19999]
    p = [1.0, 0.9, 0.6, 0.95, 1.0, 1.0]
    m = [0.0, 0.0, 0.0, 0.0, 0.0, 0.5]
    u = rng.random(n).astype(np.float32)
    _check(kernels, l, t, k, p, m, u, apart=1e-9)


@pytest.mark.parametrize("V", [700, 5003, 40001])
def test_logits_further_apart_than_f32_goes(kernels, V):
    """Distances from the largest overflow, logits and masses do not."""
    rng = np.random.default_rng(V + 1)
    n = 10
    l = ((rng.random((n, V)) * 2 - 1) * 3.3e38).astype(np.float32)
    l[:, ::7] = -np.inf
    t = [3e38, 1e38, 3e38, 3e38, 1.0, 3e38, 1e38, 3e38, 3e38, 3e38]
    k = [0, 0, V // 2, V * 4 // 5, V // 2, 300, 448, 449, V // 3, 0]
    p = [1.0, 0.9, 0.9, 1.0, 1.0, 0.99, 1.0, 0.99, 1.0, 0.999]
    m = [0.0, 0.0, 0.0, 0.0, 0.0, 0.1, 0.0, 0.0, 0.3, 0.2]
    _check(kernels, l, t, k, p, m, rng.random(n), apart=1e-9)


def test_extreme_numbers(kernels):
    rng = np.random.default_rng(66)
    V = 3001
    l = np.round(rng.standard_normal((12, V)) * 4, 1)
    l[:, 17] = l.max(1)  # two largest at least
    top = np.float32(1 - 2.0 ** -24)
    t = [1e-40, 1e-38, 3e38, 1.0, 1.0, 1.0, 1e-3, 1.0, 1.0, 1.0, 1e-45, 0.5]
    k = [0, 5, 0, 2 ** 31 - 1, -2 ** 31, V, 0, V - 1, 0, 0, 600, 600]
    p = [1.0, 1e-38, 1.0, np.finfo(np.float32).max, 1.0, np.inf, 0.5, 0.999, 1e-45, top, 0.5, 1.0]
    m = [1e-45, 1.0, 0.0, 1.0, 1e-38, 0.0, 1.0, 0.0, 0.0, 0.0, 0.0, 1e-30]
    u = [top, 0.0, 0.3, top, 1e-45, top, 0.4, 0.7, 0.2, 0.6, 0.9, top]
    _check(kernels, l, t, k, p, m, u, apart=None)


def test_rows_without_a_value_and_bad_numbers(kernels):
    import streamoe_amd as sa

    V = 5000
    rng = np.random.default_rng(1)
    l = rng.standard_normal((4, V)).astype(np.float32)
    l[0] = -np.inf
    l[1] = np.nan
    l[2] = np.where(rng.random(V) < 0.5, -np.inf, np.nan)
    one = np.ones(4, np.float32)
    tok, lp = _run(kernels, l, one, [5, 0, 0, 0], one * 0.9, one * 0, one * 0.5, V)
    kernels.sync()  # no error
    assert list(tok[:3]) == [-1, -1, -1] and np.all(np.isnan(lp[:3])) and tok[3] >= 0
    good = dict(t=1.0, k=10, p=0.9, m=0.1, u=0.5)
    bad = [dict(t=-1.0), dict(t=np.inf), dict(t=np.nan), dict(p=-0.1), dict(p=np.nan), dict(m=-0.1), dict(m=1.5), dict(m=np.nan),
           dict(u=1.0), dict(u=-0.1), dict(u=np.nan)]
    rows = [dict(good, **b) for b in bad for b in (b, {})]
    x = rng.standard_normal((len(rows), V)).astype(np.float32)
    col = lambda c: [r[c] for r in rows]
    tok, lp = _run(kernels, x, col("t"), col("k"), col("p"), col("m"), col("u"), V)
    with pytest.raises(sa.SmoeError, match="INVALID_ARG"):
        kernels.sync()
    kernels.sync()
    for i, r in enumerate(rows):
        if i % 2 == 0:
            assert tok[i] == -1 and np.isnan(lp[i])
        else:
            assert tok[i] == want_of(x[i], 1.0, 10, np.float32(0.9), np.float32(0.1), 0.5)[0]


def test_the_most_rows(kernels):
    rng = np.random.default_rng(65)
    n, V = 65535, 7
    l = (rng.standard_normal((n, V)) * 2).astype(np.float32)
    t, k = rng.choice([0.0, 1.0, 2.0], n).astype(np.float32), rng.choice([0, 1, 3], n)
    p, u = rng.choice([1.0, 0.7], n).astype(np.float32), rng.random(n).astype(np.float32)
    tok, _ = _run(kernels, l, t, k, p, np.zeros(n), u, V)
    kernels.sync()
    for i in rng.permutation(n)[:3000]:
        a, _, near = want_of(l[i], t[i], k[i], p[i], 0.0, u[i])
        assert tok[i] == a or near < 1e-9, i


@pytest.mark.parametrize("V", [400, 3000, 20000])
def test_more_ties_than_top_k(kernels, V):
    """Top-k's bin holds more tokens than a block sorts: a few larger ones, then
    thousands of equal ones, with every filter."""
    rng = np.random.default_rng(V)
    n = 8
    l = np.full((n, V), 0.5, np.float32)
    at = rng.permutation(V)[:37]
    l[:, at] = (2 + rng.random((n, 37))).astype(np.float32)
    k = [38, 50, 448, 449, 300, 700, 37, 1]
    p = [1.0, 0.9, 1.0, 1.0, 0.97, 0.99, 0.5, 1.0]
    _check(kernels, l, np.ones(n), k, p, [0.0, 0.0, 0.0, 0.0, 0.05, 0.0, 0.9, 0.0], rng.random(n), apart=1e-9)


def test_the_same_bits_again(kernels):
    rng = np.random.default_rng(12)
    l = np.round(rng.standard_normal((40, 30011)) * 3).astype(np.float32)
    a = [rng.choice([0.7, 1.0], 40), rng.choice([0, 500], 40), rng.choice([1.0, 0.9], 40), np.zeros(40), rng.random(40)]
    first = _run(kernels, l, *a, 30011)
    for _ in range(3):
        again = _run(kernels, l, *a, 30011)
        assert np.array_equal(first[0], again[0]) and np.array_equal(first[1], again[1])


def test_the_largest_vocabulary(kernels):
    import torch

    V = 1 << 24
    l = torch.zeros(2, V, device="cuda")
    l[1, 123456] = 30.0
    tok, lp = _run(kernels, l, [1.0, 1.0], [0, 9], [1.0, 0.5], [0.0, 0.0], [0.75, 0.999], V)
    kernels.sync()
    assert tok[0] == V * 3 // 4 and tok[1] == 123456
    assert abs(lp[0] + 24 * np.log(2)) <= 2 * U * 17 and lp[1] == 0
