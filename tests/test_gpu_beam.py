"""smoe_beam_select and smoe_beam_reorder.

Picks are compared with the definition in 64 bits on the host; a pick may
differ only where its value lies within the error of the sums. With u = 2^-24:
a term exp(l - m) is off by 2 u (the exponential's last place), by u |l - m|
(the difference's rounding) and 0.25 u |l - m| (log2 e in 24 bits); weighted as
in the sum, |l - m| is at most the entropy, ln V <= 13.4 for the sizes here, so
that is 19 u; partial sums of 16 terms round by up to 16 u. A value is off by at
most 36 u, its f32 score by u |score| more. Within a row the log-sum-exp is
one number, so there the order is exact; and so it is between rows of the same
logits. Rows whose log-sum-exps are equal only as real numbers (one row another
one's permutation) may come in either order, each value being off by up to
36 u: two picks of different rows whose 64-bit values are within 72 u.

Of many rows a wave takes several tiles of 4096 in turn; a tile with a larger
logit scales the sum before it by one more exponential, 2 u per tile (what the
differences' rounding adds is in the 19 u: they add up to |l - m|)."""
import numpy as np
import pytest

pytestmark = pytest.mark.gpu

U = 2.0 ** -24


def _want(logits, scores, done, pad, R, W, V, P):
    """(values, rows, tokens) in f64 by the definition."""
    l = np.asarray(logits, np.float64).reshape(R, W, V)
    sc = np.asarray(scores, np.float64).reshape(R, W)
    cand = np.full((R, W, V), -np.inf)
    order = np.zeros((R, W, V))  # within a row, equal values compare by logits
    with np.errstate(all="ignore"):
        for q in range(R):
            for b in range(W):
                if done is not None and done[q * W + b]:
                    if sc[q, b] > -np.inf:
                        cand[q, b, pad] = sc[q, b]
                    continue
                x = np.where(np.isnan(l[q, b]), -np.inf, l[q, b])
                m = x.max()
                if not np.isfinite(m) or not sc[q, b] > -np.inf:
                    continue
                cand[q, b] = sc[q, b] + (x - (m + np.log(np.exp(x - m).sum())))
                order[q, b] = x
    out = []
    for q in range(R):
        c, o = cand[q].ravel(), order[q].ravel()
        beam = np.repeat(np.arange(W), V)
        i = np.lexsort((np.arange(W * V), -np.where(c == -np.inf, 0, o), beam, -c))[:P]
        out.append((c[i], i // V + q * W, i % V))
    return tuple(np.stack(z) for z in zip(*out))


def _run(kernels, logits, scores, done, pad, R, W, V, P):
    import torch

    dev = lambda a, t: None if a is None else torch.tensor(np.asarray(a), dtype=t, device="cuda")
    lg = logits if isinstance(logits, torch.Tensor) else dev(logits, torch.float32)
    sc, dn = dev(scores, torch.float32), dev(done, torch.uint8)
    v = torch.full((R + 1, P), 7.0, device="cuda")
    rows = torch.full((R + 1, P), 77, dtype=torch.int32, device="cuda")
    tok = torch.full((R + 1, P), 77, dtype=torch.int32, device="cuda")
    ws = torch.empty(kernels.beam_select_workspace_size(R, W, V, P), dtype=torch.uint8, device="cuda")
    assert kernels.beam_select(lg, sc, dn, pad, R, W, V, P, v, rows, tok, ws) == 0
    kernels.sync()
    assert torch.all(v[R] == 7) and torch.all(rows[R] == 77) and torch.all(tok[R] == 77)
    return v[:R].double().cpu().numpy(), rows[:R].cpu().numpy(), tok[:R].cpu().numpy()


def _either_order(logits, scores, done, pad, R, W, V, P, rows, tok, wv, wr):
    av, ar, at = _want(logits, scores, done, pad, R, W, V, min(W * V, 4 * P))
    for q in range(R):
        value = {(r, t): v for v, r, t in zip(av[q], ar[q], at[q])}
        for j in range(P):
            if (rows[q, j], tok[q, j]) != (ar[q, j], at[q, j]):
                assert rows[q, j] != wr[q, j] and abs(value[rows[q, j], tok[q, j]] - wv[q, j]) <= 72 * U
        for r in set(rows[q]):  # a row's own picks: the first of its order
            own = tok[q][rows[q] == r]
            assert np.array_equal(own, at[q][ar[q] == r][:len(own)])


def _check(kernels, logits, scores, done, pad, R, W, V, P, tiles=1):
    import torch

    host = logits.cpu().numpy() if isinstance(logits, torch.Tensor) else logits
    v, rows, tok = _run(kernels, logits, scores, done, pad, R, W, V, P)
    wv, wr, wt = _want(host, scores, done, pad, R, W, V, P)
    if not (np.array_equal(rows, wr) and np.array_equal(tok, wt)):
        _either_order(host, scores, done, pad, R, W, V, P, rows, tok, wv, wr)
    fin = np.isfinite(wv)
    assert np.array_equal(v[~fin], wv[~fin])
    assert np.all(np.abs(v - wv)[fin] <= (34 + 2 * tiles) * U + U * np.abs(wv[fin]))


@pytest.mark.parametrize("R,W,V,P", [
    (1, 1, 1, 1), (1, 1, 2, 2), (2, 3, 5, 15), (1, 4, 31, 8), (3, 2, 4093, 4), (2, 4, 4096, 8), (2, 4, 4097, 32),
    (1, 16, 8191, 32), (5, 5, 12289, 10), (2, 4, 151936, 8), (1, 3, 262145, 6), (1, 2, 600001, 32),
])
@pytest.mark.parametrize("masked", [0.0, 0.6])
def test_select(kernels, R, W, V, P, masked):
    rng = np.random.default_rng(V + P)
    l = (rng.standard_normal((R * W, V)) * 2.5).astype(np.float32)
    l[rng.random((R * W, V)) < masked] = -np.inf
    sc = (-10 * rng.random(R * W)).astype(np.float32)
    done = (rng.random(R * W) < 0.3).astype(np.uint8) if masked else None
    _check(kernels, l, sc, done, min(1, V - 1), R, W, V, P)


def test_all_logits_equal(kernels):
    # Every thread holds the same values: only the token decides.
    for V in (40, 5000, 20000):
        _check(kernels, np.full((3, V), 1.5, np.float32), np.zeros(3, np.float32), None, 0, 1, 3, V, 32)


@pytest.mark.parametrize("R,W,V,P", [(64, 16, 5000, 32), (40, 4, 30000, 8), (300, 2, 12289, 4), (70, 2, 40001, 15)])
@pytest.mark.parametrize("kind", ["random", "rising", "falling", "steps", "late", "nan"])
def test_several_tiles_in_turn(kernels, R, W, V, P, kind):
    rng = np.random.default_rng(R + P)
    l = (rng.standard_normal((R * W, V)) * 2.5).astype(np.float32)
    if kind == "rising":      # every tile has more than the list holds
        l = np.broadcast_to(np.arange(V, dtype=np.float32) / 64, (R * W, V)).copy()
    elif kind == "falling":
        l = np.broadcast_to(-np.arange(V, dtype=np.float32) / 64, (R * W, V)).copy()
    elif kind == "steps":     # ties everywhere, larger ones later
        l = np.broadcast_to(np.floor(np.arange(V) / 1500).astype(np.float32), (R * W, V)).copy()
    elif kind == "late":      # nothing in the first tiles, ties of few values behind
        l = np.round(l)
        l[:, : V // 2] = -np.inf
    elif kind == "nan":       # of both signs and kinds
        bits = l.view(np.uint32)
        at = rng.random(l.shape)
        bits[at < 0.4] = 0x7FC00000
        bits[at < 0.3] = 0xFFC00001
        bits[at < 0.2] = 0x7F800001
        bits[at < 0.1] = 0xFF8FFFFF
    sc = (-10 * rng.random(R * W)).astype(np.float32)
    _check(kernels, l, sc, None, 0, R, W, V, P, tiles=10)


def test_ties_across_rows_and_zeros_of_both_signs(kernels):
    rng = np.random.default_rng(5)
    l = np.round(rng.standard_normal((4, 9000)) * 2).astype(np.float32)
    l[l == 0] = rng.choice([0.0, -0.0], (l == 0).sum())
    l[1] = l[0]
    l[3] = l[2][::-1]
    _check(kernels, l, np.zeros(4, np.float32), None, 0, 1, 4, 9000, 24)


def test_first_step_only_one_open_beam(kernels):
    rng = np.random.default_rng(6)
    l = rng.standard_normal((8, 1000)).astype(np.float32)
    sc = np.full((2, 4), -np.inf, np.float32)
    sc[:, 0] = 0
    _check(kernels, l, sc.ravel(), None, 0, 2, 4, 1000, 8)
    _check(kernels, l[:, :3].copy(), sc.ravel(), None, 0, 2, 4, 3, 8)  # -inf picks in order


def test_nan_infinities_and_empty_rows(kernels):
    rng = np.random.default_rng(7)
    l = rng.standard_normal((6, 5000)).astype(np.float32)
    l[0, ::2] = np.nan
    l[1, 17] = np.inf           # no value in the whole row
    l[2] = -np.inf              # all masked
    l[3] = np.nan
    l[4, 1:] = -np.inf          # one token left
    sc = np.array([0, 0, 0, 0, -1, np.nan], np.float32)
    _check(kernels, l, sc, None, 0, 1, 6, 5000, 16)
    _check(kernels, l[1:4].copy(), sc[1:4], None, 0, 1, 3, 5000, 8)  # nothing at all
    _check(kernels, l, sc, None, 0, 6, 1, 5000, 3)


def test_extreme_logits_and_scores(kernels):
    rng = np.random.default_rng(8)
    l = (rng.standard_normal((4, 3000)) * 1e4).astype(np.float32)
    l[1] = -3e38
    l[1, 5] = 3e38
    sc = np.array([-1e4, 0, -3e38, -5], np.float32)
    v, rows, tok = _run(kernels, l, sc, None, 0, 1, 4, 3000, 8)
    wv, wr, wt = _want(l, sc, None, 0, 1, 4, 3000, 8)
    assert np.array_equal(rows, wr) and np.array_equal(tok, wt)


def test_all_beams_ended(kernels):
    rng = np.random.default_rng(9)
    l = rng.standard_normal((8, 50)).astype(np.float32)
    sc = (-rng.random(8)).astype(np.float32)
    sc[5] = -np.inf
    for pad in (0, 2, 49):
        _check(kernels, l, sc, np.ones(8, np.uint8), pad, 2, 4, 50, 8)


def test_scores_in_place_and_the_same_bits(kernels):
    import torch

    R, W, V = 3, 4, 30000
    g = torch.Generator(device="cuda").manual_seed(3)
    l = torch.randn(R * W, V, generator=g, device="cuda") * 2
    sc = -torch.rand(R * W, generator=g, device="cuda")
    ws = torch.empty(kernels.beam_select_workspace_size(R, W, V, W), dtype=torch.uint8, device="cuda")
    got = []
    for place in (False, True, True):
        s = sc.clone()
        v = s if place else torch.empty_like(s)
        rows, tok = (torch.empty(R, W, dtype=torch.int32, device="cuda") for _ in range(2))
        assert kernels.beam_select(l, s, None, 0, R, W, V, W, v, rows, tok, ws) == 0
        kernels.sync()
        got.append((v.clone().view(-1), rows, tok))
    for o in got[1:]:
        assert all(torch.equal(a, b) for a, b in zip(got[0], o))


@pytest.mark.parametrize("shape,used,dt", [
    ((6, 64), None, "float32"), ((6, 3, 20), None, "int8"), ((6, 3, 20), 13, "int8"), ((6, 2, 50000), 66666, "bfloat16"),
    ((6, 100003), None, "uint8"), ((6, 5, 32), 0, "float32"), ((6, 4, 9000), 16388, "float32"),
])
def test_reorder(kernels, shape, used, dt):
    import torch

    import streamoe_amd as sa

    g = torch.Generator(device="cuda").manual_seed(1)
    dtype = getattr(torch, dt)
    size = torch.empty(0, dtype=dtype).element_size()
    rows = torch.tensor([5, 0, 0, 3], dtype=torch.int32, device="cuda")
    states, wants = [], []
    for i in range(3):
        src = torch.randint(0, 100, shape, generator=g, device="cuda").to(dtype)
        dst = torch.full(shape, 101, device="cuda").to(dtype)
        want = dst.clone()
        n = shape[-1] if used is None else used // size
        want[:4, ..., :n] = src[rows.long()][..., :n]
        if used is not None and used % size:
            want.view(torch.uint8)[:4, ..., :used] = src[rows.long()].view(torch.uint8)[..., :used]
        states.append(sa.BeamState(src, dst, used))
        wants.append(want)
    assert kernels.beam_reorder(states, rows) == 0
    kernels.sync()
    for s, w in zip(states, wants):
        assert torch.equal(s.dst, w)


def test_reorder_many_states_strided(kernels):
    """More states than one launch takes; rows, pieces and starts of any stride."""
    import torch

    import streamoe_amd as sa

    rows = torch.tensor([1, 2, 0], dtype=torch.int32, device="cuda")
    states, wants = [], []
    for i in range(75):
        big = torch.randint(0, 255, (3, 7, 1000 + i), device="cuda", dtype=torch.uint8)
        out = torch.full((7, 3, 1200), 255, device="cuda", dtype=torch.uint8)
        src = big[:, 1:5, i % 3:900]
        dst = out.transpose(0, 1)[:, 2:6, 5:5 + src.shape[2]]  # pieces outside, rows inside
        want = out.clone()
        want.transpose(0, 1)[:, 2:6, 5:5 + src.shape[2]] = src[rows.long()]
        states.append(sa.BeamState(src, dst))
        wants.append((out, want))
    assert kernels.beam_reorder(states, rows) == 0
    kernels.sync()
    for out, want in wants:
        assert torch.equal(out, want)


def test_reorder_bad_row_is_reported(kernels):
    import torch

    import streamoe_amd as sa

    src = torch.arange(40, device="cuda", dtype=torch.float32).view(4, 10)
    dst = torch.full((4, 10), -1.0, device="cuda")
    rows = torch.tensor([3, -1, 4, 1], dtype=torch.int32, device="cuda")
    assert kernels.beam_reorder([sa.BeamState(src, dst)], rows) == 0
    with pytest.raises(sa.SmoeError, match="INVALID_ARG"):
        kernels.sync()
    assert torch.equal(dst[0], src[3]) and torch.equal(dst[3], src[1]) and torch.all(dst[1:3] == -1)
    kernels.sync()


def test_misfit_tensors_are_refused(kernels):
    import torch

    import streamoe_amd as sa

    src, dst = torch.zeros(4, 10, device="cuda"), torch.zeros(4, 10, device="cuda")
    rows = torch.zeros(4, dtype=torch.int32, device="cuda")
    assert kernels.beam_reorder([], rows) == 1
    assert kernels.beam_reorder([sa.BeamState(src, dst)], rows.long()) == 1
    assert kernels.beam_reorder([sa.BeamState(src, dst[:3])], rows) == 1
    assert kernels.beam_reorder([sa.BeamState(src, src)], rows) == 1
    for bad in (sa.BeamState(src, dst.half()), sa.BeamState(src, dst[:, :9]), sa.BeamState(src, dst, 41),
                sa.BeamState(src.t(), dst.t())):
        with pytest.raises(sa.SmoeError):
            kernels.beam_reorder([bad], rows)


def test_graph_of_a_beam_step(kernels):
    """Selection and reordering captured together and replayed."""
    import torch

    import streamoe_amd as sa

    R, W, V = 2, 4, 20000
    g = torch.Generator(device="cuda").manual_seed(4)
    l = torch.randn(R * W, V, generator=g, device="cuda")
    sc = -torch.rand(R * W, generator=g, device="cuda")
    v = torch.empty(R, W, device="cuda")
    rows, tok = (torch.empty(R, W, dtype=torch.int32, device="cuda") for _ in range(2))
    ws = torch.empty(kernels.beam_select_workspace_size(R, W, V, W), dtype=torch.uint8, device="cuda")
    src = torch.randn(R * W, 5000, generator=g, device="cuda")
    dst = torch.empty_like(src)

    def step():
        sa.check(kernels.beam_select(l, sc, None, 0, R, W, V, W, v, rows, tok, ws), "select")
        sa.check(kernels.beam_reorder([sa.BeamState(src, dst)], rows.view(-1)), "reorder")

    graph = sa.capture_graph(kernels, step)
    for _ in range(3):
        l.normal_(generator=g)
        graph.replay()
        torch.cuda.synchronize()
        got = [t.clone() for t in (v, rows, tok, dst)]
        step()
        kernels.sync()
        assert all(torch.equal(a, b) for a, b in zip(got, (v, rows, tok, dst)))
        wv, wr, wt = _want(l.cpu().numpy(), sc.cpu().numpy(), None, 0, R, W, V, W)
        assert np.array_equal(got[1].cpu().numpy(), wr) and np.array_equal(got[2].cpu().numpy(), wt)
