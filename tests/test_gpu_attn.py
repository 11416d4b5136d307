"""smoe_attn_decode against the definition in 64 bits (kv_cases.attention has the
bounds). Everything in the cache, its scales and its table that a token does not
see is garbage."""
import numpy as np
import pytest

from kv_cases import BF16, Cache, attention, ints

pytestmark = pytest.mark.gpu


def _run(kernels, cache, tok, q, scale, window, out_bf16, heads, ws=None):
    import torch

    n = len(tok)
    out = torch.full((n + 1, heads, cache.dim), 7.0, dtype=torch.bfloat16 if out_bf16 else torch.float32, device="cuda")
    if ws is None:
        size = kernels.attn_decode_workspace_size(cache.c, heads, n)
        ws = torch.randint(0, 256, (size,), dtype=torch.uint8, device="cuda")  # anything
    assert kernels.attn_decode(cache.c, cache.table, ints(tok[:, 0]), ints(tok[:, 1]), q, scale, window, out, heads, n, ws) == 0
    kernels.sync()
    assert torch.all(out[n] == 7)
    return out[:n]


def _check(cache, tok, q, scale, window, got, out_bf16):
    got = got.double().cpu().numpy()
    qh = q.double().cpu().numpy().reshape(len(tok), -1, cache.dim)
    for i, (s, p) in enumerate(tok.tolist()):
        if s < 0:
            assert np.all(got[i] == 0), i
            continue
        lo = max(0, p + 1 - window) if window else 0
        k, v = (cache.rows(j, s, p + 1)[lo:] for j in range(2))
        want, room = attention(k, v, qh[i], scale)
        if out_bf16:
            room = room + BF16 * (np.abs(want) + room)
        assert np.all(np.abs(got[i] - want) <= room), (i, s, p, np.max(np.abs(got[i] - want) / room))


def _queries(rng, n, heads, dim, bf16, fused=False, sigma=1.0):
    import torch

    q = torch.tensor(rng.standard_normal((n, heads * dim * (2 if fused else 1))) * sigma, device="cuda")
    q = q.to(torch.bfloat16 if bf16 else torch.float32)
    return (q[:, heads * dim:] if fused else q).unflatten(1, (heads, dim))


HEADS = [(16, 2, 256), (16, 16, 128), (32, 8, 128), (8, 1, 64), (6, 3, 80), (40, 2, 128), (20, 4, 96), (9, 3, 160), (7, 7, 16),
         (33, 1, 48), (2, 2, 240), (16, 1, 64), (48, 3, 256)]


@pytest.mark.parametrize("heads,kv_heads,dim", HEADS)
@pytest.mark.parametrize("bits", [16, 8])
@pytest.mark.parametrize("x_bf16,out_bf16", [(True, True), (False, False), (True, False)])
def test_ragged_batch(kernels, heads, kv_heads, dim, bits, x_bf16, out_bf16):
    rng = np.random.default_rng(heads * dim + bits)
    lens = [1, 2, 15, 16, 17, 31, 33, 127, 128, 129, 300, 1025]
    cache = Cache(lens, kv_heads, dim, bits, 16 if heads % 3 else 48, seed=heads + dim)
    tok = np.array([(s, n - 1) for s, n in enumerate(lens)] + [(-1, 0), (11, 700), (-1, -3), (3, 0)])
    tok = tok[rng.permutation(len(tok))]
    q = _queries(rng, len(tok), heads, dim, x_bf16)
    got = _run(kernels, cache, tok, q, dim ** -0.5, 0, out_bf16, heads)
    _check(cache, tok, q, dim ** -0.5, 0, got, out_bf16)


@pytest.mark.parametrize("layout", ["slots", "both", "apart"])
@pytest.mark.parametrize("bits", [16, 8])
@pytest.mark.parametrize("heads,kv_heads,dim", [(8, 2, 256), (12, 4, 64), (5, 1, 112), (4, 4, 128)])
def test_layouts(kernels, layout, bits, heads, kv_heads, dim):
    rng = np.random.default_rng(dim)
    lens = [500, 3, 130]
    cache = Cache(lens, kv_heads, dim, bits, 64, seed=dim, layout=layout)
    tok = np.array([(s, n - 1) for s, n in enumerate(lens)])
    q = _queries(rng, 3, heads, dim, True, fused=True)
    got = _run(kernels, cache, tok, q, 0.1, 0, False, heads)
    _check(cache, tok, q, 0.1, 0, got, False)


@pytest.mark.parametrize("heads,kv_heads,dim", [(16, 2, 256), (8, 8, 64), (32, 8, 128), (34, 2, 96)])
@pytest.mark.parametrize("bits", [16, 8])
@pytest.mark.parametrize("window", [0, 1, 5, 16, 100, 1000, 2 ** 32 - 1])
def test_tokens_of_one_sequence_and_windows(kernels, heads, kv_heads, dim, bits, window):
    """Runs of positions that share tiles, at any place of the call; each sees
    its own positions."""
    rng = np.random.default_rng(window % 1000 + dim)
    lens = [700, 260, 40]
    cache = Cache(lens, kv_heads, dim, bits, 32, seed=window % 99)
    tok = [(0, p) for p in range(640, 700)] + [(2, p) for p in range(40)] + [(-1, 0)] * 3
    tok += [(1, p) for p in (255, 256, 257, 259, 258, 257, 0, 1, 2, 128)] + [(0, 5), (0, 6), (1, 7)]
    tok = np.array(tok)
    q = _queries(rng, len(tok), heads, dim, False)
    got = _run(kernels, cache, tok, q, dim ** -0.5, window, False, heads)
    _check(cache, tok, q, dim ** -0.5, min(window, 1 << 30), got, False)


@pytest.mark.parametrize("n", [300, 1000])
def test_many_rows(kernels, n):
    rng = np.random.default_rng(n)
    lens = [int(x) for x in rng.integers(1, 200, 50)]
    cache = Cache(lens, 2, 64, 16, 16, seed=n)
    tok = np.array([(s, int(rng.integers(0, lens[s]))) if rng.random() < 0.9 else (-1, 0) for s in rng.integers(0, 50, n)])
    q = _queries(rng, n, 6, 64, True)
    got = _run(kernels, cache, tok, q, 0.125, 0, True, 6)
    _check(cache, tok, q, 0.125, 0, got, True)


@pytest.mark.parametrize("heads,kv_heads,dim,bits", [(256, 256, 16, 8), (4096, 1, 16, 16), (480, 240, 32, 16), (4080, 240, 16, 8)])
def test_many_heads(kernels, heads, kv_heads, dim, bits):
    rng = np.random.default_rng(heads)
    cache = Cache([70, 200], kv_heads, dim, bits, 16, seed=heads, spare=1)
    tok = np.array([(1, 199), (0, 69), (-1, 0), (0, 3)])
    q = _queries(rng, 4, heads, dim, True)
    got = _run(kernels, cache, tok, q, 0.25, 0, False, heads)
    _check(cache, tok, q, 0.25, 0, got, False)


def test_the_most_tokens(kernels):
    """16384 rows: prompts of many sequences in one call, one row in seven padding."""
    rng = np.random.default_rng(16)
    lens = [64] * 220
    cache = Cache(lens, 1, 64, 16, 32, seed=16)
    tok = np.array([(s, p) for s in range(220) for p in range(64)], np.int64)
    tok = np.concatenate([tok, np.full((16384 - len(tok), 2), -1)])
    tok[::7, 0] = -1
    q = _queries(rng, len(tok), 4, 64, True)
    got = _run(kernels, cache, tok, q, 0.125, 0, False, 4)
    some = np.sort(rng.permutation(len(tok))[:700])
    _check(cache, tok[some], q[some], 0.125, 0, got[some], False)


@pytest.mark.parametrize("bits", [16, 8])
@pytest.mark.parametrize("length,page", [(70001, 64), (66000, 16), (65536, 1 << 17)])
def test_one_long_sequence(kernels, bits, length, page):
    rng = np.random.default_rng(length)
    cache = Cache([length, 5], 2, 64, bits, page, seed=3, spare=1)
    tok = np.array([(0, length - 1), (1, 4)])
    q = _queries(rng, 2, 8, 64, False)
    got = _run(kernels, cache, tok, q, 0.125, 0, False, 8)
    _check(cache, tok, q, 0.125, 0, got, False)


def test_scores_of_any_size(kernels):
    """One key far above the others, late and early; queries large and zero."""
    def kv(rng, shape, i):
        x = rng.standard_normal(shape)
        if i == 0:
            x[:, :, 5] *= 30
        return x

    rng = np.random.default_rng(8)
    cache = Cache([600, 200, 6], 2, 128, 16, 16, seed=4, kv=kv)
    tok = np.array([(0, 599), (1, 199), (2, 5), (0, 3)])
    for sigma in (0.0, 1.0, 8.0):
        q = _queries(rng, 4, 8, 128, False, sigma=sigma)
        for scale in (0.09, -0.09, 0.0):
            got = _run(kernels, cache, tok, q, scale, 0, False, 8)
            _check(cache, tok, q, scale, 0, got, False)


@pytest.mark.parametrize("bits", [16, 8])
@pytest.mark.parametrize("bad", [float("nan"), float("inf")])
@pytest.mark.parametrize("window", [0, 6])
def test_what_one_token_must_not_see_may_hold_anything(kernels, bits, bad, window):
    """A NaN or an infinity at position 37 of a run of tokens: those that see it
    have no number (but where a key's infinity makes a score of -inf), the others
    are as if it were not there."""
    import torch

    rng = np.random.default_rng(2)
    for which in ("k", "v"):
        cache = Cache([50], 2, 128, bits, 16, seed=6)
        at = int(cache.table_host[0, 37 // 16])
        if bits == 16:
            getattr(cache, which)[at, :, 37 % 16, 3] = bad
        else:
            getattr(cache, which + "s")[at, :, 37 % 16] = bad
        tok = np.array([(0, p) for p in range(30, 50)])
        q = _queries(rng, len(tok), 4, 128, True)
        got = _run(kernels, cache, tok, q, 0.09, window, False, 4)
        sees = [p >= 37 and (not window or p - window < 37) for p in range(30, 50)]
        rest = np.array([i for i in range(20) if not sees[i]])
        _check(cache, tok[rest], q[rest], 0.09, window, got[rest], False)
        for i in range(20):
            if sees[i] and (bad != bad or which == "v"):
                assert not bool(torch.isfinite(got[i]).all())


def test_what_is_out_of_range_is_reported(kernels):
    import streamoe_amd as sa

    import torch

    rng = np.random.default_rng(3)
    cache = Cache([300, 60, 20], 2, 64, 16, 16, seed=7)
    held = cache.table_host.copy()
    cache.table[0, 4] = -1           # positions 64 .. 79 of sequence 0
    cache.table[0, 7] = cache.pages  # 112 .. 127
    tok = np.array([(0, 299), (1, 59), (3, 0), (-2, 1), (1, -1), (1, cache.width * 16), (2, 19), (2, 20 * 2 ** 25)])
    q = _queries(rng, len(tok), 4, 64, False)
    n = len(tok)
    out = torch.empty(n, 4, 64, device="cuda")
    ws = torch.empty(kernels.attn_decode_workspace_size(cache.c, 4, n), dtype=torch.uint8, device="cuda")
    assert kernels.attn_decode(cache.c, cache.table, ints(tok[:, 0]), ints(tok[:, 1]), q, 0.125, 0, out, 4, n, ws) == 0
    with pytest.raises(sa.SmoeError, match="INVALID_ARG"):
        kernels.sync()
    kernels.sync()
    good = np.array([1, 6])
    _check(cache, tok[good], q[good], 0.125, 0, out[good], False)
    assert torch.all(out[torch.tensor([2, 3, 4, 5, 7])] == 0)
    # The row whose pages are missing: the others' positions.
    p = np.array([x for x in range(300) if x // 16 not in (4, 7)])
    k, v = (cache.value[j][held[0, p // 16], :, p % 16] for j in range(2))
    want, room = attention(k, v, q[0].double().cpu().numpy(), 0.125)
    assert np.all(np.abs(out[0].double().cpu().numpy() - want) <= room)
    # A missing page alone is reported too, but not where no token sees it.
    for pos, window, code in ((299, 0, True), (299, 100, False), (60, 0, False), (130, 3, False), (130, 5, True)):
        one = np.array([(0, pos)])
        assert kernels.attn_decode(cache.c, cache.table, ints([0]), ints([pos]), q[:1], 0.125, window, out, 4, 1, ws) == 0
        if code:
            with pytest.raises(sa.SmoeError, match="INVALID_ARG"):
                kernels.sync()
        else:
            kernels.sync()
            _check(cache, one, q[:1], 0.125, window, out[:1], False)


def test_nothing_but_padding(kernels):
    import torch

    cache = Cache([5], 2, 64, 8, 16, seed=1)
    for n in (1, 5, 700):
        tok = np.full((n, 2), -1)
        q = torch.full((n, 4, 64), float("nan"), device="cuda")
        got = _run(kernels, cache, tok, q, 0.1, 0, n == 5, 4)
        assert torch.all(got == 0)


def test_offsets_past_32_bits(kernels):
    import torch

    import streamoe_amd as sa

    for bits, t in ((16, torch.bfloat16), (8, torch.int8)):
        pages = 11 << 10 if bits == 16 else 22 << 10
        k, v = (torch.zeros(pages, 2, 1024, 128, dtype=t, device="cuda") for _ in range(2))
        sc = [torch.full((pages, 2, 1024), 0.01, device="cuda") if bits == 8 else None for _ in range(2)]
        g = torch.Generator(device="cuda").manual_seed(1)
        for x in (k, v):
            for p in (pages - 1, pages - 2):
                x[p] = (torch.randn(2, 1024, 128, generator=g, device="cuda") * (1 if bits == 16 else 40)).clamp(-127, 127).to(t)
        cache = sa.KvCache(k, v, *sc)
        table = ints([[pages - 1, pages - 2]])
        q = torch.randn(1, 4, 128, generator=g, device="cuda")
        out = torch.empty(1, 4, 128, device="cuda")
        ws = torch.empty(kernels.attn_decode_workspace_size(cache, 4, 1), dtype=torch.uint8, device="cuda")
        assert kernels.attn_decode(cache, table, ints([0]), ints([1500]), q, 0.09, 0, out, 4, 1, ws) == 0
        kernels.sync()
        f = 1 if bits == 16 else float(np.float32(0.01))
        kk, vv = (torch.cat([x[pages - 1], x[pages - 2]], 1)[:, :1501].transpose(0, 1).double().cpu().numpy() * f for x in (k, v))
        want, room = attention(kk, vv, q[0].double().cpu().numpy(), 0.09)
        assert np.all(np.abs(out[0].double().cpu().numpy() - want) <= room)
        del k, v, sc, cache
        torch.cuda.empty_cache()
