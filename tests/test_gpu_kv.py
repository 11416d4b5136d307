"""smoe_kv_append and smoe_kv_gather against plain indexing: bf16 rows and codes
bit for bit (each is one correctly rounded operation), values read back as the
f32 product rounded once."""
import numpy as np
import pytest

from kv_cases import Cache, ints

pytestmark = pytest.mark.gpu


def _bits(t):
    import torch

    return t.contiguous().view({2: torch.int16, 1: torch.int8, 4: torch.int32}[t.element_size()]).cpu().numpy()


def _tokens(cache, rng, n, pad):
    """n different held positions in any order, and padding among them."""
    every = [(s, p) for s, m in enumerate(cache.lens) for p in range(m)]
    some = [every[i] for i in rng.permutation(len(every))[:n]]
    for _ in range(pad):
        some.insert(int(rng.integers(0, len(some) + 1)), (-1, int(rng.integers(-5, 5))))
    return np.array(some, np.int64)


def _place(cache, tok):
    on = tok[:, 0] >= 0
    s, p = tok[on, 0], tok[on, 1]
    return on, cache.table_host[s, p // cache.page], p % cache.page


def _rows(rng, n, heads, dim, bf16, fused=True):
    import torch

    kv = torch.tensor(rng.standard_normal((n, 3 * heads * dim)), dtype=torch.bfloat16 if bf16 else torch.float32, device="cuda")
    w = heads * dim
    k, v = kv[:, w:2 * w].unflatten(1, (heads, dim)), kv[:, 2 * w:].unflatten(1, (heads, dim))
    return (k, v) if fused else (k.contiguous(), v.contiguous())


def _codes(x):
    """codes and scale of rows [.., dim] by the definition, in f32."""
    x = np.asarray(x, np.float32)
    with np.errstate(all="ignore"):
        top = np.abs(x).max(-1)
        bad = ~np.isfinite(x).all(-1)
        small = top < np.float32(2.0 ** -119)
        scale = np.where(bad, np.float32("nan"), np.where(small, np.float32(0), top / np.float32(127)))
        q = np.where((bad | small)[..., None], 0, np.rint(x / scale[..., None]))
    return q.astype(np.int8), scale.astype(np.float32)


SHAPES = [(2, 256, 16), (8, 128, 16), (1, 64, 32), (3, 80, 48), (5, 16, 16), (16, 128, 64), (2, 240, 1024)]


@pytest.mark.parametrize("heads,dim,page", SHAPES)
@pytest.mark.parametrize("bits", [16, 8])
@pytest.mark.parametrize("x_bf16", [True, False])
@pytest.mark.parametrize("layout", ["heads", "slots", "both", "apart"])
def test_append(kernels, heads, dim, page, bits, x_bf16, layout):
    import torch

    rng = np.random.default_rng(heads + dim + bits)
    cache = Cache([1, 40, 17, 129], heads, dim, bits, page, seed=dim, layout=layout)
    tok = _tokens(cache, rng, 61, 4)
    n = len(tok)
    k, v = _rows(rng, n, heads, dim, x_bf16)
    before = [_bits(t) for t in (cache.k, cache.v)] + [None if t is None else _bits(t) for t in (cache.ks, cache.vs)]
    gap = _bits(cache.k._base) if layout == "apart" else None
    assert kernels.kv_append(cache.c, cache.table, ints(tok[:, 0]), ints(tok[:, 1]), k, v, n) == 0
    kernels.sync()
    on, page_of, slot = _place(cache, tok)
    for i, (x, got, sc) in enumerate(((k, cache.k, cache.ks), (v, cache.v, cache.vs))):
        x = x.float().cpu().numpy()[on]
        want = before[i].copy()
        if bits == 16:
            want[page_of, :, slot] = _bits(torch.tensor(x).to(torch.bfloat16))
        else:
            q, s = _codes(x)
            want[page_of, :, slot] = q
            scales = before[2 + i].copy()
            scales[page_of, :, slot] = s.view(np.int32)
            assert np.array_equal(_bits(sc), scales)
        assert np.array_equal(_bits(got), want)
    if gap is not None:  # what lies between rows
        now = _bits(cache.k._base)
        assert np.array_equal(now[..., :16], gap[..., :16]) and np.array_equal(now[..., 16 + dim:], gap[..., 16 + dim:])


@pytest.mark.parametrize("heads,dim,page", SHAPES)
@pytest.mark.parametrize("bits", [16, 8])
@pytest.mark.parametrize("out_bf16", [True, False])
@pytest.mark.parametrize("layout", ["heads", "slots", "both", "apart"])
def test_gather(kernels, heads, dim, page, bits, out_bf16, layout):
    import torch

    rng = np.random.default_rng(heads + dim + bits)
    cache = Cache([3, 70, 16, 201], heads, dim, bits, page, seed=dim, layout=layout)
    tok = _tokens(cache, rng, 77, 5)
    tok = np.concatenate([tok, tok[:9]])  # some again
    n = len(tok)
    t = torch.bfloat16 if out_bf16 else torch.float32
    out = torch.full((n + 1, 2 * heads * dim + 16), 7.0, dtype=t, device="cuda")
    k, v = out[:, :heads * dim], out[:, heads * dim:2 * heads * dim]
    assert kernels.kv_gather(cache.c, cache.table, ints(tok[:, 0]), ints(tok[:, 1]), k, v, n) == 0
    kernels.sync()
    on, page_of, slot = _place(cache, tok)
    for i, got in enumerate((k, v)):
        want = np.zeros((n, heads, dim), np.float32)
        if bits == 16:
            want[on] = cache.value[i][page_of, :, slot]
        else:
            c = (cache.k, cache.v)[i].cpu().numpy()[page_of, :, slot].astype(np.float32)
            want[on] = c * cache.scale_host[i].numpy()[page_of, :, slot][..., None]
        assert np.array_equal(_bits(got[:n]).reshape(n, -1), _bits(torch.tensor(want.reshape(n, -1)).to(t)))
    assert torch.all(out[n] == 7) and torch.all(out[:, 2 * heads * dim:] == 7)


@pytest.mark.parametrize("bits", [16, 8])
@pytest.mark.parametrize("n", [1, 2, 3, 4, 5, 300, 1000, 1025, 1030, 2049, 5001, 16384])
def test_the_last_of_a_position_stays(kernels, bits, n):
    """Few positions, named over and over: each holds its last row, whole."""
    import torch

    rng = np.random.default_rng(n)
    cache = Cache([40, 7], 2, 64, bits, 16, seed=n)
    tok = np.array([(0, p) if p < 40 else (1, p - 40) for p in rng.integers(0, 47, n)])
    k, v = _rows(rng, n, 2, 64, False, fused=False)
    assert kernels.kv_append(cache.c, cache.table, ints(tok[:, 0]), ints(tok[:, 1]), k, v, n) == 0
    kernels.sync()
    last = {(s, p): i for i, (s, p) in enumerate(tok.tolist())}
    for (s, p), i in last.items():
        at = cache.table_host[s, p // 16]
        for x, c, sc in ((k, cache.k, cache.ks), (v, cache.v, cache.vs)):
            got = c[at, :, p % 16].cpu()
            if bits == 16:
                assert torch.equal(got, x[i].to(torch.bfloat16).cpu())
            else:
                q, scale = _codes(x[i].cpu().numpy())
                assert np.array_equal(got.numpy(), q) and np.array_equal(sc[at, :, p % 16].cpu().numpy(), scale)


def test_rows_that_are_no_numbers(kernels):
    import torch

    cache = Cache([30], 1, 64, 8, 16, seed=5)
    x = torch.randn(6, 1, 64, device="cuda")
    x[0, 0, 3] = float("nan")
    x[1, 0, 63] = float("inf")
    x[2, 0, 0] = -float("inf")
    x[3] = 0
    x[4] = 1e-37
    x[5] *= 1e37
    assert kernels.kv_append(cache.c, cache.table, ints([0] * 6), ints(range(6)), x, x, 6) == 0
    k, v = (torch.empty(6, 64, device="cuda") for _ in range(2))
    assert kernels.kv_gather(cache.c, cache.table, ints([0] * 6), ints(range(6)), k, v, 6) == 0
    kernels.sync()
    q, s = _codes(x.cpu().numpy())
    at = cache.table_host[0, 0]
    assert np.array_equal(cache.k[at, :, :6].cpu().numpy(), q.transpose(1, 0, 2))
    got = cache.ks[at, :, :6].cpu().numpy()
    assert np.array_equal(got, s.T, equal_nan=True)
    assert torch.all(k[:3].isnan()) and torch.all(k[3:5] == 0) and torch.equal(k.nan_to_num(), v.nan_to_num())


def test_what_is_out_of_range_is_reported_and_left_out(kernels):
    import torch

    import streamoe_amd as sa

    for bits in (16, 8):
        cache = Cache([40, 40], 2, 64, bits, 16, seed=9)
        cache.table[1, 1] = cache.pages  # no page
        cache.table[1, 0] = -1
        good = [(0, 3), (0, 39), (1, 33)]
        bad = [(2, 0), (-2, 0), (0, -1), (0, cache.width * 16), (1, 17), (1, 2), (2 ** 31 - 1, 2 ** 31 - 1), (-2 ** 31, 5)]
        tok = np.array([x for pair in zip(bad, good * 3) for x in pair])
        n = len(tok)
        k, v = _rows(np.random.default_rng(1), n, 2, 64, True)
        before = _bits(cache.k)
        assert kernels.kv_append(cache.c, cache.table, ints(tok[:, 0]), ints(tok[:, 1]), k, v, n) == 0
        with pytest.raises(sa.SmoeError, match="INVALID_ARG"):
            kernels.sync()
        kernels.sync()
        want = before.copy()
        for i, (s, p) in enumerate(tok.tolist()):
            if (s, p) in good:
                x = k[i]
                want[cache.table_host[s, p // 16], :, p % 16] = _bits(x) if bits == 16 else _codes(x.float().cpu().numpy())[0]
        assert np.array_equal(_bits(cache.k), want)
        ko, vo = (torch.full((n, 2, 64), 7.0, device="cuda") for _ in range(2))
        assert kernels.kv_gather(cache.c, cache.table, ints(tok[:, 0]), ints(tok[:, 1]), ko, vo, n) == 0
        with pytest.raises(sa.SmoeError, match="INVALID_ARG"):
            kernels.sync()
        for i, (s, p) in enumerate(tok.tolist()):
            assert ((s, p) in good) != bool(torch.all(ko[i] == 0))


def test_offsets_past_32_bits(kernels):
    """Pages 5 GB apart from the first."""
    import torch

    import streamoe_amd as sa

    for bits, t in ((16, torch.bfloat16), (8, torch.int8)):
        pages = 11 << 10 if bits == 16 else 22 << 10
        k, v = (torch.zeros(pages, 2, 1024, 128, dtype=t, device="cuda") for _ in range(2))
        ks, vs = (torch.zeros(pages, 2, 1024, device="cuda") if bits == 8 else None for _ in range(2))
        cache = sa.KvCache(k, v, ks, vs)
        table = ints([[pages - 1, 0]])
        x, y = torch.randn(2, 2, 2, 128, device="cuda").to(torch.bfloat16)
        seq, pos = ints([0, 0]), ints([1023, 1024])
        assert kernels.kv_append(cache, table, seq, pos, x, y, 2) == 0
        ko, vo = (torch.empty(2, 2, 128, dtype=torch.bfloat16, device="cuda") for _ in range(2))
        assert kernels.kv_gather(cache, table, seq, pos, ko, vo, 2) == 0
        kernels.sync()
        room = 0 if bits == 16 else 0.5 / 127 + 2 ** -8
        for a, b in ((x, ko), (y, vo)):
            assert torch.all((a.float() - b.float()).abs() <= room * a.float().abs().amax(2, keepdim=True))
        assert bool(k[pages - 1, :, 1023].any()) and bool(k[0, :, 0].any()) and not bool(k[0, :, 1:].any())
        del k, v, ks, vs, cache
        torch.cuda.empty_cache()
