"""How near to a border the rows of tests/test_gpu_sample.py come, on the CPU.

smoe_sample holds a mass as an integer of 2^-s, s = 62 - bits of vocab but at most
51, off by half of it, out of an exponential off by 2^-44 of itself. A running sum of
V masses, and top_p (at most once) or u (less than once) of another, are each off by
up to V 2^-s / 2 + 2^-44 of the sum. A mass next to min_p is off by its exponential.
So a row whose borders are further than

  V 2^-s + 2^-43 sum

from every running sum has one token, which the kernels have to give; nearer ones
may fall to either side. Here every row that those tests hold to one token is held to
that distance, and its token formed again, with sums in 80 bits (off by V 2^-63 of
themselves, which is added), but for rows of equal masses, whose sums are exact on
both sides, and vocabularies of three and less."""
import numpy as np
import pytest

import test_gpu_sample as rows


def _token(l, t, k, p, m, u):
    """(token, distance of the nearest border, what that may be off by)."""
    V, L = len(l), np.longdouble
    at = np.flatnonzero(~np.isnan(l) & (l > -np.inf))
    at = at[np.lexsort((at, -l[at].astype(np.float64)))]
    if not len(at) or t == 0:
        return (at[0] if len(at) else -1), 1.0, 0.0
    e = (l[at] == np.inf).astype(L) if l[at[0]] == np.inf else np.exp((l[at].astype(L) - L(l[at[0]])) / L(t))
    room = V * 2.0 ** -min(51, 62 - (V - 1).bit_length()) + float(2.0 ** -43 + V * 2.0 ** -62) * float(e.sum())
    near, keep = [1.0], len(at) if k <= 0 else min(k, len(at))
    if p < 1:
        before = np.concatenate([[L(0)], np.cumsum(e[:keep])])
        target = L(p) * before[-1]
        inner = before[1:-1]  # of the second key and on: the first is kept in any case
        near += [abs(inner - target).min()] if len(inner) and p > 0 else []
        keep = 1 + int((inner < target).sum())
    if 0 < m < 1:
        near.append(abs(e - L(m)).min())
    keep = min(keep, int((e >= L(m)).sum()))
    by = np.argsort(at[:keep])
    upto = np.cumsum(e[:keep][by])
    near += [abs(upto[:-1] - L(u) * upto[-1]).min()] if keep > 1 else []
    return at[by[min(int((upto <= L(u) * upto[-1]).sum()), keep - 1)]], float(min(near)), room


def _held(monkeypatch, call):
    """Rows nearer to a border than the room, of those that `call` checks."""
    near_ones, n = [], 0

    def check(kernels, l, t, k, p, m, u, apart=1e-7):
        nonlocal n
        f = lambda a: np.asarray(a, np.float32)
        l, t, p, m, u = f(l), f(t), f(p), f(m), f(u)
        for i in range(len(u)):
            n += 1
            token, near, room = _token(l[i], t[i], k[i], p[i], m[i], u[i])
            assert token == rows.want_of(l[i], t[i], k[i], p[i], m[i], u[i])[0]
            if near <= room:
                near_ones.append((i, near, room))

    monkeypatch.setattr(rows, "_check", check)
    call()
    assert n
    return near_ones


@pytest.mark.parametrize("V", [31, 1000, 1024, 1025, 5003, 50000, 151936, 262145])
@pytest.mark.parametrize("sigma", [0.3, 2.5, 20.0])
def test_filters(monkeypatch, V, sigma):
    assert not _held(monkeypatch, lambda: rows.test_filters(None, V, sigma))


@pytest.mark.parametrize("n", [1, 2, 33, 200, 1100])
def test_batches(monkeypatch, n):
    assert not _held(monkeypatch, lambda: rows.test_batches(None, n))


@pytest.mark.parametrize("kind", ["equal", "zeros", "masked_most", "lowest", "inf", "two_inf", "steps", "huge", "tiny"])
def test_kinds(monkeypatch, kind):
    assert not _held(monkeypatch, lambda: rows.test_rows_of_all_kinds(None, kind))


@pytest.mark.parametrize("V", [700, 5003, 40001])
def test_far(monkeypatch, V):
    assert not _held(monkeypatch, lambda: rows.test_logits_further_apart_than_f32_goes(None, V))


@pytest.mark.parametrize("V", [400, 3000, 20000])
def test_ties(monkeypatch, V):
    assert not _held(monkeypatch, lambda: rows.test_more_ties_than_top_k(None, V))
