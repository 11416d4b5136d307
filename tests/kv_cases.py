"""A paged cache with shuffled pages, what its positions hold in 64 bits, and the
definitions that the cache and attention tests compare with."""
import numpy as np

U = 2.0 ** -24
BF16 = 2.0 ** -8  # half a step of bf16, relative


class Cache:
    """seqs: positions held of every sequence. Everything that no position holds
    (other slots, pages, scales, table entries) is garbage: NaN, or codes and ids
    of any kind."""

    def __init__(self, lens, heads, dim, bits, page, seed, layout="heads", spare=3, kv=None):
        import torch

        import streamoe_amd as sa

        rng = np.random.default_rng(seed)
        self.lens, self.heads, self.dim, self.bits, self.page = list(lens), heads, dim, bits, page
        need = [(n + page - 1) // page for n in lens]
        self.width = max(need) + 2
        self.pages = sum(need) + spare
        ids = rng.permutation(self.pages)
        self.table_host = np.where(rng.random((len(lens), self.width)) < 0.5, -7, 10 ** 9).astype(np.int64)
        at = 0
        for s, m in enumerate(need):
            self.table_host[s, :m] = ids[at:at + m]
            at += m
        shape = (self.pages, heads, page, dim)
        held = np.zeros((self.pages, page), bool)
        for s, n in enumerate(lens):
            for p in range(n):
                held[self.table_host[s, p // page], p % page] = True
        self.held = held
        where = held[:, None, :, None]
        data, self.value, self.scale_host = [], [], []
        for i in range(2):
            if bits == 16:
                x = torch.tensor(rng.standard_normal(shape) if kv is None else kv(rng, shape, i), dtype=torch.float32)
                x = x.to(torch.bfloat16)
                self.value.append(x.double().numpy())
                data.append(torch.where(torch.tensor(where), x, torch.tensor(float("nan"), dtype=torch.bfloat16)))
                self.scale_host.append(None)
            else:
                c = rng.integers(-127, 128, shape).astype(np.int8)
                sc = (0.005 + 0.02 * rng.random(shape[:3])).astype(np.float32)
                self.value.append(c.astype(np.float64) * sc.astype(np.float64)[..., None])
                data.append(torch.tensor(c))
                self.scale_host.append(torch.tensor(np.where(held[:, None, :], sc, np.float32("nan"))))
        t = data[0].dtype
        if layout == "heads":                     # [page, head, slot, dim]
            place = [torch.empty(shape, dtype=t, device="cuda") for _ in range(2)]
        elif layout == "slots":                   # [page, slot, head, dim]
            place = [torch.empty(self.pages, page, heads, dim, dtype=t, device="cuda").transpose(1, 2) for _ in range(2)]
        elif layout == "both":                    # keys and values of a page side by side
            one = torch.empty(self.pages, 2, heads, page, dim, dtype=t, device="cuda")
            place = [one[:, 0], one[:, 1]]
        else:                                     # rows apart, heads outermost
            one = torch.full((2, heads, self.pages, page, dim + 32), 7, dtype=t, device="cuda")
            place = [one[i, :, :, :, 16:16 + dim].transpose(0, 1) for i in range(2)]
        for d, x in zip(place, data):
            d.copy_(x)
        self.k, self.v = place
        self.ks, self.vs = (None if x is None else x.cuda().contiguous() for x in self.scale_host)
        self.c = sa.KvCache(self.k, self.v, self.ks, self.vs)
        self.table = torch.tensor(self.table_host, dtype=torch.int32, device="cuda")

    def rows(self, i, s, upto):
        """Positions 0 .. upto of sequence s as [upto, heads, dim] in 64 bits."""
        p = np.arange(upto)
        return self.value[i][self.table_host[s, p // self.page], :, p % self.page]


def ints(a):
    import torch

    return torch.tensor(np.asarray(a), dtype=torch.int32, device="cuda")


def attention(k, v, q, scale):
    """(out, what an output may be off by) of q [heads, dim] over k, v
    [positions, kv heads, dim], in 64 bits.

    A score is a sum of products that are exact in f32: 32 of them in a matrix
    instruction and up to 3 dim / 32 instructions one after another, so it is
    off by (32 + 3 dim / 32) u of the sum of magnitudes, and by 4 u of itself for
    the factors behind it; the difference to the maximum rounds by u of it, the
    power of two by 2 u. A weight's relative error is that of its score and of
    its maximum's. The output's sums round like the scores': 32 terms, three
    parts of a tile one after another, tiles of 128 positions (a wave has one of
    four), a few joins; the weights' own sum 8 terms a tile."""
    n, hk, d = k.shape
    h = q.shape[0]
    g = h // hk
    kk, vv = np.repeat(k, g, 1), np.repeat(v, g, 1)
    s = scale * np.einsum("phd,hd->ph", kk, q)
    mag = abs(scale) * np.einsum("phd,hd->ph", np.abs(kk), np.abs(q))
    m = s.max(0)
    w = np.exp(s - m)
    total = w.sum(0)
    out = np.einsum("ph,phd->hd", w, vv) / total[:, None]
    tiles = n // 128 + 2
    score = (32 + 3 * d / 32) * U * mag + 4 * U * np.abs(s)
    rel = score + score[s.argmax(0), np.arange(h)] + U * 1.5 * np.abs(s - m) + 4 * U
    rel += (32 + 3 * tiles + 24 + 8 * tiles + 24) * U
    room = np.einsum("ph,phd->hd", w * rel, np.abs(vv)) / total[:, None] + np.abs(out) * ((w * rel).sum(0) / total)[:, None]
    return out, room + 1e-37
