"""Operators of a decode step over many requests' caches, and the draw of its
token: their calls at the sizes a serving process meets them, and their plain
forms.

New tokens' keys and values go into pages of a cache (`append`, in bf16 or in 8
bits with a scale per token and head), are read back as rows (`gather`), and
each new token's queries attend to its sequence's pages (`attn`); behind the LM
head the next token is drawn from the filtered distribution (`sample`).

A token is a pair (sequence, position): position p of sequence s lies in page
table[s, p // page], slot p % page; sequence -1 is a padding row.

`own = False`: elementary torch operations. `own = True`: the library's calls.
Keys, values and queries are N(0, 1), pages lie in a shuffled order, logits are
N(0, 2.5).
"""
import math

import torch

own = False

DEV = "cuda:0"


def listed():
    return [
        # One decoded token of one request: the smallest write, all latency.
        dict(name="append_token", op="append", seqs=1, lo=300, hi=300, take=1, pad=0, kv_heads=2, dim=256, bits=16, page=16,
             x="f32"),
        # Prompts of three requests, packed one after the other, into a cache of
        # 8 bits, and the values that it then holds.
        dict(name="append_prompt_i8", op="append", seqs=3, lo=150, hi=500, take=500, pad=7, kv_heads=2, dim=256, bits=8,
             page=16, x="bf16"),
        # The last positions of two requests, for another process to go on with.
        dict(name="gather_span", op="gather", seqs=2, lo=301, hi=999, take=50, kv_heads=2, dim=256, bits=16, page=16,
             out="f32"),
        # Long prefixes that a prompt chunk attends to, out of a cache of 8 bits.
        dict(name="gather_prefix_i8", op="gather", seqs=4, lo=1000, hi=7001, take=7001, kv_heads=8, dim=128, bits=8, page=64,
             out="bf16"),
        # One request in a short conversation: all latency.
        dict(name="attn_one", op="attn", seqs=1, lo=700, hi=700, take=1, pad=0, heads=16, kv_heads=2, dim=256, bits=16,
             page=16, window=0, x="f32"),
        # One request with a book in its context: the cache's length is all there
        # is to split.
        dict(name="attn_long", op="attn", seqs=1, lo=131001, hi=131001, take=1, pad=0, heads=16, kv_heads=2, dim=256, bits=16,
             page=64, window=0, x="bf16"),
        # A batch of requests of very different lengths, padded, 8-bit cache.
        dict(name="attn_batch_i8", op="attn", seqs=61, lo=200, hi=9001, take=1, pad=3, heads=16, kv_heads=2, dim=256, bits=8,
             page=64, window=0, x="bf16"),
        # A key and value head for every query head.
        dict(name="attn_heads", op="attn", seqs=48, lo=33, hi=2500, take=1, pad=0, heads=16, kv_heads=16, dim=128, bits=16,
             page=16, window=0, x="f32"),
        # Four tokens of each sequence at once, a layer with a sliding window.
        dict(name="attn_window", op="attn", seqs=8, lo=500, hi=20001, take=4, pad=0, heads=32, kv_heads=8, dim=128, bits=16,
             page=32, window=1000, x="bf16"),
        # One request's token: few candidates.
        dict(name="sample_one", op="sample", n=1, vocab=151936, temperature=0.7, top_k=20, top_p=0.8, min_p=0.0, masked=0.0),
        # A batch whose requests ask for all kinds of filters, some for none,
        # some for the largest logit.
        dict(name="sample_mixed", op="sample", n=64, vocab=151936, temperature=-1.0, top_k=-1, top_p=-1.0, min_p=-1.0,
             masked=0.05),
        # No top-k and a wide nucleus: thousands of candidates.
        dict(name="sample_wide", op="sample", n=16, vocab=50000, temperature=1.0, top_k=0, top_p=0.95, min_p=0.0, masked=0.0),
    ]


def _log_int(rng, lo, hi):
    return max(lo, min(hi, round(math.exp(rng.uniform(math.log(lo), math.log(hi + 1))))))


def draw(rng):
    op = rng.choice(["append", "gather", "attn", "attn", "attn", "sample", "sample"])
    if op == "sample":
        vocab = _log_int(rng, 2, 151936)
        n = _log_int(rng, 1, max(1, min(200, 9000000 // vocab)))
        if rng.random() < 0.4:
            t = k = p = m = -1
        else:
            t, k = rng.choice([0.3, 0.7, 1.0, 1.5]), rng.choice([0, 0, _log_int(rng, 1, 1000)])
            p, m = rng.choice([1.0, 0.95, 0.5]), rng.choice([0.0, 0.0, 0.05])
        return dict(op=op, n=n, vocab=vocab, temperature=float(t), top_k=k, top_p=float(p), min_p=float(m),
                    masked=rng.choice([0.0, 0.05, 0.5]))
    heads, kv_heads, dim = rng.choice([(16, 2, 256), (16, 16, 128), (32, 2, 256), (32, 8, 128), (8, 1, 64), (12, 4, 64),
                                       (40, 2, 128), (6, 3, 80), (20, 4, 96), (14, 2, 112), (9, 3, 160), (7, 7, 16)])
    c = dict(op=op, kv_heads=kv_heads, dim=dim, bits=rng.choice([16, 8]), page=rng.choice([16, 32, 64, 256, 48, 1024]))
    values = (1 << 24) if op != "attn" else (1 << 26)
    most = max(2, values // (kv_heads * dim))  # positions of the whole case
    seqs = _log_int(rng, 1, max(1, min(100, most // 300)))
    hi = _log_int(rng, 1, max(1, most // seqs))
    c.update(seqs=seqs, lo=_log_int(rng, 1, hi), hi=hi)
    if op == "gather":
        return dict(c, take=_log_int(rng, 1, hi), out=rng.choice(["f32", "bf16"]))
    c.update(pad=rng.choice([0, 1, 5]), x=rng.choice(["f32", "bf16"]))
    if op == "append":
        return dict(c, take=_log_int(rng, 1, hi))
    if hi * (seqs * 4) > most * 2:  # the plain form holds a copy of the cache for every row
        c["take"] = 1
    else:
        c["take"] = rng.choice([1, 1, 2, 4])
    return dict(c, heads=heads, window=rng.choice([0, 0, _log_int(rng, 1, 4000)]))


def _lengths(case):
    """Positions of every sequence: lo, hi and, between, spread over the logarithm."""
    lo, hi, n = case["lo"], case["hi"], case["seqs"]
    spread = [round(lo * (hi / lo) ** ((i * 0.6180339887) % 1.0)) for i in range(n)]
    return ([hi] + spread[1:-1] + [lo])[:n] if n > 1 else [hi]


def _tokens(case):
    """(sequence, position) of every row: the last `take` positions of each
    sequence in order, then padding rows."""
    out = [(s, p) for s, n in enumerate(_lengths(case)) for p in range(max(0, n - case["take"]), n)]
    return out + [(-1, 0)] * case.get("pad", 0)


# -- inputs ------------------------------------------------------------------


def _gen(seed, salt):
    return torch.Generator(device=DEV).manual_seed((seed * 1000003 + salt) % (1 << 62))


def _normal(g, *shape, sigma=1.0):
    return torch.randn(*shape, generator=g, device=DEV, dtype=torch.float32) * sigma


def _cache_inputs(case, seed):
    g = _gen(seed, 1)
    H, D, ps = case["kv_heads"], case["dim"], case["page"]
    lens = _lengths(case)
    width = max((n + ps - 1) // ps for n in lens)
    need = sum((n + ps - 1) // ps for n in lens)
    pages = need + 3
    order = torch.randperm(pages, generator=g, device=DEV).to(torch.int32)
    at, table = 0, torch.zeros(len(lens), width, dtype=torch.int32, device=DEV)
    for s, n in enumerate(lens):
        m = (n + ps - 1) // ps
        table[s, :m] = order[at:at + m]
        at += m
    tok = torch.tensor(_tokens(case), dtype=torch.int32, device=DEV)
    s = dict(table=table, seq=tok[:, 0].contiguous(), pos=tok[:, 1].contiguous())
    for name in ("kc", "vc"):
        if case["bits"] == 8:
            s[name] = torch.randint(-127, 128, (pages, H, ps, D), generator=g, device=DEV, dtype=torch.int8)
            s[name + "_scales"] = (0.02 + 0.02 * torch.rand(pages, H, ps, generator=g, device=DEV)).contiguous()
        else:
            s[name] = torch.randn(pages, H, ps, D, generator=g, device=DEV, dtype=torch.bfloat16)
            s[name + "_scales"] = None
    n = tok.shape[0]
    if case["op"] == "append":  # keys and values as the projections leave them, side by side
        kv = _normal(g, n, 2 * H * D).to(torch.bfloat16 if case["x"] == "bf16" else torch.float32)
        s.update(k=kv[:, :H * D].unflatten(1, (H, D)), v=kv[:, H * D:].unflatten(1, (H, D)))
    elif case["op"] == "attn":
        q = _normal(g, n, case["heads"], D)
        s["q"] = q.to(torch.bfloat16) if case["x"] == "bf16" else q
    return s


def _sample_inputs(case, seed):
    g = _gen(seed, 2)
    n, V = case["n"], case["vocab"]
    logits = _normal(g, n, V, sigma=2.5)
    if case["masked"]:
        logits[torch.rand(n, V, generator=g, device=DEV) < case["masked"]] = -math.inf
        logits[:, -1] = 0.5
    row = torch.arange(n, device=DEV)
    each = lambda v, kinds, t: (torch.full((n,), v, device=DEV, dtype=t) if v >= 0
                                else torch.tensor(kinds, device=DEV, dtype=t)[row % len(kinds)])
    return dict(logits=logits, u=torch.rand(n, generator=g, device=DEV),
                temperature=each(case["temperature"], [0.7, 1.0, 0.0, 1.3, 0.9], torch.float32),
                top_k=each(case["top_k"], [50, 0, 0, 1000, 20, 1, 0], torch.int32),
                top_p=each(case["top_p"], [0.9, 1.0, 0.95], torch.float32),
                min_p=each(case["min_p"], [0.0, 0.05, 0.0, 0.0], torch.float32))


def prepare(case, seed):
    s = dict(case=case)
    s.update(_sample_inputs(case, seed) if case["op"] == "sample" else _cache_inputs(case, seed))
    if own:
        _prepare_own(s)
    return s


# -- plain forms -------------------------------------------------------------


def _places(s):
    """Rows that are no padding, their page and slot."""
    ps = s["case"]["page"]
    rows = (s["seq"] >= 0).nonzero()[:, 0]
    seq, pos = s["seq"][rows].long(), s["pos"][rows].long()
    return rows, s["table"][seq, pos // ps].long(), pos % ps


def _read(s, name, page, slot):
    """Rows [.., heads, dim] of the cache in 32 bits."""
    x = s[name][page, :, slot].float()
    return x if s["case"]["bits"] == 16 else x * s[name + "_scales"][page, :, slot][..., None]


def _plain_append(s):
    rows, page, slot = _places(s)
    out = []
    for name, x in (("kc", s["k"]), ("vc", s["v"])):
        x = x[rows].float()
        if s["case"]["bits"] == 16:
            s[name][page, :, slot] = x.to(torch.bfloat16)
            out.append(s[name])
            continue
        scale = x.abs().amax(2) / 127
        s[name][page, :, slot] = torch.round(x / scale[..., None]).to(torch.int8)
        s[name + "_scales"][page, :, slot] = scale
        back = torch.zeros(s["k"].shape, dtype=torch.bfloat16, device=DEV)
        back[rows] = _read(s, name, page, slot).to(torch.bfloat16)
        out += [back, s[name + "_scales"]]
    return out


def _plain_gather(s):
    _, page, slot = _places(s)
    t = torch.bfloat16 if s["case"]["out"] == "bf16" else torch.float32
    return [_read(s, name, page, slot).to(t) for name in ("kc", "vc")]


def _plain_attn(s):
    case = s["case"]
    ps, H, D = case["page"], case["kv_heads"], case["dim"]
    n, L = s["seq"].shape[0], max(_lengths(case))
    t = torch.arange(L, device=DEV)
    page = s["table"][s["seq"].clamp(min=0).long()][:, t // ps].long()
    last = torch.where(s["seq"] < 0, -1, s["pos"])[:, None]
    seen = t <= last
    if case["window"]:
        seen &= t > last - case["window"]
    k, v = (_read(s, name, page, (t % ps).expand(n, L)).permute(0, 2, 1, 3) for name in ("kc", "vc"))
    q = s["q"].float().view(n, H, -1, D)
    sc = torch.matmul(q, k.transpose(2, 3).contiguous()) * D ** -0.5
    sc = torch.where(seen[:, None, None], sc, -math.inf)
    top = sc.amax(3, keepdim=True)
    e = torch.where(seen[:, None, None], torch.exp(sc - top), 0.0)
    total = e.sum(3, keepdim=True)
    out = torch.matmul(e, v.contiguous()) / torch.where(total == 0, 1.0, total)
    return out.view(n, -1, D).to(s["q"].dtype)


def _plain_sample(s):
    case = s["case"]
    n, V = case["n"], case["vocab"]
    l, order = torch.sort(s["logits"], dim=1, descending=True, stable=True)
    t = s["temperature"].double()[:, None]
    d = (l.double() - l[:, :1].double()) / torch.where(t == 0, 1.0, t)  # borders are told apart in 64 bits
    mass = torch.exp(d)
    rank = torch.arange(V, device=DEV)[None]
    k = s["top_k"][:, None].long()
    kept = (rank < torch.where(k <= 0, V, k)) & (l > -math.inf)
    mass = torch.where(kept, mass, 0.0)
    before = mass.cumsum(1) - mass
    p = s["top_p"].double()[:, None]
    kept &= (before < p * mass.sum(1, keepdim=True)) | (p >= 1) | (rank == 0)
    kept &= torch.exp(d) >= s["min_p"].double()[:, None]
    kept = torch.where(t == 0, rank == 0, kept)
    mass = torch.where(kept, mass, 0.0)
    by_token = torch.zeros(n, V, dtype=torch.float64, device=DEV).scatter_(1, order, mass)
    total = mass.sum(1, keepdim=True)
    run_ = by_token.cumsum(1)
    token = (run_ <= s["u"].double()[:, None] * total).sum(1).clamp(max=V - 1)
    prob = by_token.gather(1, token[:, None]) / total
    return [token.to(torch.int32), torch.log(prob[:, 0]).float()]


# -- the library's calls -----------------------------------------------------


def _prepare_own(s):
    import streamoe_amd as sa

    case = s["case"]
    k = s["kernels"] = sa.Kernels(0)
    if case["op"] == "sample":
        size = k.sample_workspace_size(case["n"], case["vocab"])
    else:
        s["cache"] = sa.KvCache(s["kc"], s["vc"], s["kc_scales"], s["vc_scales"])
        size = k.attn_decode_workspace_size(s["cache"], case["heads"], s["seq"].shape[0]) if case["op"] == "attn" else 0
    s["ws"] = torch.empty(size, dtype=torch.uint8, device=DEV)


def _own_append(s):
    from streamoe_amd import check

    k, n = s["kernels"], s["seq"].shape[0]
    check(k.kv_append(s["cache"], s["table"], s["seq"], s["pos"], s["k"], s["v"], n), "kv_append")
    if s["case"]["bits"] == 16:
        return [s["kc"], s["vc"]]
    kb, vb = (torch.empty(s["k"].shape, dtype=torch.bfloat16, device=DEV) for _ in range(2))
    check(k.kv_gather(s["cache"], s["table"], s["seq"], s["pos"], kb, vb, n), "kv_gather")
    return [kb, s["kc_scales"], vb, s["vc_scales"]]


def _own_gather(s):
    from streamoe_amd import check

    case, n = s["case"], s["seq"].shape[0]
    t = torch.bfloat16 if case["out"] == "bf16" else torch.float32
    kb, vb = (torch.empty(n, case["kv_heads"], case["dim"], dtype=t, device=DEV) for _ in range(2))
    check(s["kernels"].kv_gather(s["cache"], s["table"], s["seq"], s["pos"], kb, vb, n), "kv_gather")
    return [kb, vb]


def _own_attn(s):
    from streamoe_amd import check

    case = s["case"]
    out = torch.empty_like(s["q"])
    check(s["kernels"].attn_decode(s["cache"], s["table"], s["seq"], s["pos"], s["q"], case["dim"] ** -0.5, case["window"],
                                   out, case["heads"], s["seq"].shape[0], s["ws"]), "attn_decode")
    return out


def _own_sample(s):
    from streamoe_amd import check

    case = s["case"]
    token = torch.empty(case["n"], dtype=torch.int32, device=DEV)
    logprob = torch.empty(case["n"], dtype=torch.float32, device=DEV)
    check(s["kernels"].sample(s["logits"], s["temperature"], s["top_k"], s["top_p"], s["min_p"], s["u"], case["n"],
                              case["vocab"], token, logprob, s["ws"]), "sample")
    return [token, logprob]


def run(state):
    op = state["case"]["op"]
    if own:
        return {"append": _own_append, "gather": _own_gather, "attn": _own_attn, "sample": _own_sample}[op](state)
    return {"append": _plain_append, "gather": _plain_gather, "attn": _plain_attn, "sample": _plain_sample}[op](state)


def work(case):
    if case["op"] == "sample":
        n, V = case["n"], case["vocab"]
        return dict(bytes=n * V * 4 + n * 28, flops=6 * n * V)
    H, D = case["kv_heads"], case["dim"]
    tok = _tokens(case)
    rows = sum(s >= 0 for s, _ in tok)
    held = 2 * H * (D * 2 if case["bits"] == 16 else D + 4)  # a position's bytes in the cache
    if case["op"] == "append":
        size = 4 if case["x"] == "f32" else 2
        by = rows * (2 * H * D * size + held) + 8 * len(tok)
        if case["bits"] == 8:
            by += rows * held + len(tok) * 2 * H * D * 2
        return dict(bytes=by, flops=rows * 2 * H * D * (1 if case["bits"] == 16 else 6))
    if case["op"] == "gather":
        return dict(bytes=rows * (held + 2 * H * D * (4 if case["out"] == "f32" else 2)) + 8 * len(tok), flops=rows * 2 * H * D)
    w = case["window"]
    seen = sum(min(p + 1, w) if w else p + 1 for s, p in tok if s >= 0)
    # Positions that several tokens of a sequence see are read once.
    read = sum(n - (max(0, max(0, n - case["take"]) + 1 - w) if w else 0) for n in _lengths(case))
    size = 4 if case["x"] == "f32" else 2
    return dict(bytes=read * held + 2 * len(tok) * case["heads"] * D * size + 8 * len(tok), flops=4 * seen * case["heads"] * D)


# -- the definitions in 64 bits ----------------------------------------------


def _sequence(i, name, s, n, page):
    """Positions 0..n of a sequence as [heads, n, dim], page after page."""
    ids = i["table"][s, :(n + page - 1) // page].long()
    x = i[name].index_select(0, ids).to(torch.float64)
    if i[name + "_scales"] is not None:
        x = x * i[name + "_scales"].index_select(0, ids).to(torch.float64).unsqueeze(3)
    return x.transpose(0, 1).flatten(1, 2)[:, :n]


def _exact_append(case, seed):
    i = _cache_inputs(case, seed)
    ps, tok = case["page"], i["seq"].tolist()
    table, pos = i["table"].tolist(), i["pos"].tolist()
    at = [(r, table[q][p // ps], p % ps) for r, (q, p) in enumerate(zip(tok, pos)) if q >= 0]
    r, page, slot = (torch.tensor(c, device=DEV) for c in zip(*at))
    out = []
    for name, x in (("kc", i["k"]), ("vc", i["v"])):
        x = x.to(torch.float64).index_select(0, r)
        if case["bits"] == 16:
            c = i[name].to(torch.float64).transpose(1, 2).contiguous()
            c.view(-1, *x.shape[1:]).index_copy_(0, page * ps + slot, x)
            out.append(c.transpose(1, 2))
            continue
        top = torch.linalg.vector_norm(x, ord=math.inf, dim=2, keepdim=True)
        back = torch.zeros(i["k"].shape, dtype=torch.float64, device=DEV)
        back.index_copy_(0, r, torch.round(x * (127.0 / top)) * top / 127.0)
        sc = i[name + "_scales"].to(torch.float64).transpose(1, 2).contiguous()
        sc.view(-1, x.shape[1]).index_copy_(0, page * ps + slot, top[:, :, 0] / 127.0)
        out += [back, sc.transpose(1, 2)]
    return out


def _exact_gather(case, seed):
    i = _cache_inputs(case, seed)
    out = []
    for name in ("kc", "vc"):
        rows = [_sequence(i, name, s, n, case["page"])[:, -case["take"]:].transpose(0, 1)
                for s, n in enumerate(_lengths(case))]
        out.append(torch.cat(rows))
    return out


def _exact_attn(case, seed):
    i = _cache_inputs(case, seed)
    D, w, lens = case["dim"], case["window"], _lengths(case)
    out = torch.zeros(i["q"].shape, dtype=torch.float64, device=DEV)
    held = (None, None, None)
    for r, (s, p) in enumerate(zip(i["seq"].tolist(), i["pos"].tolist())):
        if s < 0:
            continue
        if held[0] != s:
            held = (s, *(_sequence(i, name, s, lens[s], case["page"]) for name in ("kc", "vc")))
        lo = max(0, p + 1 - w) if w else 0
        k, v = held[1][:, lo:p + 1], held[2][:, lo:p + 1]
        q = i["q"][r].to(torch.float64).view(case["kv_heads"], -1, D)
        sc = torch.bmm(k, q.transpose(1, 2).contiguous()) / math.sqrt(D)
        weight = torch.softmax(sc, dim=1).transpose(1, 2).contiguous()
        out[r] = torch.bmm(weight, v.contiguous()).reshape(case["heads"], D)
    return out


def _exact_sample(case, seed):
    """Log-probabilities only: tokens are whole numbers."""
    i = _sample_inputs(case, seed)
    out = torch.zeros(case["n"], dtype=torch.float64, device=DEV)
    for r in range(case["n"]):
        t, k, p, m, u = (i[name][r].item() for name in ("temperature", "top_k", "top_p", "min_p", "u"))
        if t == 0:
            continue
        l = i["logits"][r].to(torch.float64)
        tokens = torch.argsort(l, descending=True, stable=True)
        tokens = tokens[: k if k > 0 else len(tokens)]
        tokens = tokens[l[tokens] > -math.inf]
        prob = torch.softmax(l[tokens] / t, dim=0)
        keep = len(prob)
        if p < 1:
            keep = min(keep, max(1, int((prob.cumsum(0) < p).sum()) + 1))
        keep = min(keep, int((prob >= m * prob[0]).sum()))
        tokens = tokens[:keep].sort().values
        prob = torch.softmax(l[tokens] / t, dim=0)
        at = int(torch.searchsorted(prob.cumsum(0), torch.tensor([u], dtype=torch.float64, device=DEV), right=True))
        out[r] = prob[min(at, keep - 1)].log()
    return [None, out]


def exact(case, seed):
    return {"append": _exact_append, "gather": _exact_gather, "attn": _exact_attn, "sample": _exact_sample}[case["op"]](case, seed)
