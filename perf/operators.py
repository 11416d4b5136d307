"""Serving operators around the MoE block and the LM head: their calls at the
sizes a batch of requests meets them, and their plain forms.

One decode or prompt step of many requests runs: the residual's addition with
the RMSNorm in front of a block (`rmsnorm`, with an 8-bit copy of the rows), a
quantized projection or the LM head over the 8-bit rows (`qmm_i8`), the
requests' own low-rank adapters beside it (`lora`), and, where several
continuations are kept, the selection over beams and vocabulary (`beam_select`)
and the reordering of the beams' states (`beam_reorder`).

`own = False`: elementary torch operations. `own = True`: the library's calls.
Inputs have the distributions the layers see: codes uniform, scales
bf16 |N(0, .02)|, biases bf16 N(0, .01), hidden rows N(0, 1), adapter weights
bf16 N(0, .02), logits N(0, 2.5).
"""
import math

import torch

own = False

DEV = "cuda:0"
EPS = 1e-6


def listed():
    return [
        # One decoded token in front of a block: the smallest call, all latency.
        dict(name="norm_token", op="norm", n=1, hidden=2048, x="f32", out="f32", q=None),
        # A prompt chunk in front of a block: rows for the router and the
        # experts, and the same rows in 8 bits for the dense projections.
        dict(name="norm_prompt_i8", op="norm", n=1000, hidden=4096, x="bf16", out="bf16", q=64),
        # A projection of a few requests' tokens: one round trip to memory.
        dict(name="qmm_i8_few", op="qmm", n=4, out_dim=4096, in_dim=2048, bits=4, group=64, x_group=0),
        # The LM head of a batch of beams.
        dict(name="qmm_i8_vocab", op="qmm", n=16, out_dim=151936, in_dim=2048, bits=4, group=64, x_group=0),
        # A prompt chunk with a ragged tail through a wide projection, the
        # rows' scales per group.
        dict(name="qmm_i8_prompt", op="qmm", n=1000, out_dim=7168, in_dim=4096, bits=4, group=64, x_group=64),
        # Decode of a few requests, each with its adapter.
        dict(name="lora_few", op="lora", n=8, in_dim=2048, out_dim=2048, adapters=4, rank=16, without=0,
             segments=False, mixed=False, x="f32"),
        # Decode of a large batch over many adapters of mixed ranks, one row
        # in four without any.
        dict(name="lora_batch", op="lora", n=200, in_dim=4096, out_dim=4096, adapters=40, rank=64, without=50,
             segments=False, mixed=True, x="f32"),
        # Prompts of three requests, packed one after the other.
        dict(name="lora_prompts", op="lora", n=1000, in_dim=2048, out_dim=4096, adapters=3, rank=32, without=0,
             segments=True, mixed=False, x="bf16"),
        # One request's four beams.
        dict(name="beam_one", op="beam", requests=1, beams=4, picks=8, vocab=151936, masked=0.0, done=False),
        # Sixteen requests' beams, some of them ended, with forbidden tokens.
        dict(name="beam_many", op="beam", requests=16, beams=4, picks=8, vocab=151936, masked=0.05, done=True),
        # One request's beams: recurrent states of some layers.
        dict(name="reorder_one", op="reorder", requests=1, beams=4, states=8, pieces=1, used=65536, room=65536),
        # Sixteen requests' beams: caches of several heads, used in part.
        dict(name="reorder_many", op="reorder", requests=16, beams=4, states=40, pieces=4, used=150016, room=262144),
    ]


def _log_int(rng, lo, hi):
    return max(lo, min(hi, round(math.exp(rng.uniform(math.log(lo), math.log(hi + 1))))))


def draw(rng):
    op = rng.choice(["norm", "norm", "qmm", "qmm", "qmm", "lora", "lora", "lora", "beam", "beam", "reorder"])
    if op == "norm":
        q = rng.choice([None, 0, 32, 64, 128])
        hidden = rng.choice([512, 2048, 2560, 4096, 7168, _log_int(rng, 64, 8192)])
        if q:
            hidden = max(q, hidden // q * q)
        n = _log_int(rng, 1, min(1024, (1 << 22) // hidden))
        return dict(op=op, n=n, hidden=hidden, x=rng.choice(["f32", "bf16"]), out=rng.choice(["f32", "bf16"]), q=q)
    if op == "qmm":
        group = rng.choice([32, 64, 64, 128])
        out_dim, in_dim = rng.choice([(512, 2048), (2048, 512), (4096, 2048), (640, 2560), (2560, 640), (1024, 4096),
                                      (4096, 1024), (2048, 7168), (7168, 2048), (_log_int(rng, 500, 151936), 2048),
                                      (_log_int(rng, 100, 8192), group * _log_int(rng, 1, 4096 // group))])
        most = 64 if out_dim > 16384 else 1000
        return dict(op=op, n=_log_int(rng, 1, most), out_dim=out_dim, in_dim=in_dim, bits=rng.choice([3, 4, 4, 8]),
                    group=group, x_group=rng.choice([0, group]))
    if op == "lora":
        n = _log_int(rng, 1, 1000)
        return dict(op=op, n=n, in_dim=rng.choice([512, 2048, 2560, 4096, 8 * _log_int(rng, 8, 512)]),
                    out_dim=rng.choice([512, 2048, 640, 4096, _log_int(rng, 64, 4096)]),
                    adapters=_log_int(rng, 1, 64), rank=8 * _log_int(rng, 1, 8), without=rng.choice([0, n // 4, n // 2]),
                    segments=rng.random() < 0.4, mixed=rng.random() < 0.5, x=rng.choice(["f32", "bf16"]))
    if op == "beam":
        beams = rng.randint(1, 8)
        vocab = _log_int(rng, 500, 151936)
        most = min(64, (64 * 151936) // (beams * vocab))
        return dict(op=op, requests=_log_int(rng, 1, max(1, most)), beams=beams, picks=rng.randint(beams, 2 * beams),
                    vocab=vocab, masked=rng.choice([0.0, 0.05, 0.5]), done=rng.random() < 0.5)
    room = _log_int(rng, 1024, 262144) // 16 * 16
    used = max(16, round(room * rng.uniform(0.1, 1.0)) // 2 * 2)
    return dict(op=op, requests=_log_int(rng, 1, 16), beams=rng.randint(1, 4), states=_log_int(rng, 1, 40),
                pieces=rng.choice([1, 2, 4]), used=used, room=room)


# -- inputs ------------------------------------------------------------------


def _gen(seed, salt):
    return torch.Generator(device=DEV).manual_seed((seed * 1000003 + salt) % (1 << 62))


def _normal(g, *shape, sigma=1.0):
    return torch.randn(*shape, generator=g, device=DEV, dtype=torch.float32) * sigma


def _norm_inputs(case, seed):
    g = _gen(seed, 1)
    n, H = case["n"], case["hidden"]
    x = _normal(g, n, H)
    if case["x"] == "bf16":
        x = x.to(torch.bfloat16)
    return dict(x=x, residual=_normal(g, n, H, sigma=3.0), w=(1.0 + 0.1 * _normal(g, H)).to(torch.bfloat16))


def _qmm_inputs(case, seed):
    g = _gen(seed, 2)
    n, O, K, bits, group = (case[k] for k in ("n", "out_dim", "in_dim", "bits", "group"))
    codes = O * K * bits // 8
    at = (codes + 15) // 16 * 16
    sb = O * (K // group) * 2
    at_b = at + (sb + 15) // 16 * 16
    buf = torch.zeros(at_b + sb, dtype=torch.uint8, device=DEV)
    buf[:codes] = torch.randint(0, 256, (codes,), generator=g, device=DEV, dtype=torch.uint8)
    buf[at:at + sb] = _normal(g, sb // 2, sigma=0.02).abs_().to(torch.bfloat16).view(torch.uint8)
    buf[at_b:] = _normal(g, sb // 2, sigma=0.01).to(torch.bfloat16).view(torch.uint8)
    xg = case["x_group"] or K
    rows = _normal(g, n, K // xg, xg)
    sx = rows.abs().amax(2, keepdim=True) / 127
    c8 = torch.round(rows / sx).clamp_(-127, 127).to(torch.int8).view(n, K)
    return dict(buf=buf, at=(0, at, at_b), c8=c8, sx=sx.reshape(n, K // xg).contiguous())


def _ranks(case):
    r = case["rank"]
    return [r if not case["mixed"] or a % 2 == 0 else max(1, r * 3 // 4 - 1) for a in range(case["adapters"])]


def _lora_counts(case):
    """Rows with an adapter, and how many of them each adapter in use has."""
    rows = case["n"] - min(case["without"], case["n"] - 1)
    used = min(case["adapters"], rows)
    return rows, [rows // used + (1 if i < rows % used else 0) for i in range(used)]


def _lora_inputs(case, seed):
    g = _gen(seed, 3)
    n, K, O, N, r = (case[k] for k in ("n", "in_dim", "out_dim", "adapters", "rank"))
    rows, counts = _lora_counts(case)
    order = torch.randperm(N, generator=g, device=DEV)
    ids = torch.full((n,), -1, dtype=torch.int32, device=DEV)
    ids[:rows] = torch.repeat_interleave(order[:len(counts)], torch.tensor(counts, device=DEV)).to(torch.int32)
    if not case["segments"]:
        ids = ids[torch.randperm(n, generator=g, device=DEV)].contiguous()
    x = _normal(g, n, K)
    if case["x"] == "bf16":
        x = x.to(torch.bfloat16)
    return dict(x=x, base=_normal(g, n, O), ids=ids, a=_normal(g, N, r, K, sigma=0.02).to(torch.bfloat16),
                b=_normal(g, N, O, r, sigma=0.02).to(torch.bfloat16), scale=0.5 + _normal(g, N).abs_(),
                ranks=torch.tensor(_ranks(case), dtype=torch.int32, device=DEV))


def _beam_inputs(case, seed):
    g = _gen(seed, 4)
    R, W, V = case["requests"], case["beams"], case["vocab"]
    logits = _normal(g, R * W, V, sigma=2.5)
    if case["masked"]:
        logits[torch.rand(R * W, V, generator=g, device=DEV) < case["masked"]] = -math.inf
    scores = -10.0 * torch.rand(R, W, generator=g, device=DEV)
    done = (torch.rand(R, W, generator=g, device=DEV) < 0.2).to(torch.uint8) if case["done"] else None
    return dict(logits=logits, scores=scores, done=done, pad=min(2, V - 1))


def _reorder_inputs(case, seed):
    g = _gen(seed, 5)
    R, W, S = case["requests"], case["beams"], case["states"]
    keep = (W + 1) // 2  # beams of a request that go on
    pick = torch.rand(R, W, generator=g, device=DEV).argsort(1)[:, :keep]
    slot = torch.arange(W, device=DEV) % keep
    rows = (pick[:, slot] + W * torch.arange(R, device=DEV)[:, None]).to(torch.int32).reshape(-1)
    src = [torch.randint(0, 1 << 15, (R * W, case["pieces"], case["room"] // 2), generator=g, device=DEV,
                         dtype=torch.int16) for _ in range(S)]
    return dict(rows=rows.contiguous(), src=src)


def prepare(case, seed):
    op = case["op"]
    s = dict(case=case)
    if op == "norm":
        s.update(_norm_inputs(case, seed))
    elif op == "qmm":
        s.update(_qmm_inputs(case, seed))
    elif op == "lora":
        s.update(_lora_inputs(case, seed))
    elif op == "beam":
        s.update(_beam_inputs(case, seed))
    else:
        s.update(_reorder_inputs(case, seed))
        # The other of the two buffers that an engine swaps between steps.
        s["dst"] = [torch.zeros_like(t) for t in s["src"]]
    if own:
        _prepare_own(s)
    return s


# -- plain forms -------------------------------------------------------------


def _plain_norm(s):
    case = s["case"]
    n, H, q = case["n"], case["hidden"], case["q"]
    r = s["x"].float() + s["residual"]
    y = r * torch.rsqrt((r * r).mean(1, keepdim=True) + EPS) * s["w"].float()
    out = [r, y.to(torch.bfloat16) if case["out"] == "bf16" else y]
    if q is not None:
        v = y.view(n, H // (q or H), q or H)
        sc = v.abs().amax(2, keepdim=True) / 127
        codes = torch.round(v / sc).clamp(-127, 127)
        # 8-bit values, as what they stand for, in a type of 8 bits' precision.
        out += [(codes * sc).view(n, H).to(torch.bfloat16), sc.view(n, -1)]
    return out


def _codes(buf, rows, cols, bits):
    """Codes of a packed matrix as [rows, cols] uint8."""
    b = buf[:rows * cols * bits // 8]
    if bits == 8:
        return b.view(rows, cols)
    if bits == 4:
        return torch.stack([b & 15, b >> 4], 1).view(rows, cols)
    p = b.view(-1, 3).int()
    p = p[:, 0] | (p[:, 1] << 8) | (p[:, 2] << 16)
    return torch.stack([((p >> (3 * i)) & 7).to(torch.uint8) for i in range(8)], 1).view(rows, cols)


def _plain_qmm(s):
    case = s["case"]
    n, O, K, bits, group = (case[k] for k in ("n", "out_dim", "in_dim", "bits", "group"))
    gs = O * (K // group) * 2
    sw = s["buf"][s["at"][1]:s["at"][1] + gs].view(torch.bfloat16).float().view(O, K // group, 1)
    bw = s["buf"][s["at"][2]:s["at"][2] + gs].view(torch.bfloat16).float().view(O, K // group, 1)
    w = (_codes(s["buf"], O, K, bits).float().view(O, K // group, group) * sw + bw).view(O, K)
    xg = case["x_group"] or K
    x = (s["c8"].float().view(n, K // xg, xg) * s["sx"][:, :, None]).view(n, K)
    return x @ w.t()


def _plain_lora(s):
    case = s["case"]
    y = s["base"].clone()
    x = s["x"].float()
    ids = s["ids"].long()
    for a, r in enumerate(_ranks(case)):
        at = (ids == a).nonzero()[:, 0]
        u = x[at] @ s["a"][a, :r].float().t()
        y[at] += s["scale"][a] * (u @ s["b"][a, :, :r].float().t())
    return y


def _plain_beam(s):
    case = s["case"]
    R, W, V, P = (case[k] for k in ("requests", "beams", "vocab", "picks"))
    l = s["logits"].double().view(R, W, V)  # candidates of several beams can lie close together
    m = l.amax(2, keepdim=True)
    lse = m + torch.log(torch.exp(l - m).sum(2, keepdim=True))
    sc = s["scores"].double()[:, :, None]
    cand = sc + (l - lse)
    if s["done"] is not None:
        ended = torch.full_like(cand, -math.inf)
        ended[:, :, s["pad"]] = sc[:, :, 0]
        cand = torch.where(s["done"].bool()[:, :, None], ended, cand)
    cand = torch.where(cand.isnan(), -math.inf, cand).view(R, W * V)
    v, i = torch.sort(cand, dim=1, descending=True, stable=True)
    v, i = v[:, :P], i[:, :P]
    rows = i // V + W * torch.arange(R, device=DEV)[:, None]
    return [v.float(), rows.to(torch.int32), (i % V).to(torch.int32)]


def _plain_reorder(s):
    at, used = s["rows"].long(), s["case"]["used"] // 2
    for src, dst in zip(s["src"], s["dst"]):
        dst[:, :, :used] = src[at, :, :used]
    return s["dst"]


# -- the library's calls -----------------------------------------------------


def _prepare_own(s):
    import streamoe_amd as sa

    case, op = s["case"], s["case"]["op"]
    k = s["k"] = sa.Kernels(0)
    if op == "qmm":
        s["qw"] = sa.QuantWeights(s["buf"], *s["at"], case["group"], case["bits"])
    elif op == "lora":
        s["set"] = sa.Adapters(s["a"], s["b"], s["scale"], s["ranks"] if case["mixed"] else None)
        s["ws"] = torch.empty(k.lora_workspace_size(s["set"], case["n"]), dtype=torch.uint8, device=DEV)
    elif op == "beam":
        s["ws"] = torch.empty(k.beam_select_workspace_size(case["requests"], case["beams"], case["vocab"], case["picks"]),
                              dtype=torch.uint8, device=DEV)
    elif op == "reorder":
        s["list"] = [sa.BeamState(a, b, case["used"]) for a, b in zip(s["src"], s["dst"])]


def _own_norm(s):
    from streamoe_amd import check

    case, k = s["case"], s["k"]
    n, H, q = case["n"], case["hidden"], case["q"]
    r = torch.empty(n, H, dtype=torch.float32, device=DEV)
    y = torch.empty(n, H, dtype=torch.bfloat16 if case["out"] == "bf16" else torch.float32, device=DEV)
    if q is None:
        check(k.rmsnorm(s["x"], s["residual"], s["w"], EPS, n, H, r, y), "rmsnorm")
        return [r, y]
    codes = torch.empty(n, H, dtype=torch.int8, device=DEV)
    sc = torch.empty(n, H // (q or H), dtype=torch.float32, device=DEV)
    check(k.rmsnorm(s["x"], s["residual"], s["w"], EPS, n, H, r, y, codes, sc, q), "rmsnorm")
    return [r, y, (codes.view(n, H // (q or H), q or H) * sc[:, :, None]).view(n, H).to(torch.bfloat16), sc]


def _own_qmm(s):
    from streamoe_amd import check

    case = s["case"]
    y = torch.empty(case["n"], case["out_dim"], dtype=torch.float32, device=DEV)
    check(s["k"].qmm_i8(s["qw"], s["c8"], s["sx"], case["x_group"], y, case["out_dim"], case["in_dim"], case["n"]),
          "qmm_i8")
    return y


def _own_lora(s):
    from streamoe_amd import check

    case = s["case"]
    y = torch.empty(case["n"], case["out_dim"], dtype=torch.float32, device=DEV)
    check(s["k"].lora(s["set"], s["ids"], s["x"], s["base"], y, case["out_dim"], case["in_dim"], case["n"], s["ws"]),
          "lora")
    return y


def _own_beam(s):
    from streamoe_amd import check

    case = s["case"]
    R, W, V, P = (case[k] for k in ("requests", "beams", "vocab", "picks"))
    v = torch.empty(R, P, dtype=torch.float32, device=DEV)
    rows = torch.empty(R, P, dtype=torch.int32, device=DEV)
    tokens = torch.empty(R, P, dtype=torch.int32, device=DEV)
    check(s["k"].beam_select(s["logits"], s["scores"], s["done"], s["pad"], R, W, V, P, v, rows, tokens, s["ws"]),
          "beam_select")
    return [v, rows, tokens]


def _own_reorder(s):
    from streamoe_amd import check

    check(s["k"].beam_reorder(s["list"], s["rows"]), "beam_reorder")
    return s["dst"]


def run(state):
    op = state["case"]["op"]
    if own:
        return {"norm": _own_norm, "qmm": _own_qmm, "lora": _own_lora, "beam": _own_beam, "reorder": _own_reorder}[op](state)
    return {"norm": _plain_norm, "qmm": _plain_qmm, "lora": _plain_lora, "beam": _plain_beam,
            "reorder": _plain_reorder}[op](state)


def work(case):
    op = case["op"]
    if op == "norm":
        n, H, q = case["n"], case["hidden"], case["q"]
        size = {"f32": 4, "bf16": 2}
        by = n * H * (size[case["x"]] + 4 + 4 + size[case["out"]]) + 2 * H
        if q is not None:
            by += n * H + n * (H // (q or H)) * 4
        return dict(bytes=by, flops=n * H * (6 if q is None else 9))
    if op == "qmm":
        n, O, K = case["n"], case["out_dim"], case["in_dim"]
        by = O * K * case["bits"] // 8 + 4 * O * (K // case["group"]) + n * K + 4 * n * (K // (case["x_group"] or K)) + 4 * n * O
        return dict(bytes=by, flops=2 * n * O * K)
    if op == "lora":
        n, K, O = case["n"], case["in_dim"], case["out_dim"]
        rows, counts = _lora_counts(case)
        r = sum(_ranks(case)) / case["adapters"]  # which adapters are used goes by the seed: the mean
        by = len(counts) * r * (K + O) * 2 + rows * K * (4 if case["x"] == "f32" else 2) + 8 * n * O + 4 * n
        return dict(bytes=int(by), flops=int(2 * rows * r * (K + O)) + n * O)
    if op == "beam":
        rows = case["requests"] * case["beams"]
        return dict(bytes=rows * case["vocab"] * 4 + case["requests"] * case["picks"] * 12 + rows * 4,
                    flops=4 * rows * case["vocab"])
    rows, W = case["requests"] * case["beams"], case["beams"]
    read = case["requests"] * ((W + 1) // 2)
    return dict(bytes=(rows + read) * case["states"] * case["pieces"] * case["used"], flops=0)


# -- the definitions in 64 bits ----------------------------------------------


def _exact_norm(case, seed):
    i = _norm_inputs(case, seed)
    r = i["residual"].to(torch.float64) + i["x"].to(torch.float64)
    H = case["hidden"]
    rms = ((r ** 2).sum(dim=-1) / H + EPS).sqrt()
    y = torch.einsum("th,h->th", r / rms[:, None], i["w"].to(torch.float64))
    if case["q"] is None:
        return [r, y]
    parts = y.split(case["q"] or H, dim=-1)
    tops = [p.abs().max(dim=-1, keepdim=True).values for p in parts]
    vals = [torch.round(p * 127.0 / t) * t / 127.0 for p, t in zip(parts, tops)]
    return [r, y, torch.cat(vals, -1), torch.cat(tops, -1) / 127.0]


def _exact_qmm(case, seed):
    i = _qmm_inputs(case, seed)
    n, O, K, bits, group = (case[k] for k in ("n", "out_dim", "in_dim", "bits", "group"))
    raw = i["buf"][:O * K * bits // 8].view(O, -1)
    shift = torch.arange(8, device=DEV)
    bit = ((raw[:, :, None] >> shift.to(torch.uint8)) & 1).view(O, K, bits) if O * K <= 1 << 26 else None
    if bit is not None:
        q = sum(bit[:, :, j].to(torch.float64) * 2.0 ** j for j in range(bits))
    elif bits == 8:
        q = raw.to(torch.float64)
    elif bits == 4:
        q = torch.empty(O, K, dtype=torch.float64, device=DEV)
        q[:, 0::2] = raw.remainder(16).to(torch.float64)
        q[:, 1::2] = raw.div(16, rounding_mode="floor").to(torch.float64)
    else:
        b = raw.view(O, K // 8, 3).to(torch.int64)
        word = b[:, :, 0] + 256 * b[:, :, 1] + 65536 * b[:, :, 2]
        q = torch.empty(O, K, dtype=torch.float64, device=DEV)
        for j in range(8):
            q[:, j::8] = (word.div(8 ** j, rounding_mode="floor") % 8).to(torch.float64)
    at_s, at_b = i["at"][1:]
    size = O * (K // group) * 2
    s = i["buf"][at_s:at_s + size].view(torch.bfloat16).to(torch.float64).view(O, -1)
    b = i["buf"][at_b:at_b + size].view(torch.bfloat16).to(torch.float64).view(O, -1)
    x = i["c8"].to(torch.float64) * i["sx"].to(torch.float64).repeat_interleave(case["x_group"] or K, dim=1)
    y = torch.zeros(n, O, dtype=torch.float64, device=DEV)
    for g in range(K // group):
        xs = x[:, g * group:(g + 1) * group]
        y += (xs @ q[:, g * group:(g + 1) * group].t()) * s[:, g] + xs.sum(1, keepdim=True) * b[:, g]
    return y


def _exact_lora(case, seed):
    i = _lora_inputs(case, seed)
    y = i["base"].to(torch.float64)
    ranks = _ranks(case)
    x = i["x"].to(torch.float64)
    for t, a in enumerate(i["ids"].tolist()):
        if a < 0:
            continue
        r = ranks[a]
        low = torch.mv(i["a"][a, :r].to(torch.float64), x[t])
        y[t] += torch.mv(i["b"][a, :, :r].to(torch.float64), low) * float(i["scale"][a])
    return y


def _exact_beam(case, seed):
    """Scores only: the picks are whole numbers."""
    i = _beam_inputs(case, seed)
    R, W, V, P = (case[k] for k in ("requests", "beams", "vocab", "picks"))
    best = []
    for q in range(R):
        vals = []
        for b in range(W):
            if i["done"] is not None and bool(i["done"][q, b]):
                vals.append(i["scores"][q, b].to(torch.float64)[None])
                continue
            l = i["logits"][q * W + b].to(torch.float64)
            vals.append((torch.log_softmax(l, 0) + i["scores"][q, b].to(torch.float64)).topk(min(P, V)).values)
        vals = torch.cat(vals + [torch.full((P,), -math.inf, dtype=torch.float64, device=DEV)])
        best.append(vals.topk(P).values)
    return [torch.stack(best), None, None]


def exact(case, seed):
    op = case["op"]
    if op == "reorder":
        return None
    return {"norm": _exact_norm, "qmm": _exact_qmm, "lora": _exact_lora, "beam": _exact_beam}[op](case, seed)
