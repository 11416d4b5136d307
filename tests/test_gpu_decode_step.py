"""The cache, the attention and the sampling together, as a decode step of
several requests runs them behind the operators that were there: norm with an
8-bit copy, the fused projection on it, the new keys and values into the pages,
the attention over them, the LM head, one token each. Checked against 64-bit
arithmetic on what each step was given, over several tokens, on a stream of its
own, captured and replayed, and on two handles at once."""
import numpy as np
import pytest

from kv_cases import U, attention, ints
from test_gpu_qmm_i8 import _weights
from test_gpu_sample import want_of

pytestmark = pytest.mark.gpu

H, HQ, HK, D, PAGE, V, G = 512, 8, 2, 64, 16, 5003, 64
WIDTH = (HQ + 2 * HK) * D
START = [1, 16, 45, 130, 0]  # positions held at first; one sequence begins


class Step:
    """A batch of requests and its calls on a handle. Row 3 is padding."""

    def __init__(self, kernels, seed, bits):
        import torch

        import streamoe_amd as sa

        self.k, self.bits = kernels, bits
        g = torch.Generator(device="cuda").manual_seed(seed)
        rn = lambda *s: torch.randn(*s, generator=g, device="cuda")
        e = lambda *s, t=torch.float32: torch.empty(*s, dtype=t, device="cuda")
        self.rows = 1 + len(START)
        self.seq = ints([0, 1, 2, -1, 3, 4])
        self.pos = ints([START[0], START[1], START[2], 0, START[3], START[4]])
        self.one = ints([1] * 3 + [0] + [1] * 2)
        self.w = (1 + 0.1 * rn(H)).to(torch.bfloat16)
        rng = np.random.default_rng(seed)
        self.wqkv, self.head = _weights(rng, WIDTH, H, 4, G), _weights(rng, V, HQ * D, 4, G)
        self.qqkv = sa.QuantWeights(self.wqkv[0], *self.wqkv[1], G, 4)
        self.qhead = sa.QuantWeights(self.head[0], *self.head[1], G, 4)
        width = 12
        pages = width * len(START) + 3
        self.table = torch.randperm(pages, generator=g, device="cuda")[:width * len(START)].to(torch.int32).view(-1, width)
        shape = (pages, PAGE, HK, D)  # heads behind slots
        if bits == 16:
            self.kc, self.vc = (rn(*shape).to(torch.bfloat16).transpose(1, 2) for _ in range(2))
            self.ks = self.vs = None
        else:
            self.kc, self.vc = (torch.randint(-127, 128, shape, generator=g, device="cuda", dtype=torch.int8).transpose(1, 2)
                                for _ in range(2))
            self.ks, self.vs = (0.01 + 0.01 * torch.rand(pages, HK, PAGE, generator=g, device="cuda") for _ in range(2))
        self.cache = sa.KvCache(self.kc, self.vc, self.ks, self.vs)
        n = self.rows
        self.x, self.norm = rn(n, H), e(n, H)
        self.codes, self.sc = e(n, H, t=torch.int8), e(n, H // G)
        self.qkv = e(n, WIDTH)
        self.q = self.qkv[:, :HQ * D].unflatten(1, (HQ, D))
        self.knew = self.qkv[:, HQ * D:(HQ + HK) * D].unflatten(1, (HK, D))
        self.vnew = self.qkv[:, (HQ + HK) * D:].unflatten(1, (HK, D))
        self.attn = e(n, HQ, D)
        self.acodes, self.asc = e(n, HQ * D, t=torch.int8), e(n, HQ * D // G)
        self.logits = e(n, V)
        self.u = torch.rand(n, generator=g, device="cuda")
        self.t = torch.tensor([1.0, 0.7, 0.0, 1.0, 1.3, 1.0], device="cuda")
        self.topk, self.topp = ints([0, 50, 0, 1, 0, 600]), torch.tensor([0.9, 1.0, 1.0, 1.0, 0.95, 0.8], device="cuda")
        self.minp = torch.tensor([0.0, 0.0, 0.0, 0.0, 0.01, 0.0], device="cuda")
        self.tok, self.lp = e(n, t=torch.int32), e(n)
        self.aws = e(kernels.attn_decode_workspace_size(self.cache, HQ, n), t=torch.uint8)
        self.sws = e(kernels.sample_workspace_size(n, V), t=torch.uint8)
        torch.cuda.synchronize()

    def run(self):
        k, n = self.k, self.rows
        for status in (
                k.rmsnorm(self.x, None, self.w, 1e-6, n, H, None, self.norm, self.codes, self.sc, G),
                k.qmm_i8(self.qqkv, self.codes, self.sc, G, self.qkv, WIDTH, H, n),
                k.kv_append(self.cache, self.table, self.seq, self.pos, self.knew, self.vnew, n),
                k.attn_decode(self.cache, self.table, self.seq, self.pos, self.q, D ** -0.5, 0, self.attn, HQ, n, self.aws),
                k.rmsnorm(self.attn.view(n, -1), None, None, 1e-6, n, HQ * D, None, None, self.acodes, self.asc, G),
                k.qmm_i8(self.qhead, self.acodes, self.asc, G, self.logits, V, HQ * D, n),
                k.sample(self.logits, self.t, self.topk, self.topp, self.minp, self.u, n, V, self.tok, self.lp, self.sws)):
            assert status == 0, status

    def outputs(self):
        return [t.clone() for t in (self.qkv, self.attn, self.logits, self.tok, self.lp, self.kc, self.vc)]

    def held(self, seq, upto):
        """Keys and values of a sequence's positions 0 .. upto in 64 bits."""
        import torch

        p = torch.arange(upto, device="cuda")
        page, slot = self.table[seq, p // PAGE].long(), p % PAGE
        out = []
        for c, sc in ((self.kc, self.ks), (self.vc, self.vs)):
            x = c[page, :, slot].double()
            out.append((x if sc is None else x * sc[page, :, slot].double()[..., None]).cpu().numpy())
        return out

    def check(self, before):
        """`before`: held() of every sequence before the step."""
        f = lambda t: t.double().cpu().numpy()
        seq, pos = self.seq.tolist(), self.pos.tolist()
        assert np.all(f(self.attn[3]) == 0)
        for r, (s, p) in enumerate(zip(seq, pos)):
            if s < 0:
                continue
            k, v = self.held(s, p + 1)
            for now, old, new in ((k, before[s][0], f(self.knew[r])), (v, before[s][1], f(self.vnew[r]))):
                assert np.array_equal(now[:p], old[:p])  # nothing else changed
                step = np.abs(new).max(1, keepdims=True) / 127 if self.bits == 8 else np.abs(new) * 2 ** -7
                assert np.all(np.abs(now[p] - new) <= step * (0.5 + 1e-6))
            want, room = attention(k, v, f(self.q[r]), D ** -0.5)
            assert np.all(np.abs(f(self.attn[r]) - want) <= room)
        logits = f(self.logits)
        for r in range(self.rows):
            a, b, near = want_of(logits[r], *(x[r].item() for x in (self.t, self.topk, self.topp, self.minp, self.u)))
            assert near > 1e-9 and int(self.tok[r]) == a
            assert abs(float(self.lp[r]) - b) <= U * abs(b) + 2.0 ** -25

    def all_held(self):
        return [self.held(s, int(p)) for s, p in zip(range(len(START)), [x for s, x in zip(self.seq.tolist(), self.pos.tolist()) if s >= 0])]


@pytest.mark.parametrize("bits", [16, 8])
def test_tokens_one_after_another(kernels, bits):
    step = Step(kernels, bits, bits)
    for _ in range(20):  # past several pages' ends
        before = step.all_held()
        step.run()
        kernels.sync()
        step.check(before)
        step.pos += step.one
        step.x.normal_()
        step.u.uniform_(0, 0.999)


def test_on_another_stream(kernels):
    import torch

    step = Step(kernels, 3, 8)
    own, side = torch.cuda.current_stream(), torch.cuda.Stream()
    try:
        kernels.set_stream(side)
        before = step.all_held()
        step.run()
        kernels.sync()  # waits for the handle's stream
        step.check(before)
    finally:
        kernels.set_stream(own)


@pytest.mark.parametrize("bits", [16, 8])
def test_replayed_with_eager_work_between(kernels, bits):
    """One graph for every length: positions are read on the device."""
    import torch

    import streamoe_amd as sa

    step, other = Step(kernels, 4, bits), Step(kernels, 5, bits)
    graph = sa.capture_graph(kernels, step.run)
    for i in range(5):
        step.x.normal_()
        step.u.uniform_(0, 0.999)
        before, other_before = step.all_held(), other.all_held()
        graph.replay()
        other.run()  # eager work of another step, own workspaces
        torch.cuda.synchronize()
        got = step.outputs()
        step.check(before)
        other.check(other_before)
        step.run()
        kernels.sync()
        assert all(torch.equal(a, b) for a, b in zip(got, step.outputs()))
        step.pos += step.one * 7
        other.pos += other.one


def test_two_graphs_share_workspaces(kernels):
    """Captured steps of two batches with the same workspaces, replayed in turn."""
    import torch

    import streamoe_amd as sa

    a, b = Step(kernels, 8, 16), Step(kernels, 9, 8)
    b.aws, b.sws = a.aws, a.sws
    graphs = [sa.capture_graph(kernels, s.run) for s in (a, b)]
    for i in range(4):
        for s, graph in ((a, graphs[0]), (b, graphs[1])):
            s.x.normal_()
            s.u.uniform_(0, 0.999)
            before = s.all_held()
            graph.replay()
            if i % 2:
                a.aws.fill_(255)  # holds nothing between calls
                a.sws.fill_(255)
            torch.cuda.synchronize()
            s.check(before)
            s.pos += s.one


def test_two_handles_at_once(kernels):
    import torch

    import streamoe_amd as sa

    side = torch.cuda.Stream()
    second = sa.Kernels(0, side)
    try:
        a, b = Step(kernels, 6, 16), Step(second, 7, 8)
        held = a.all_held(), b.all_held()
        for _ in range(3):
            a.run()
            b.run()
        kernels.sync()
        second.sync()
        a.check(held[0])
        b.check(held[1])
    finally:
        second.close()


@pytest.mark.parametrize("bits", [16, 8])
def test_a_prompt_at_once_and_a_shared_prefix(kernels, bits):
    """Tokens of a prompt appended and attended to in one call see what they
    would one by one; a second sequence goes on from the first one's pages."""
    import torch

    step = Step(kernels, 8, bits)
    n = 100
    g = torch.Generator(device="cuda").manual_seed(9)
    x = torch.randn(n + 30, (HQ + 2 * HK) * D, generator=g, device="cuda")
    q, k, v = (t.unflatten(1, (-1, D)) for t in (x[:, :HQ * D], x[:, HQ * D:(HQ + HK) * D], x[:, (HQ + HK) * D:]))
    step.table[1, :6] = step.table[0, :6]  # 96 positions shared
    seq = ints([0] * n + [1] * 30)
    pos = ints(list(range(n)) + list(range(96, 126)))
    out = torch.empty(n + 30, HQ, D, device="cuda")
    ws = torch.empty(kernels.attn_decode_workspace_size(step.cache, HQ, n + 30), dtype=torch.uint8, device="cuda")
    assert kernels.kv_append(step.cache, step.table, seq, pos, k, v, n + 30) == 0
    assert kernels.attn_decode(step.cache, step.table, seq, pos, q, 0.125, 0, out, HQ, n + 30, ws) == 0
    kernels.sync()
    for r, (s, p) in enumerate(zip(seq.tolist(), pos.tolist())):
        want, room = attention(*step.held(s, p + 1), q[r].double().cpu().numpy(), 0.125)
        assert np.all(np.abs(out[r].double().cpu().numpy() - want) <= room), (s, p)
