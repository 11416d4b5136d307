"""The serving operators together, as a decode step of several requests' beams
runs them: residual and norm with an 8-bit copy, the LM head over the 8-bit
rows, each request's adapter beside it, the selection, the reordering of the
beams' states. Checked against 64-bit arithmetic, on a stream of its own,
captured and replayed, and on two handles with workspaces of their own."""
import numpy as np
import pytest

from test_gpu_beam import _want as beam_want
from test_gpu_qmm_i8 import _weights

pytestmark = pytest.mark.gpu

U = 2.0 ** -24
R, W, H, V, N, RANK, G = 3, 4, 512, 5003, 5, 16, 64
ROWS = R * W


class Step:
    """One step's buffers and calls on a handle."""

    def __init__(self, kernels, seed):
        import torch

        import streamoe_amd as sa

        self.k = kernels
        g = torch.Generator(device="cuda").manual_seed(seed)
        rn = lambda *s: torch.randn(*s, generator=g, device="cuda")
        self.x, self.res = rn(ROWS, H), rn(ROWS, H) * 3
        self.w = (1 + 0.1 * rn(H)).to(torch.bfloat16)
        self.head = _weights(np.random.default_rng(seed), V, H, 4, G)
        self.qw = sa.QuantWeights(self.head[0], *self.head[1], G, 4)
        self.set = sa.Adapters((rn(N, RANK, H) * 0.05).to(torch.bfloat16), (rn(N, V, RANK) * 0.05).to(torch.bfloat16),
                               rn(N))
        self.ids = torch.tensor([2, 2, 2, 2, -1, -1, -1, -1, 0, 0, 0, 0], dtype=torch.int32, device="cuda")
        self.scores = -torch.rand(ROWS, generator=g, device="cuda")
        self.done = torch.zeros(ROWS, dtype=torch.uint8, device="cuda")
        self.done[5] = 1
        e = lambda *s, t=torch.float32: torch.empty(*s, dtype=t, device="cuda")
        self.sum, self.norm = e(ROWS, H), e(ROWS, H)
        self.codes, self.sc = e(ROWS, H, t=torch.int8), e(ROWS, H // G)
        self.logits = e(ROWS, V)
        self.v, self.rows, self.tok = e(R, W), e(R, W, t=torch.int32), e(R, W, t=torch.int32)
        self.src, self.dst = rn(ROWS, 700), torch.zeros(ROWS, 700, device="cuda")
        self.states = [sa.BeamState(self.src, self.dst)]
        self.lws = e(kernels.lora_workspace_size(self.set, ROWS), t=torch.uint8)
        self.bws = e(kernels.beam_select_workspace_size(R, W, V, W), t=torch.uint8)
        torch.cuda.synchronize()

    def run(self):
        k = self.k
        for status in (
                k.rmsnorm(self.x, self.res, self.w, 1e-6, ROWS, H, self.sum, self.norm, self.codes, self.sc, G),
                k.qmm_i8(self.qw, self.codes, self.sc, G, self.logits, V, H, ROWS),
                k.lora(self.set, self.ids, self.norm, self.logits, self.logits, V, H, ROWS, self.lws),
                k.beam_select(self.logits, self.scores, self.done, 1, R, W, V, W, self.v, self.rows, self.tok, self.bws),
                k.beam_reorder(self.states, self.rows.view(-1))):
            assert status == 0, status

    def outputs(self):
        return [t.clone() for t in (self.sum, self.norm, self.codes, self.sc, self.logits, self.v, self.rows, self.tok,
                                    self.dst)]

    def check(self):
        f = lambda t: t.double().cpu().numpy()
        s64 = f(self.x) + f(self.res)
        y64 = s64 / np.sqrt((s64 ** 2).mean(1, keepdims=True) + 1e-6) * f(self.w)
        assert np.all(np.abs(f(self.norm) - y64) <= (H / 512 + 14) * U * np.abs(y64) + 1e-30)
        # The product's inputs are the codes it was given, the adapters' the f32 rows.
        q, s, b = self.head[2:]
        x = f(self.codes).reshape(ROWS, -1, G) * f(self.sc)[:, :, None]
        wq = q.reshape(V, -1, G) * s[:, :, None] + b[:, :, None]
        want = np.einsum("tgc,vgc->tv", x, wq)
        # As test_gpu_qmm_i8 and test_gpu_lora bound each of them, coarsely.
        bound = (2 * (H // G) + 24) * U * np.einsum("tgc,vgc->tv", np.abs(x), np.abs(wq) + 15 * s[:, :, None] + 2 * np.abs(b)[:, :, None])
        for t, i in enumerate(self.ids.tolist()):
            if i >= 0:
                A, B, sc = f(self.set.a[i]), f(self.set.b[i]), float(self.set.scale[i])
                want[t] += sc * (B @ (A @ y64[t]))
                bound[t] += (2.0 ** -15 + (H + RANK + 60) * U) * abs(sc) * (np.abs(B) @ (np.abs(A) @ np.abs(y64[t])))
        got = f(self.logits)
        assert np.all(np.abs(got - want) <= bound + 4 * U * np.abs(want))
        wv, wr, wt = beam_want(got, f(self.scores), self.done.cpu().numpy(), 1, R, W, V, W)
        assert np.array_equal(self.rows.cpu().numpy(), wr) and np.array_equal(self.tok.cpu().numpy(), wt)
        assert np.allclose(f(self.v), wv, rtol=2 * U, atol=36 * U)
        assert np.array_equal(f(self.dst), f(self.src)[wr.ravel()])


def test_chain(kernels):
    step = Step(kernels, 1)
    step.run()
    kernels.sync()
    step.check()


def test_chain_on_another_stream(kernels):
    import torch

    step = Step(kernels, 2)
    own, side = torch.cuda.current_stream(), torch.cuda.Stream()
    try:
        kernels.set_stream(side)
        step.run()
        kernels.sync()  # waits for the handle's stream
        step.check()
    finally:
        kernels.set_stream(own)


def test_chain_replayed_with_eager_work_between(kernels):
    import torch

    import streamoe_amd as sa

    step, other = Step(kernels, 3), Step(kernels, 4)
    graph = sa.capture_graph(kernels, step.run)
    for i in range(4):
        step.x.normal_()
        step.ids.copy_(torch.randint(-1, N, (ROWS,), device="cuda", dtype=torch.int32))
        graph.replay()
        other.run()  # eager work of another step, own workspaces
        torch.cuda.synchronize()
        got = step.outputs()
        step.check()
        other.check()
        step.run()
        kernels.sync()
        assert all(torch.equal(a, b) for a, b in zip(got, step.outputs()))


def test_two_handles_at_once(kernels):
    import torch

    import streamoe_amd as sa

    side = torch.cuda.Stream()
    second = sa.Kernels(0, side)
    try:
        a, b = Step(kernels, 5), Step(second, 6)
        for _ in range(3):
            a.run()
            b.run()
        kernels.sync()
        second.sync()
        a.check()
        b.check()
    finally:
        second.close()
