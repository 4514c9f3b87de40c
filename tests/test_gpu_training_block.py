"""A training step around a block as its operators are used together: a norm, a 4-bit linear layer, the gated activation, a 4-bit linear layer, and a norm after it with gate,
residual and the next norm; its gradients through a dynamic-bitrate bucket, the norm that clips, and AdamW."""
import math
import os
import sys
import threading

import pytest
import torch

pytestmark = pytest.mark.gpu
DEV = "cuda:0"
BF = torch.bfloat16
ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
TOKENS, WIDTH, HIDDEN = 70, 96, 160


@pytest.fixture(scope="module")
def lib():
    if not torch.cuda.is_available():
        pytest.skip("needs a GPU")
    from dynamiq_sigcomm_artifact_amd import activations, capi, dynamiq_pipeline, microscale, optimizer
    return activations, capi, dynamiq_pipeline, microscale, optimizer


class Model(object):
    def __init__(self, lib, eight, capturable=False):
        self.act, capi, pipeline, self.ms, self.optimizer = lib
        self.eight = eight
        g = torch.Generator(device=DEV).manual_seed(4)
        self.x, self.aim = (torch.randn(TOKENS, WIDTH, generator=g, device=DEV).to(BF) for _ in range(2))
        self.weights = [(torch.randn(r, c, generator=g, device=DEV) / math.sqrt(c)).to(BF) for r, c in ((2 * HIDDEN, WIDTH), (WIDTH, HIDDEN))]
        self.weights += [(1 + 0.2 * torch.randn(WIDTH, generator=g, device=DEV)).to(BF) for _ in range(4)]
        self.weights = [w.requires_grad_() for w in self.weights]
        sizes = [w.numel() for w in self.weights]
        total = -(-sum(sizes) // 256) * 256
        self.bucket, self.reduced = (torch.zeros(total, dtype=BF, device=DEV) for _ in range(2))
        self.parts, self.grads = ([v.view_as(w) for v, w in zip(f[:sum(sizes)].split(sizes), self.weights)] for f in (self.bucket, self.reduced))
        self.signs = {}
        for k, n in enumerate((TOKENS, WIDTH, 2 * HIDDEN)):
            self.signs[n] = torch.empty(-(-n // 256) * 8, dtype=torch.int32, device=DEV)
            capi.rand_diag_bits(self.signs[n], self.signs[n].numel() * 32, k + 1)
        self.count = torch.zeros(1, dtype=torch.int64, device=DEV)
        self.pipe = pipeline.SinglePassBuckets(DEV, seed=3, u=45.0)
        self.opt = self.optimizer.AdamW(self.weights, lr=1e-2, bits=8, capturable=capturable)
        self.norm = torch.zeros(2, device=DEV)

    def forward(self):
        up, down, before, after, gate, following = self.weights
        eight = self.eight
        h, r, *c = self.act.residual_norm(self.x, weight=before, checkpoint=eight)
        both = self.ms.linear(h, up, sign=(self.signs[2 * HIDDEN], self.signs[TOKENS]), seed=1, step=self.count, checkpoint=c[0] if eight else None)
        a, c = self.act.gated(both, checkpoint=True) if eight else (self.act.gated(both), None)
        y = self.ms.linear(a, down, sign=(self.signs[WIDTH], self.signs[TOKENS]), seed=2, step=self.count, checkpoint=c)
        return self.act.residual_norm(y, r, following, gate=gate, after=True, after_weight=after, checkpoint=eight)[0], (h, both, a, y)

    def step(self):
        h, _ = self.forward()
        for part, v in zip(self.parts, torch.autograd.grad((h - self.aim).float().square().mean(), self.weights)):
            part.copy_(v)
        self.count.add_(1)
        self.pipe.begin_step()
        self.pipe.run(self.bucket, self.reduced)
        self.optimizer.grad_norm(self.grads, 0.01, work=self.opt.work, out=self.norm)
        for w, g in zip(self.weights, self.grads):
            w.grad = g
        self.opt.step(grad_scale=self.norm[1:])


def exact(m):
    """the same in 64 bits, without a rounding"""
    w = [v.detach().double().cpu().requires_grad_() for v in m.weights]
    up, down, before, after, gate, following = w

    def norm(v, weight):
        return v * torch.rsqrt(v.square().mean(1, keepdim=True) + 1e-6) * weight
    x = m.x.double().cpu()
    both = norm(x, before) @ up.t()
    g, u = both[:, :HIDDEN], both[:, HIDDEN:]
    y = (g * torch.sigmoid(g) * u) @ down.t()
    out = norm(x + gate * norm(y, after), following)
    return torch.autograd.grad((out - m.aim.double().cpu()).square().mean(), w)


@pytest.mark.parametrize("eight", [False, True])
def test_gradients_against_the_exact_ones(lib, eight):
    m = Model(lib, eight)
    for _ in range(3):
        want = exact(m)
        m.step()
        # E2M1 to the nearest is off by a sixth of a value at most, stochastically by twice that, E4M3 by a sixteenth; a gradient takes three such factors at most, and those of
        # the layers around it: what they add up to stays below the gradient's own norm
        for part, e in zip(m.parts, want):
            assert float((part.double().cpu() - e).norm() / e.norm()) < 1.0
        assert torch.isfinite(m.reduced).all()


@pytest.mark.parametrize("eight", [False, True])
def test_gradients_are_the_operators(lib, eight):
    """what autograd makes of the block is what each operator's backward pass gives on what it is handed"""
    m = Model(lib, eight)
    out, (h, both, a, y) = m.forward()
    loss = (out - m.aim).float().square().mean()
    dout, dy, da, dboth, dh, *weights = torch.autograd.grad(loss, [out, y, a, both, h] + m.weights)
    leaf = lambda t: t.detach().requires_grad_()          # noqa: E731
    up, down, before, after, gate, following = (leaf(w) for w in m.weights)

    v = leaf(y)
    got = m.act.residual_norm(v, m.x, following, gate=gate, after=True, after_weight=after, checkpoint=eight)
    grads = torch.autograd.grad(got[0], (v, following, gate, after), dout)
    assert torch.equal(got[0], out) and all(torch.equal(p, q) for p, q in zip(grads, (dy, weights[5], weights[4], weights[3])))

    kw = dict(seed=2, step=m.count, sign=(m.signs[WIDTH], m.signs[TOKENS]))
    v = leaf(a)
    got = m.ms.linear(v, down, checkpoint=m.act.compress(v) if eight else None, **kw)
    grads = torch.autograd.grad(got, (v, down), dy)
    assert torch.equal(got, y) and torch.equal(grads[0], da) and torch.equal(grads[1], weights[1])

    v = leaf(both)
    got = m.act.gated(v, checkpoint=eight)
    got = got[0] if eight else got
    assert torch.equal(got, a) and torch.equal(torch.autograd.grad(got, v, da)[0], dboth)

    kw = dict(seed=1, step=m.count, sign=(m.signs[2 * HIDDEN], m.signs[TOKENS]))
    v = leaf(h)
    got = m.ms.linear(v, up, checkpoint=m.act.compress(v) if eight else None, **kw)
    grads = torch.autograd.grad(got, (v, up), dboth)
    assert torch.equal(got, both) and torch.equal(grads[0], dh) and torch.equal(grads[1], weights[0])

    got = m.act.residual_norm(m.x, weight=before, checkpoint=eight)
    assert torch.equal(got[0], h) and torch.equal(torch.autograd.grad(got[0], before, dh)[0], weights[2])


@pytest.mark.parametrize("eight", [False, True])
def test_recorded_steps_are_the_eager_ones(lib, eight):
    a, b = Model(lib, eight, True), Model(lib, eight, True)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        a.step()
        a.pipe.join()
    torch.cuda.current_stream().wait_stream(side)
    b.step()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        a.step()
    for _ in range(3):
        a.pipe.join()
        graph.replay()
        b.step()
        torch.cuda.synchronize()
        assert torch.equal(a.bucket, b.bucket) and torch.equal(a.reduced, b.reduced) and torch.equal(a.norm, b.norm)
        assert all(torch.equal(v, w) for v, w in zip(a.weights, b.weights))


def test_threads_on_their_own_streams(lib):
    def run(k, out):
        with torch.cuda.stream(torch.cuda.Stream()):
            m = Model(lib, k % 2 == 0)
            m.x.add_(k)
            for _ in range(8):
                m.step()
            m.pipe.join()
            torch.cuda.current_stream().synchronize()
            out[k] = [v.detach().clone() for v in m.weights] + [m.norm.clone()]
            torch.cuda.current_stream().synchronize()
    alone, together = {}, {}
    for k in range(4):
        run(k, alone)
    threads = [threading.Thread(target=run, args=(k, together)) for k in range(4)]
    [t.start() for t in threads]
    [t.join() for t in threads]
    for k in range(4):
        assert all(torch.equal(v, w) for v, w in zip(alone[k], together[k])), k


def test_command(lib):
    """evaluate.py --training-step, its part with the block, runs to its end"""
    sys.path.insert(0, ROOT)
    import evaluate
    lines = []
    emit, evaluate._emit = evaluate._emit, lambda **kw: lines.append(kw)
    try:
        evaluate.training_block(torch.device(DEV), tokens=300, width=320, hidden=256, steps=2)
    finally:
        evaluate._emit = emit
    assert [v["training_block"] for v in lines] == ["run", "layers", "layers_16_bits", "step"]
    assert math.isfinite(lines[0]["loss_last"]) and all(v["us"] > 0 for v in lines[1:])
    assert lines[0]["held_bytes_8_bits"] < 0.7 * lines[0]["held_bytes_16_bits"]
