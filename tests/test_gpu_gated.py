"""The gated activation and its gradients against their definition in 64 bits (ref_activations.py)."""
import math
import threading

import numpy as np
import pytest
import torch

import ref_activations as A

pytestmark = pytest.mark.gpu
DEV = "cuda:0"
BF, HF, FP = torch.bfloat16, torch.float16, torch.float32
NAME = {BF: "bfloat16", HF: "float16", FP: "float32"}
U = 2.0 ** -24


@pytest.fixture(scope="module")
def act(capi):
    from dynamiq_sigcomm_artifact_amd import activations
    return activations


def f64(t):
    return t.detach().double().cpu().numpy()


def normal(shape, dtype, seed, spread=1.5):
    g = torch.Generator(device=DEV).manual_seed(seed)
    return (torch.randn(shape, generator=g, device=DEV) * spread).to(dtype)


def half_step(t):
    """a rounding to the type: relative, and half of its smallest number"""
    return torch.finfo(t).eps / 2, torch.finfo(t).smallest_normal * torch.finfo(t).eps / 2


def exponent(g, kind):
    g = np.clip(g, -20, 20)
    return g if kind == "silu" else 2 * np.sqrt(2 / np.pi) * (g + 0.044715 * g ** 3)


def check(out, want, size, dtype, q, beside):
    """size: the sum of the magnitudes of what is added up.  In binary32: q is off by four roundings of it (it is made of terms of one sign), and so is, relatively, exp(-|q|),
    whose own product with log2(e) and power are two more of |q| and two; a reciprocal good to a unit in the last place, and ten products and sums: (20 + 6 |q|) 2^-24.
    What the exponential flushes to zero is below 2^-126; where it is all there is of the sigmoid, that times what the sigmoid is multiplied by, beside, is lost of the result
    (silu of -87.5 times 2: e^-87.5 < 2^-126, and 175 2^-126 = 2.1e-36 of it)."""
    rel, least = half_step(dtype)
    tolerance = rel * np.abs(want) + least + (1 + rel) * ((20 + 6 * np.abs(q)) * U * size + 2.0 ** -126 * (1 + beside))
    assert np.all(np.abs(out - want) <= tolerance), float((np.abs(out - want) - tolerance).max())


def against_definition(act, x, da, kind, eight, gate=None, up=None):
    """through autograd, packed where x is given"""
    leaves = [t.detach().requires_grad_() for t in ((x,) if x is not None else (gate, up))]
    got = act.gated(*leaves, kind=kind, checkpoint=eight)
    a, c = got if eight else (got, None)
    grads = torch.autograd.grad(a, leaves, da)
    dtype, cols = a.dtype, a.shape[-1]
    if x is not None:
        v = f64(x).reshape(-1, 2 * cols)
        g, u = v[:, :cols], v[:, cols:]
        d = f64(grads[0]).reshape(-1, 2 * cols)
        dg, du = d[:, :cols], d[:, cols:]
    else:
        g, u, dg, du = (f64(t).reshape(-1, cols) for t in (gate, up) + tuple(grads))
    assert all(t.dtype == dtype for t in grads)
    q = exponent(g, kind)
    value = A.act(g, kind)[0]
    check(f64(a).reshape(-1, cols), value * u, np.abs(value * u), dtype, q, np.abs(g * u))
    if eight:
        assert torch.equal(c.data, act.compress(a.detach()).data) and c.shape == (a.numel() // cols if cols else 0, cols)
        g, u = A.restored(g, NAME[dtype]), A.restored(u, NAME[dtype])
        q = exponent(g, kind)
    value, slope = A.act(g, kind)
    s = np.abs(slope) + 2 * np.abs(g) * np.minimum(np.exp(-np.abs(q)), 1) * (1 + 1.6 * 3 * 0.044715 * np.clip(g, -20, 20) ** 2 * (kind != "silu")) + 1
    d = f64(da).reshape(-1, cols)
    check(dg, d * u * slope, np.abs(d * u) * s, dtype, q, np.abs(d * u) * (1 + np.abs(g) * (1 + np.clip(g, -20, 20) ** 2)))
    check(du, d * value, np.abs(d * value), dtype, q, np.abs(d * g))


SHAPES = [(1, 1), (3, 7), (2, 8), (5, 33), (7, 256), (130, 257), (33, 1000)]


@pytest.mark.parametrize("r,c", SHAPES)
@pytest.mark.parametrize("kind", ["silu", "gelu_tanh"])
@pytest.mark.parametrize("eight", [False, True])
@pytest.mark.parametrize("dtype", [FP, BF, HF], ids=str)
def test_definition(act, r, c, kind, eight, dtype):
    against_definition(act, normal((r, 2 * c), dtype, r + c), normal((r, c), dtype, 9), kind, eight)


@pytest.mark.parametrize("kind", ["silu", "gelu_tanh"])
@pytest.mark.parametrize("eight", [False, True])
def test_wide_values(act, kind, eight):
    """gates far out, where the sigmoid is 0 or 1, and at zero"""
    g = torch.cat((torch.linspace(-130, 130, 521), torch.tensor([0.0, -0.0, 1e-30, -1e-30, 1e4, -1e4, 3e4, -3e4, 19.9, 20.1, -19.9, -20.1]))).to(DEV)
    for dtype in (FP, BF):
        gate = g.to(dtype).view(1, -1)
        against_definition(act, None, normal(gate.shape, dtype, 2), kind, eight, gate, normal(gate.shape, dtype, 1))


@pytest.mark.parametrize("kind", ["silu", "gelu_tanh"])
def test_largest_gates_have_gradients(act, kind):
    top = torch.finfo(FP).max
    gate = torch.tensor([[top, -top, 1e30, -1e30]], device=DEV).requires_grad_()
    up = torch.full((1, 4), 1e-3, device=DEV)
    dg, = torch.autograd.grad(act.gated(gate, up, kind=kind), gate, torch.ones(1, 4, device=DEV))
    assert torch.equal(dg, torch.tensor([[1e-3, 0.0, 1e-3, 0.0]], device=DEV))


@pytest.mark.parametrize("bad", [math.nan, math.inf])
def test_what_is_not_finite_stays_in_its_place(act, bad):
    x = normal((6, 80), BF, 1)
    x[2, 50] = bad                           # of up
    x[4, 3] = math.nan                       # of the gate
    leaf = x.clone().requires_grad_()
    a, c = act.gated(leaf, checkpoint=True)
    hit = torch.zeros(6, 40, dtype=torch.bool, device=DEV)
    hit[2, 10] = hit[4, 3] = True
    assert torch.equal(~torch.isfinite(a), hit)
    # in 8 bits a block of 32 is NaN as one: the gate's block of row 4, and that of up in row 2
    d, = torch.autograd.grad(a, leaf, torch.ones_like(a))
    want = torch.zeros(6, 80, dtype=torch.bool, device=DEV)
    want[2, :32] = True                      # dgate takes up
    want[4, :32] = want[4, 40:72] = True
    assert torch.equal(torch.isnan(d), want)
    leaf = x.clone().requires_grad_()
    d, = torch.autograd.grad(act.gated(leaf), leaf, torch.ones_like(a))
    want = torch.zeros(6, 80, dtype=torch.bool, device=DEV)
    want[2, 10] = want[4, 3] = want[4, 43] = True
    assert torch.equal(~torch.isfinite(d), want)


def test_views(act):
    big = normal((40, 300), BF, 3)
    da = normal((40, 70), BF, 4)
    for x in (big[:, 5:145], big[:, 8:148], normal((140, 40), BF, 5).t(), normal((80, 140), BF, 6)[::2]):
        against_definition(act, x, da, "silu", False)
        against_definition(act, x, da, "silu", True)
        assert torch.equal(act.gated(x), act.gated(x.contiguous()))
    against_definition(act, None, da, "silu", False, big[:, 3:73], big[:, 101:171])
    against_definition(act, None, da.view(2, 20, 70), "gelu_tanh", True, normal((2, 20, 70), BF, 7), normal((20, 2, 70), BF, 8).transpose(0, 1))
    against_definition(act, normal((2, 4, 5, 140), HF, 7), normal((40, 70), HF, 1).view(2, 4, 5, 70), "silu", True)
    against_definition(act, normal((140,), FP, 7), normal((70,), FP, 1), "silu", False)
    odd = normal((40 * 140 + 1,), BF, 9)[1:].view(40, 140)             # an address that is aligned to an element only
    against_definition(act, odd, da, "silu", True)
    t = normal((70, 40), BF, 10).t()                                    # a gradient that is not contiguous
    against_definition(act, big[:, :140], t, "silu", False)
    same = normal((40, 70), BF, 11).requires_grad_()                    # the same tensor twice
    dx, = torch.autograd.grad(act.gated(same, same), same, da)
    g = f64(same)
    v, s = A.act(g, "silu")
    assert np.all(np.abs(f64(dx) - f64(da) * (g * s + v)) <= (2.0 ** -8 + 100 * U) * np.abs(f64(da)) * (np.abs(g * s) + np.abs(v)) * 2 + 1e-30)


def test_partial_gradients_and_none(act):
    g, u, da = normal((9, 50), BF, 1), normal((9, 50), BF, 2), normal((9, 50), BF, 3)
    whole = [t.clone().requires_grad_() for t in (g, u)]
    want = torch.autograd.grad(act.gated(*whole), whole, da)
    for k in range(2):
        leaves = [g.clone(), u.clone()]
        leaves[k].requires_grad_()
        got, = torch.autograd.grad(act.gated(*leaves), leaves[k], da)
        assert torch.equal(got, want[k])
    assert not act.gated(g, u).requires_grad
    with torch.no_grad():
        assert not act.gated(*whole).requires_grad
    out, c = act.gated(g, u, checkpoint=True)
    assert not out.requires_grad and torch.equal(c.data, act.compress(out).data) and not c.data.requires_grad
    with torch.inference_mode():
        assert torch.equal(act.gated(g, u), out)


@pytest.mark.parametrize("eight", [False, True])
def test_hinted_loads(act, eight):
    """what is beyond the cache against parts of it that are not"""
    x, da = normal((3001, 2 * 8000), BF, 1), normal((3001, 8000), BF, 2)

    def run(x, da):
        leaf = x.detach().requires_grad_()
        out = act.gated(leaf, checkpoint=eight)
        out, c = out if eight else (out, None)
        return [out.detach(), torch.autograd.grad(out, leaf, da)[0]] + ([c.codes, c.scales] if eight else [])
    whole = run(x, da)
    for k in range(0, 3001, 700):
        assert all(torch.equal(a[k:k + 700], b) for a, b in zip(whole, run(x[k:k + 700], da[k:k + 700])))


def test_empty(act):
    for shape in ((0, 10), (5, 0), (0,)):
        x = torch.empty(shape, device=DEV, requires_grad=True)
        a, c = act.gated(x, checkpoint=True)
        assert a.shape == shape[:-1] + (shape[-1] // 2,) and c.rows == a.shape[:-1].numel()
        d, = torch.autograd.grad(a.sum(), x)
        assert d.shape == shape


def test_holds_eight_bits(act):
    x = normal((2048, 4096), BF, 1).requires_grad_()
    torch.cuda.synchronize()
    before = torch.cuda.memory_allocated()
    a, c = act.gated(x * 1, checkpoint=True)
    held = torch.cuda.memory_allocated() - before - a.numel() * 2 - c.data.numel()
    assert held <= 2048 * 4096 * 33 // 32 + 4096


def test_refusals(act):
    x = normal((4, 10), BF, 1).requires_grad_()
    for call, text in ((lambda: act.gated(x, kind="relu"), "unknown activation"), (lambda: act.gated(x[:, :9]), "2 cols"), (lambda: act.gated(x, x[:, :5]), "one shape"),
                       (lambda: act.gated(x, x.float()), "one type"), (lambda: act.gated(x.double()), "element dtype"), (lambda: act.gated(x.cpu()), "must live on the GPU"),
                       (lambda: act.gated(x, x.cpu()), "must live on the GPU"), (lambda: act.gated(None), "a tensor argument"), (lambda: act.gated(x[0, 0]), "required"),
                       (lambda: torch.autograd.grad(act.gated(x).sum(), x, create_graph=True), "cannot be differentiated again")):
        with pytest.raises(RuntimeError, match=text):
            call()
    a = act.gated(x)
    with torch.no_grad():
        x.add_(1)
    with pytest.raises(RuntimeError, match="modified by an inplace operation"):
        a.sum().backward()


def test_graph_streams_and_threads(act):
    def work(x, da):
        leaf = x.detach().requires_grad_()
        a, c = act.gated(leaf, checkpoint=True)
        d, = torch.autograd.grad(a, leaf, da)
        b = act.gated(leaf.detach(), kind="gelu_tanh")
        return a.detach(), c.data, d, b
    x, da = normal((200, 320), BF, 1), normal((200, 160), BF, 2)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        work(x, da)
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = work(x, da)
    for k in range(4):
        x.normal_()
        graph.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(p, q) for p, q in zip(out, work(x, da))), k
        torch.cuda.synchronize()
    want, got = work(x, da), {}

    def run(k):
        with torch.cuda.stream(torch.cuda.Stream()):
            torch.cuda.current_stream().wait_stream(torch.cuda.default_stream())
            for _ in range(20):
                got[k] = work(x, da)
            torch.cuda.current_stream().synchronize()
    torch.cuda.synchronize()
    threads = [threading.Thread(target=run, args=(k,)) for k in range(4)]
    [t.start() for t in threads]
    [t.join() for t in threads]
    assert len(got) == 4 and all(torch.equal(p, q) for v in got.values() for p, q in zip(v, want))


def test_recording_beside_a_living_graph_is_refused(act):
    x, da = normal((20, 64), BF, 1).requires_grad_(), normal((20, 32), BF, 2)
    held = act.gated(x)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with pytest.raises(RuntimeError, match="made on the default stream"):
        with torch.cuda.graph(graph):
            act.gated(x)
    torch.cuda.synchronize()
    held.backward(da)
    del held


def test_c_interface_writes_where_it_is_told(act):
    """strides of the gradients, nothing outside the rows, a gradient that is not asked for"""
    import ctypes

    from dynamiq_sigcomm_artifact_amd import capi
    L, s = capi.lib(), torch.cuda.current_stream().cuda_stream
    r, c = 5, 37
    g, u, da = normal((r, c), BF, 1), normal((r, c), BF, 2), normal((r, c), BF, 3)
    leaves = [t.clone().requires_grad_() for t in (g, u)]
    want = torch.autograd.grad(act.gated(*leaves), leaves, da)
    room = torch.full((r, 100), 7.0, dtype=BF, device=DEV)
    o = capi.Gated(gate=g.data_ptr(), up=u.data_ptr(), gate_stride=c, up_stride=c, out=da.data_ptr(), dgate=room.data_ptr() + 6, dgate_stride=100, rows=r, cols=c, dtype=1, kind=0)
    assert L.dq_gated_backward(ctypes.byref(o), 0, s) == 0
    assert torch.equal(room[:, 3:40], want[0]) and bool((room[:, :3] == 7).all()) and bool((room[:, 40:] == 7).all())


def test_backward_makes_its_gradients_and_no_more(act):
    """what a backward pass takes of memory beside its results: nothing of the checkpoint's size"""
    x, da = normal((2048, 4096), BF, 1).requires_grad_(), normal((2048, 2048), BF, 2)
    for up in (None, normal((2048, 4096), BF, 3).requires_grad_()):
        d = da if up is None else normal((2048, 4096), BF, 4)
        a, c = act.gated(x, up, checkpoint=True)
        leaves = [x] if up is None else [x, up]
        torch.cuda.synchronize()
        torch.cuda.reset_peak_memory_stats()
        before = torch.cuda.memory_allocated()
        grads = torch.autograd.grad(a, leaves, d)
        peak = torch.cuda.max_memory_allocated() - before
        assert peak <= sum(g.numel() * 2 for g in grads) + 65536
        del a, c, grads


def test_forward_mode_is_refused(act):
    """a tangent is not dropped without a word, whoever else wants a gradient"""
    import torch.autograd.forward_ad as forward
    g, u, t = normal((4, 64), BF, 1), normal((4, 64), BF, 2), normal((4, 64), BF, 3)
    with forward.dual_level():
        dual = forward.make_dual(g, t)
        for wanted in (False, True):
            other = u.clone().requires_grad_(wanted)
            for call in (lambda: act.gated(dual), lambda: act.gated(dual, checkpoint=True), lambda: act.gated(dual, other), lambda: act.gated(other, dual), lambda: act.gated(dual.view(2, 2, 64))):
                with pytest.raises(RuntimeError, match="forward mode"):
                    call()
                with torch.no_grad(), pytest.raises(RuntimeError, match="forward mode"):
                    call()
        assert torch.equal(act.gated(forward.unpack_dual(dual).primal, u), act.gated(g, u))


def test_halves_of_a_batch_are_read_in_place(act):
    """as two tensors, each a view with consecutive rows of more dimensions than two: right, and nothing of their size is made beside the results"""
    x, da = normal((3, 5, 140), BF, 1), normal((3, 5, 70), BF, 2)
    for gate, up in (x.chunk(2, -1), normal((3, 5, 300), BF, 3)[:, :, 8:288].chunk(2, -1), [v.transpose(0, 1) for v in normal((5, 3, 280), BF, 4).chunk(2, -1)],
                     normal((3, 10, 280), BF, 5)[:, ::2].chunk(2, -1), normal((3, 5, 560), BF, 6)[:, :, ::2].chunk(2, -1), normal((1, 1, 280), BF, 7).expand(3, 5, 280).chunk(2, -1)):
        d = da if gate.shape[-1] == 70 else normal(gate.shape, BF, 8)
        for eight in (False, True):
            against_definition(act, None, d, "silu", eight, gate, up)
        assert torch.equal(act.gated(gate, up), act.gated(gate.contiguous(), up.contiguous()))
    x, da = normal((8, 256, 4096), BF, 1), normal((8, 256, 2048), BF, 2)
    for eight in (False, True):
        gate, up = (v.detach().requires_grad_() for v in x.chunk(2, -1))
        torch.cuda.synchronize()
        torch.cuda.reset_peak_memory_stats()
        before = torch.cuda.memory_allocated()
        got = act.gated(gate, up, checkpoint=eight)
        held = torch.cuda.memory_allocated() - before
        assert torch.cuda.max_memory_allocated() - before == held
        a = got[0] if eight else got
        assert held <= a.numel() * 2 + eight * 3 * (a.numel() * 33 // 32) + 65536
        torch.cuda.reset_peak_memory_stats()
        before = torch.cuda.memory_allocated()
        grads = torch.autograd.grad(a, (gate, up), da)
        assert torch.cuda.max_memory_allocated() - before <= 2 * 2 * a.numel() + 65536
        del got, a, grads
