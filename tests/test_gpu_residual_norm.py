"""The norms around a block with gate and residual, and their gradients, against their definition in 64 bits (ref_activations.py)."""
import ctypes
import math
import random
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
VECTORS = ("weight", "bias", "after_weight", "after_bias")


@pytest.fixture(scope="module")
def act(capi):
    from dynamiq_sigcomm_artifact_amd import activations
    return activations


def f64(t):
    return None if t is None else t.detach().double().cpu().numpy()


def normal(shape, dtype, seed, spread=1.0, mean=0.0):
    g = torch.Generator(device=DEV).manual_seed(seed)
    return (torch.randn(shape, generator=g, device=DEV) * spread + mean).to(dtype)


def near(got, want, size, operations, what, before=0.0):
    """one rounding to the result's type, another one of `before`, and `operations` of them in binary32 on what adds up to `size` in magnitude"""
    t = got.dtype
    rel, least = torch.finfo(t).eps / 2, torch.finfo(t).smallest_normal * torch.finfo(t).eps / 2
    tolerance = rel * np.abs(want) + least + (1 + rel) * (operations * U * size + rel * np.abs(before))
    off = np.abs(f64(got).reshape(want.shape) - want)
    assert np.all(off <= tolerance), (what, float((off - tolerance).max()), float(off.max()))


def shared(gate, shape):
    """a gate's row for each of y's"""
    if gate is None:
        return None
    return np.broadcast_to(f64(gate).reshape((1,) * (len(shape) - gate.dim()) + tuple(gate.shape)), shape).reshape(-1, shape[-1])


def tensors(shape, dtype, stream, parts, seed, of=None, gate=None):
    """parts: the names of what takes part beside y; of: a type for the vectors and the gate"""
    cols = shape[-1]
    t = {"y": normal(shape, dtype, seed, 1.5, 0.2)}
    if "residual" in parts:
        t["residual"] = normal(shape, stream, seed + 1, 2.0, -0.1)
    for k, name in enumerate(VECTORS):
        if name in parts:
            t[name] = normal((cols,), of or dtype, seed + 2 + k, 0.3, 1.0 if "weight" in name else 0.0)
    if gate is not None:
        t["gate"] = normal(gate, of or dtype, seed + 7, 0.4, 0.6)
    return t


def against_definition(act, t, dh=None, dr=None, eight=False, wants=None, **kw):
    """forward and backward of the tensors t; dh, dr: True for a random gradient"""
    s = {"residual_scale": 1.0, "block_scale": 1.0, "after": False, "before": True, "center": False, "eps": 1e-5, **kw}
    wants = list(t) if wants is None else wants
    leaf = {k: v.detach().requires_grad_(k in wants) for k, v in t.items()}
    got = act.residual_norm(leaf["y"], leaf.get("residual"), leaf.get("weight"), leaf.get("bias"), gate=leaf.get("gate"), after_weight=leaf.get("after_weight"),
                            after_bias=leaf.get("after_bias"), checkpoint=eight, **s)
    h, r = (got[0], got[1]) if s["before"] else (None, got)
    shape, cols = t["y"].shape, t["y"].shape[-1]
    flat = lambda x: None if x is None else f64(x).reshape(-1, cols)          # noqa: E731
    y, residual, gate = flat(t["y"]), flat(t.get("residual")), shared(t.get("gate"), shape)
    s.update({k: f64(t.get(k)) for k in VECTORS})
    want_h, want_r, st_r, st_y = A.block(y, residual, gate, s)
    stream = t["residual"].dtype if "residual" in t else t["y"].dtype

    # Sizes.  A sum of n values over threads is a chain of 8 (of 32 in the widest rows) within one, 6 steps in a wave and 16 at most between waves: at most 54 roundings of what
    # adds up; the mean takes part in the variance to second order, and a root and a quotient are two more.  With the products around them no value has seen more than 96.
    def normed(x, error, st, w, b):
        """norm of x, which is off by error (in units of 2^-24): the size of what the result is made of"""
        d, rms = np.abs(x) + np.abs(x).mean(1, keepdims=True), np.sqrt((x * x).mean(1, keepdims=True))
        inner = st[1] * (d + error + np.abs((x - st[0]) * st[1]) * (np.sqrt((error * error).mean(1, keepdims=True)) + rms * s["center"]))
        return (inner + np.abs((x - st[0]) * st[1])) * (1 if w is None else np.abs(w)) + (0 if b is None else np.abs(b))
    size = normed(y, 0 * y, st_y, s["after_weight"], s["after_bias"]) if s["after"] else np.abs(y)
    size = abs(s["block_scale"]) * size * (1 if gate is None else np.abs(gate)) + (0 if residual is None else abs(s["residual_scale"]) * np.abs(residual))
    plain = r is not None and r.data_ptr() == leaf["y"].data_ptr()
    assert r.shape == shape and r.dtype == stream
    if not plain:
        near(r, want_r, size, 96, "r")
    if s["before"]:
        assert h.shape == shape and h.dtype == t["y"].dtype
        near(h, want_h, normed(want_r, size, st_r, s["weight"], s["bias"]), 96, "h")
        if eight:
            assert torch.equal(got[2].data, act.compress(h.detach()).data) and got[2].shape == (y.shape[0], cols)
    if not wants:
        return got
    dh = normal(shape, t["y"].dtype, 101, 1e-2) if dh else None
    dr = normal(shape, stream, 102, 1e-2) if dr else None
    outputs = [(o, g) for o, g in ((h, dh), (r, dr)) if g is not None]
    grads = dict(zip(wants, torch.autograd.grad([o for o, _ in outputs], [leaf[k] for k in wants], [g for _, g in outputs], allow_unused=True)))
    # what the backward pass has of r and y: as stored, or the checkpoints of that
    kept_r, kept_y = flat(r), y
    if eight:
        kept_r, kept_y = A.restored(kept_r, NAME[stream]), A.restored(y, NAME[t["y"].dtype])
    through = dr if not plain else None
    want = A.block_gradients(kept_y, kept_r, st_r, st_y, gate, s, flat(dh), flat(through))
    before = 0.0
    if plain and dr is not None:         # r is y: what reaches it there reaches y, to whose gradient, rounded already, the engine adds it
        before = want["y"]
        want["y"] = want["y"] + flat(dr)
    # Sizes of the gradients: as above, and what r and the statistics are off by
    off_r = st_r[1] * (size + np.abs(kept_r) + np.abs(kept_r).mean(1, keepdims=True)) + np.sqrt((size * size).mean(1, keepdims=True)) * st_r[1]

    def back(g, xhat, off, st):
        """the size of the gradient through a norm"""
        x = np.abs(xhat) + off
        return st[1] * (g + g.mean(1, keepdims=True) + x * (g * x).mean(1, keepdims=True) * (1 + off.mean(1, keepdims=True)))
    total = 0 * y if through is None else np.abs(flat(through))
    sizes = {}
    if dh is not None and s["before"]:
        xhat, g = (kept_r - st_r[0]) * st_r[1], np.abs(flat(dh))
        sizes["weight"], sizes["bias"] = g * (np.abs(xhat) + off_r), g
        total = total + back(g if s["weight"] is None else g * np.abs(s["weight"]), xhat, off_r, st_r)
    sizes["residual"] = abs(s["residual_scale"]) * total
    total = abs(s["block_scale"]) * total
    if s["after"]:
        yhat = (kept_y - st_y[0]) * st_y[1]
        off_y = st_y[1] * (np.abs(y) + np.abs(y).mean(1, keepdims=True) + np.abs(kept_y)) + 2
        z = (np.abs(yhat) + off_y) * (1 if s["after_weight"] is None else np.abs(s["after_weight"])) + (0 if s["after_bias"] is None else np.abs(s["after_bias"]))
    else:
        z = np.abs(kept_y)
    if gate is not None:
        sizes["gate"] = total * z
        total = total * np.abs(gate)
    if s["after"]:
        sizes["after_weight"], sizes["after_bias"] = total * (np.abs(yhat) + off_y), total
        total = back(total if s["after_weight"] is None else total * np.abs(s["after_weight"]), yhat, off_y, st_y)
    sizes["y"] = total + (np.abs(flat(dr)) if plain and dr is not None else 0)
    rows = y.shape[0]
    for k in wants:
        if k in ("weight", "bias") and dh is None:
            assert grads[k] is None or not grads[k].any()
            continue
        g = grads[k]
        assert g.shape == t[k].shape and g.dtype == t[k].dtype, k
        if k in ("y", "residual"):
            near(g, want[k], sizes[k], 224, k, before)                           # through two norms: 96 each, and the products between them
        elif k == "gate":
            total_of = lambda x: x.reshape(shape).sum(tuple(d for d in range(len(shape) - 1) if t["gate"].dim() == 1 or (t["gate"].shape[d] == 1 and shape[d] > 1)))   # noqa: E731
            near(g, total_of(want[k]).reshape(t[k].shape), total_of(sizes[k]).reshape(t[k].shape), 224 + rows, k)
        else:
            near(g, want[k].sum(0), sizes[k].sum(0), 224 + rows, k)              # and the additions of the rows
    return got, grads


ALL = ("residual",) + VECTORS
COLS = [8, 9, 15, 31, 100, 257, 512, 513, 1001, 2048, 2055, 4096, 4099, 8192, 8193, 14336, 16390, 32768]


@pytest.mark.parametrize("cols", COLS)
@pytest.mark.parametrize("center", [False, True])
def test_widths(act, cols, center):
    """every number of threads and elements a thread, with everything taking part"""
    for k, (dtype, stream) in enumerate(((BF, BF), (HF, FP), (FP, FP))):
        t = tensors((3, cols), dtype, stream, ALL, cols + k, gate=(cols,))
        against_definition(act, t, True, True, center=center, after=True, residual_scale=0.9, block_scale=1.2)


@pytest.mark.parametrize("cols", [520, 2055, 4096, 4099, 8192, 8200, 14336, 16390])
@pytest.mark.parametrize("eight", [False, True])
def test_widths_of_few_sums(act, cols, eight):
    """every width with the kernels that keep fewer sums: the weight's, the bias' too, the gate's, the norm after the block's"""
    for k, (parts, gate, kw) in enumerate(((("residual", "weight"), None, {}), (("residual", "weight", "bias"), None, {"center": True}), (("residual",), (cols,), {}),
                                           (("weight", "after_weight"), None, {"after": True}), (("residual", "after_weight"), (5, cols), {"after": True}),
                                           (("residual", "weight", "bias"), (cols,), {"center": True}))):
        dtype, stream = ((BF, BF), (HF, FP), (FP, FP))[k % 3]
        against_definition(act, tensors((5, cols), dtype, stream, parts, cols + k, gate=gate), True, True, eight=eight, **kw)


@pytest.mark.parametrize("rows,cols", [(5001, 4096), (4100, 5000), (40001, 512), (2001, 8200)])
@pytest.mark.parametrize("parts,gate,kw", [(("residual", "weight"), False, {}), (("weight", "bias"), False, {"center": True}), (("residual", "weight", "after_weight"), True, {"after": True})],
                         ids=["lean", "centred", "sandwich"])
@pytest.mark.parametrize("eight", [False, True])
def test_many_rows(act, rows, cols, parts, gate, kw, eight):
    """what is beyond the cache, whose loads carry a hint and whose workgroups have many rows, against parts of it that are not"""
    t = tensors((rows, cols), BF, BF, parts, 9, of=FP, gate=(cols,) if gate else None)
    dh, dr = normal((rows, cols), BF, 10, 1e-2), normal((rows, cols), BF, 11, 1e-2)
    vectors = [k for k in t if k not in ("y", "residual")]

    def run(at):
        leaf = {k: (v if k in vectors else v[at]).detach().requires_grad_() for k, v in t.items()}
        got = act.residual_norm(leaf["y"], leaf.get("residual"), leaf.get("weight"), leaf.get("bias"), gate=leaf.get("gate"), after_weight=leaf.get("after_weight"),
                                checkpoint=eight, **kw)
        plain = got[1] is leaf["y"]
        grads = torch.autograd.grad(got[:1] if plain else got[:2], list(leaf.values()), (dh[at],) if plain else (dh[at], dr[at]))
        rows = [got[0].detach(), got[1].detach()] + [g for k, g in zip(leaf, grads) if k not in vectors] + ([got[2].codes, got[2].scales] if eight else [])
        return rows, {k: g.double() for k, g in zip(leaf, grads) if k in vectors}
    whole, sums = run(slice(0, rows))
    step = 700 * 4096 // cols
    total, size = {k: 0.0 for k in sums}, {k: 0.0 for k in sums}
    for at in range(0, rows, step):
        part, s = run(slice(at, at + step))
        assert all(torch.equal(a[at:at + step], b) for a, b in zip(whole, part))
        for k in s:
            total[k], size[k] = total[k] + s[k], size[k] + s[k].abs()
    # both are sums of the same terms; a chain of additions is off by 2^-24 of what it has passed at each: as many as rows at most, of terms whose magnitudes are ten times the parts' sums
    # or less where the sign is random over hundreds of rows
    for k in sums:
        assert float(((sums[k] - total[k]).abs() - rows * U * 10 * (size[k] + 1.0)).max()) <= 0, k


@pytest.mark.parametrize("dtype,stream", [(BF, BF), (BF, FP), (HF, HF), (HF, FP), (FP, FP)], ids=str)
@pytest.mark.parametrize("eight", [False, True])
def test_parts(act, dtype, stream, eight):
    """whatever takes part, and whatever does not"""
    rng = random.Random(5)
    for case in range(40):
        after, before, center = rng.random() < 0.5, rng.random() < 0.8, rng.random() < 0.5
        parts = [p for p in ALL if rng.random() < 0.6 and (after or "after" not in p) and (before or p not in ("weight", "bias"))]
        rows, cols = rng.choice(((1, 40), (7, 33), (20, 300), (5, 1030)))
        gate = rng.choice((None, None, (cols,), (rows, cols), (1, cols)))
        t = tensors((rows, cols), dtype, stream, parts, 10 * case, rng.choice((None, FP)), gate)
        plain = "residual" not in parts and gate is None and not after
        scales = dict(residual_scale=rng.choice((1.0, 0.7)), block_scale=rng.choice((1.0, 1.0 if plain else 0.5)))
        which = rng.choice(((True, True), (True, False), (False, True))) if before else (False, True)
        if plain and before and which == (False, True):
            which = (True, True)
        against_definition(act, t, *which, eight=eight, after=after, before=before, center=center, **scales)


@pytest.mark.parametrize("shape,gate", [((3000, 16), (16,)), ((3000, 16), (3000, 16)), ((1500, 2, 16), (1500, 1, 16)), ((1000, 3, 16), (1000, 1, 16)), ((30, 100, 16), (30, 1, 16)),
                                        ((2, 1500, 16), (2, 1, 16)), ((7, 1031, 24), (7, 1, 24)), ((1, 3000, 16), (1, 1, 16)), ((2, 3, 500, 16), (2, 3, 1, 16)), ((2, 3, 500, 16), (2, 1, 1, 16)),
                                        ((5, 1, 9), (5, 1, 9)), ((1100, 2, 9), (1, 1, 9))])
@pytest.mark.parametrize("after", [False, True])
def test_gates(act, shape, gate, after):
    """gates of one row, of some, of all; workgroups that have rows of one gate, and of several"""
    t = tensors(shape, BF, FP, ("residual", "weight") + ("after_weight",) * after, 3, gate=gate)
    against_definition(act, t, True, True, after=after)
    t["gate"] = t["gate"].float()
    against_definition(act, t, True, True, after=after, wants=["gate"])


def test_partial_gradients(act):
    """gradients that are not wanted change nothing of the others"""
    t = tensors((50, 200), BF, BF, ALL, 4, gate=(50, 200))
    _, whole = against_definition(act, t, True, True, after=True, center=True)
    for k in t:
        _, one = against_definition(act, t, True, True, after=True, center=True, wants=[k])
        assert torch.equal(one[k], whole[k]), k
    t = tensors((50, 200), BF, BF, ("residual", "weight"), 5)
    _, both = against_definition(act, t, True, True)
    assert both["y"].data_ptr() == both["residual"].data_ptr()          # nothing lies between them
    for k in ("y", "residual"):
        _, one = against_definition(act, t, True, True, wants=[k])
        assert torch.equal(one[k], both[k])
    _, scaled = against_definition(act, t, True, True, residual_scale=0.5)
    assert scaled["y"].data_ptr() != scaled["residual"].data_ptr()


def test_gradients_accumulate(act):
    """one gradient for y and the residual, where both are leaves that have one already, and where they are one tensor"""
    t = tensors((30, 64), FP, FP, ("residual",), 6)
    y, x = t["y"].requires_grad_(), t["residual"].requires_grad_()
    dh = normal((30, 64), FP, 7)
    first = torch.autograd.grad(act.residual_norm(y, x)[0], (y, x), dh)
    for _ in range(3):
        act.residual_norm(y, x)[0].backward(dh)
    # (g + g + g in this order)
    assert torch.equal(y.grad, first[0] + first[0] + first[0]) and torch.equal(x.grad, y.grad)
    z = normal((30, 64), FP, 8).requires_grad_()
    dz, = torch.autograd.grad(act.residual_norm(z, z)[0], z, dh)
    want = torch.autograd.grad(act.residual_norm(z.detach().requires_grad_(), z)[0], z, dh)[0]
    assert torch.equal(dz, 2 * want)


def test_backward_twice(act):
    """a graph that is kept gives the same gradients again"""
    t = {k: v.requires_grad_() for k, v in tensors((30, 130), BF, FP, ALL, 2, gate=(130,)).items()}
    h, r, _ = act.residual_norm(t["y"], t["residual"], t["weight"], t["bias"], gate=t["gate"], after=True, after_weight=t["after_weight"], after_bias=t["after_bias"], checkpoint=True)
    loss = (h.float().square().sum() + r.square().sum())
    first = torch.autograd.grad(loss, list(t.values()), retain_graph=True)
    again = torch.autograd.grad(loss, list(t.values()))
    assert all(torch.equal(a, b) for a, b in zip(first, again))


def test_not_differentiated(act):
    t = tensors((9, 50), BF, FP, ALL, 1)
    got = against_definition(act, t, center=True, after=True, wants=[])
    assert not got[0].requires_grad and not got[1].requires_grad
    got = against_definition(act, t, center=True, after=True, wants=[], eight=True)
    leaf = {k: v.clone().requires_grad_() for k, v in t.items()}
    with torch.no_grad():
        h, r = act.residual_norm(leaf["y"], leaf["residual"])
    assert not h.requires_grad and not r.requires_grad
    h, r, c = act.residual_norm(leaf["y"], leaf["residual"], checkpoint=True)
    assert h.requires_grad and r.requires_grad and not c.data.requires_grad
    y = leaf["y"]
    h, r = act.residual_norm(y)
    assert r is y
    r = act.residual_norm(y, leaf["residual"], before=False, checkpoint=True)
    assert isinstance(r, torch.Tensor)


def test_views_and_shapes(act):
    """what is not contiguous, and addresses that are aligned to an element only"""
    big = normal((60, 400), BF, 1)
    t = tensors((60, 100), BF, BF, ALL, 2, gate=(60, 100))
    for y in (big[:, 3:103], big[:, ::4], normal((100, 60), BF, 3).t()):
        t["y"] = y
        against_definition(act, t, True, True, after=True)
    flat = normal((60 * 100 + 101,), BF, 4)
    t["y"], t["weight"] = flat[1:6001].view(60, 100), flat[6001:6101]
    against_definition(act, t, True, True, after=True, eight=True)
    t = tensors((100,), FP, FP, ("residual", "weight"), 5)
    against_definition(act, t, True, True)
    t = tensors((2, 3, 4, 100), HF, HF, ("residual", "weight"), 5, gate=(2, 3, 1, 100))
    against_definition(act, t, True, True)
    y = normal((20, 64), BF, 1).requires_grad_()
    dh = normal((64, 20), BF, 2).t()
    assert torch.equal(torch.autograd.grad(act.residual_norm(y)[0], y, dh)[0], torch.autograd.grad(act.residual_norm(y)[0], y, dh.contiguous())[0])


def test_empty(act):
    t = tensors((0, 40), BF, FP, ALL, 1, gate=(40,))
    leaf = {k: v.requires_grad_() for k, v in t.items()}
    h, r, c = act.residual_norm(leaf["y"], leaf["residual"], leaf["weight"], leaf["bias"], gate=leaf["gate"], after=True, after_weight=leaf["after_weight"],
                                after_bias=leaf["after_bias"], checkpoint=True)
    assert h.shape == r.shape == (0, 40) and c.shape == (0, 40)
    grads = torch.autograd.grad(h.sum() + r.sum(), list(leaf.values()))
    assert all(g.shape == v.shape and not g.any() for g, v in zip(grads, leaf.values()))


def test_rows_are_apart(act):
    """what is not finite in a row stays there, in all but the sums over the rows; a row of zeros"""
    t = tensors((12, 70), BF, BF, ALL, 1, gate=(12, 70))
    dh, dr = normal((12, 70), BF, 2), normal((12, 70), BF, 3)

    def run(eight, center):
        leaf = {k: v.detach().requires_grad_() for k, v in t.items()}
        got = act.residual_norm(leaf["y"], leaf["residual"], leaf["weight"], leaf["bias"], gate=leaf["gate"], after=True, after_weight=leaf["after_weight"],
                                after_bias=leaf["after_bias"], center=center, checkpoint=eight)
        return list(got[:2]) + list(torch.autograd.grad(got[:2], [leaf[k] for k in ("y", "residual", "gate")], (dh, dr)))
    for eight in (False, True):
        for center in (False, True):
            t["y"][4], t["residual"][4] = 0.0, 0.0
            want = run(eight, center)
            assert all(torch.isfinite(v).all() for v in want)
            kept = t["y"].clone()
            for bad in (math.nan, math.inf):
                t["y"][7, 3] = bad
                got = run(eight, center)
                others = [i for i in range(12) if i != 7]
                assert all(torch.equal(a[others], b[others]) for a, b in zip(got, want)) and bool(torch.isnan(got[0][7]).all())
                t["y"] = kept.clone()


def test_large_and_small_values(act):
    """rows near the ends of the range of their type"""
    for scale in (1e-18, 1e-6, 1e6, 1e17):
        t = tensors((6, 90), FP, FP, ("weight",), 1)
        t["y"] = t["y"] * scale
        against_definition(act, t, True, False, eps=0.0)
    t = tensors((6, 90), HF, HF, ("residual", "weight"), 1)
    t["y"] = (t["y"] * 1e4).clamp(-6e4, 6e4)
    t["residual"] = t["residual"] * 0
    against_definition(act, t, True, True)


def test_the_same_every_time(act):
    t = tensors((3000, 130), BF, FP, ALL, 1, gate=(130,))
    first = against_definition(act, t, True, True, after=True, center=True)[1]
    for _ in range(3):
        again = against_definition(act, t, True, True, after=True, center=True)[1]
        assert all(torch.equal(first[k], again[k]) for k in first)


def test_holds_eight_bits(act):
    y, x = normal((2048, 2048), BF, 1), normal((2048, 2048), BF, 2).requires_grad_()
    torch.cuda.synchronize()
    before = torch.cuda.memory_allocated()
    h, r, c = act.residual_norm(y.clone(), x, gate=None, after=True, checkpoint=True)
    held = torch.cuda.memory_allocated() - before - (h.numel() + r.numel()) * 2 - c.data.numel()
    assert held <= 2 * 2048 * 2048 * 33 // 32 + 2048 * 16 + 4096
    del r
    assert torch.autograd.grad(h.sum(), x)[0].shape == x.shape


def test_refusals(act):
    y = normal((4, 40), BF, 1).requires_grad_()
    w = normal((40,), BF, 2)
    for call, text in ((lambda: act.residual_norm(y.double()), "element dtype"), (lambda: act.residual_norm(y.cpu()), "must live on the GPU"), (lambda: act.residual_norm(y, y.cpu()), "must live on the GPU"),
                       (lambda: act.residual_norm(y, y[:2]), "y's shape"), (lambda: act.residual_norm(y, y.half()), "float32"), (lambda: act.residual_norm(y.float(), y), "float32"),
                       (lambda: act.residual_norm(y, weight=w[:39]), r"\[cols\]"), (lambda: act.residual_norm(y, weight=w.view(1, 40)), r"\[cols\]"), (lambda: act.residual_norm(y, weight=w.half()), "float32"),
                       (lambda: act.residual_norm(y, gate=w[:39]), "a gate is"), (lambda: act.residual_norm(y, gate=y[:2]), "a gate is"), (lambda: act.residual_norm(y.view(2, 2, 40), gate=y), "a gate is"),
                       (lambda: act.residual_norm(y.view(2, 2, 40), gate=y.view(2, 2, 40)[:1]), "a gate is"), (lambda: act.residual_norm(y, after_weight=w), "after=True"),
                       (lambda: act.residual_norm(y, y, weight=w, before=False), "before=True"), (lambda: act.residual_norm(y[:, :7]), "32768"), (lambda: act.residual_norm(normal((1, 32769), BF, 1)), "32768"),
                       (lambda: act.residual_norm(y, eps=-1.0), "eps"), (lambda: act.residual_norm(y, eps=math.nan), "eps"), (lambda: act.residual_norm(y, y, residual_scale=math.inf), "scales"),
                       (lambda: act.residual_norm(None), "a tensor argument"), (lambda: act.residual_norm(y, [1.0]), "a tensor argument"), (lambda: act.residual_norm(y[0, 0]), "is required"),
                       (lambda: torch.autograd.grad(act.residual_norm(y)[0].sum(), y, create_graph=True), "cannot be differentiated again")):
        with pytest.raises(RuntimeError, match=text):
            call()
    h, r = act.residual_norm(y, y.detach())
    with torch.no_grad():
        r.add_(1)
    with pytest.raises(RuntimeError, match="modified by an inplace operation"):
        h.sum().backward()


def test_graph_streams_and_threads(act):
    t = tensors((300, 200), BF, FP, ALL, 1, gate=(200,))
    dh, dr = normal((300, 200), BF, 2), normal((300, 200), FP, 3)

    def work():
        leaf = {k: v.detach().requires_grad_() for k, v in t.items()}
        h, r, c = act.residual_norm(leaf["y"], leaf["residual"], leaf["weight"], leaf["bias"], gate=leaf["gate"], after=True, after_weight=leaf["after_weight"],
                                    after_bias=leaf["after_bias"], center=True, checkpoint=True)
        return [h.detach(), r.detach(), c.data] + list(torch.autograd.grad((h, r), list(leaf.values()), (dh, dr)))
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        work()
    torch.cuda.current_stream().wait_stream(side)
    graphs = [torch.cuda.CUDAGraph() for _ in range(2)]
    outs = []
    for graph in graphs:
        with torch.cuda.graph(graph):
            outs.append(work())
    for k in range(4):
        t["y"].normal_()
        for graph in graphs:
            graph.replay()
        torch.cuda.synchronize()
        want = work()
        for out in outs:
            assert all(torch.equal(p, q) for p, q in zip(out, want)), k
        torch.cuda.synchronize()
    got = {}

    def run(k):
        with torch.cuda.stream(torch.cuda.Stream()):
            for _ in range(20):
                got[k] = work()
            torch.cuda.current_stream().synchronize()
    threads = [threading.Thread(target=run, args=(k,)) for k in range(4)]
    [v.start() for v in threads]
    [v.join() for v in threads]
    assert len(got) == 4 and all(torch.equal(p, q) for v in got.values() for p, q in zip(v, want))


def test_recording_beside_a_living_graph_is_refused(act):
    w = normal((64,), BF, 1).requires_grad_()
    y = normal((20, 64), BF, 2)
    held = act.residual_norm(y, weight=w)[0]
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with pytest.raises(RuntimeError, match="made on the default stream"):
        with torch.cuda.graph(graph):
            act.residual_norm(y, weight=w)
    torch.cuda.synchronize()
    held.sum().backward()
    del held


def test_behind_the_results(act):
    """nothing is written outside h, r, the checkpoints, the gradients and the work buffer"""
    from dynamiq_sigcomm_artifact_amd import capi
    L, s = capi.lib(), torch.cuda.current_stream().cuda_stream
    for rows, cols in ((3, 33), (5, 100), (40, 9), (2, 2055)):
        n, bytes_ = rows * cols, (L.dq_checkpoint_bytes(rows, cols) + 15) // 16 * 16
        t = tensors((rows, cols), BF, BF, ALL, 1, gate=(cols,))

        def room(count, dtype):
            return torch.full((count + 64,), 77, dtype=dtype, device=DEV)
        buffers = {"h": room(n, BF), "r": room(n, BF), "h8": room(L.dq_checkpoint_bytes(rows, cols), torch.uint8), "kept": room(bytes_ + L.dq_checkpoint_bytes(rows, cols), torch.uint8),
                   "stats": room(4 * rows, FP), "dy": room(n, BF), "dresidual": room(n, BF), **{"d" + k: room(cols, BF) for k in ("gate",) + VECTORS}}
        sizes = {k: v.numel() - 64 for k, v in buffers.items()}
        at = {k: v.data_ptr() + 32 * v.element_size() for k, v in buffers.items()}
        dh, dr = normal((rows, cols), BF, 2), normal((rows, cols), BF, 3)
        inputs = {k: v.data_ptr() for k, v in t.items()}
        both = dict(rows=rows, cols=cols, rows_per_gate=rows, eps=1e-5, residual_scale=1.0, block_scale=1.0, dtype=1, stream_dtype=1, center=1, after=1, before=1, keep_r=1, keep_y=1)
        o = capi.ResidualNorm(**inputs, **{k: at[k] for k in ("h", "r", "h8", "kept", "stats")}, **both)
        assert L.dq_residual_norm_forward(ctypes.byref(o), 0, s) == 0, L.dq_last_error()
        o = capi.ResidualNorm(**inputs, **{k: at[k] for k in at if k not in ("h", "r", "h8")}, dh=dh.data_ptr(), dr=dr.data_ptr(), **both)
        o.work_floats = L.dq_residual_norm_work_floats(ctypes.byref(o))
        work = room(o.work_floats, FP)
        o.work = work.data_ptr() + 128
        assert L.dq_residual_norm_backward(ctypes.byref(o), 0, s) == 0, L.dq_last_error()
        for k, v in {**buffers, "work": work}.items():
            assert bool((v[:32] == 77).all()) and bool((v[v.numel() - 32:] == 77).all()), k
        # and what lies between is what the module gives
        leaf = {k: v.detach().requires_grad_() for k, v in t.items()}
        h, r, c = act.residual_norm(leaf["y"], leaf["residual"], leaf["weight"], leaf["bias"], gate=leaf["gate"], after=True, after_weight=leaf["after_weight"],
                                    after_bias=leaf["after_bias"], center=True, eps=1e-5, checkpoint=True)
        grads = dict(zip(leaf, torch.autograd.grad((h, r), list(leaf.values()), (dh, dr))))
        for k, v in {"h": h, "r": r, "h8": c.data, **{"d" + k: g for k, g in grads.items()}}.items():
            assert torch.equal(buffers[k][32:32 + sizes[k]].view(v.shape), v), k


@pytest.mark.parametrize("shape,gate", [((6, 8200), (6, 8200)), ((2, 3, 9001), (2, 1, 9001)), ((130, 2, 8195), (130, 1, 8195)), ((500, 8193), (500, 8193)), ((1, 32768), (32768,)), ((3, 16400), (16400,))])
@pytest.mark.parametrize("after", [False, True])
@pytest.mark.parametrize("eight", [False, True])
def test_wide_gates(act, shape, gate, after, eight):
    """rows that are wider than registers hold, whose gates are of one row, of some, of all"""
    if eight:
        shape, gate = (shape[0] * (shape[1] if len(shape) == 3 else 1), shape[-1]), gate[-1:]
    t = tensors(shape, BF, FP, ("residual", "weight", "bias") + ("after_weight",) * after, 3, gate=gate)
    against_definition(act, t, True, True, after=after, eight=eight, center=True)


def test_wide_parts(act):
    """whatever takes part, and whatever does not, in such rows"""
    rng = random.Random(6)
    for case in range(24):
        after, before, center, eight = rng.random() < 0.7, rng.random() < 0.7, rng.random() < 0.5, rng.random() < 0.5
        dtype, stream = rng.choice(((BF, BF), (BF, FP), (HF, HF), (HF, FP), (FP, FP)))
        parts = [p for p in ALL if rng.random() < 0.6 and (after or "after" not in p) and (before or p not in ("weight", "bias"))]
        rows, cols = rng.choice(((1, 8201), (7, 9000), (3, 16385), (2, 20003)))
        gate = rng.choice((None, (cols,), (rows, cols)))
        t = tensors((rows, cols), dtype, stream, parts, 10 * case, rng.choice((None, FP)), gate)
        plain = "residual" not in parts and gate is None and not after
        which = rng.choice(((True, True), (True, False), (False, True))) if before else (False, True)
        if plain and before and which == (False, True):
            which = (True, True)
        against_definition(act, t, *which, eight=eight, after=after, before=before, center=center, residual_scale=0.7, block_scale=1.0 if plain else 0.5)


def test_wide_rows_keep_apart(act):
    """a row with what is no number, or beyond the largest, makes no other row so"""
    t = tensors((5, 9003), BF, BF, ("residual", "weight", "after_weight"), 4, gate=(5, 9003))
    dh, dr = normal((5, 9003), BF, 5), normal((5, 9003), BF, 6)

    def run():
        leaf = {k: v.clone().requires_grad_() for k, v in t.items()}
        h, r = act.residual_norm(leaf["y"], leaf["residual"], leaf["weight"], gate=leaf["gate"], after=True, after_weight=leaf["after_weight"])
        return [h.detach(), r.detach(), *torch.autograd.grad((h, r), [leaf[k] for k in ("y", "residual", "gate")], (dh, dr))]
    clean = run()
    t["y"][1, 77], t["residual"][3, 9002] = float("nan"), float("inf")
    for a, b in zip(clean, run()):
        assert torch.equal(a[[0, 2, 4]], b[[0, 2, 4]])
        assert not torch.isfinite(b[[1, 3]]).all()


def test_wide_work(act):
    """the work buffer of such rows: nothing is written outside of it, and one that is smaller is refused"""
    from dynamiq_sigcomm_artifact_amd import capi
    L, s = capi.lib(), torch.cuda.current_stream().cuda_stream
    for rows, cols, gate in ((9, 8200, (8200,)), (9, 16392, None), (600, 8200, (600, 8200))):
        t = tensors((rows, cols), BF, BF, ("residual", "weight"), 1, gate=gate)
        leaf = {k: v.detach().requires_grad_() for k, v in t.items()}
        h, r = act.residual_norm(leaf["y"], leaf["residual"], leaf["weight"], gate=leaf.get("gate"), eps=1e-5)
        dh, dr = normal((rows, cols), BF, 2), normal((rows, cols), BF, 3)
        want = dict(zip(leaf, torch.autograd.grad((h, r), list(leaf.values()), (dh, dr))))
        stats = torch.empty(rows, 4, device=DEV)
        h2, r2 = torch.empty_like(h), torch.empty_like(r)
        got = {k: torch.empty_like(v) for k, v in want.items()}
        both = dict({k: v.data_ptr() for k, v in t.items()}, rows=rows, cols=cols, rows_per_gate=rows // (gate[0] if gate and len(gate) == 2 else 1), eps=1e-5, residual_scale=1.0, block_scale=1.0,
                    dtype=1, stream_dtype=1, before=1, stats=stats.data_ptr(), r=r2.data_ptr())
        assert L.dq_residual_norm_forward(ctypes.byref(capi.ResidualNorm(**both, h=h2.data_ptr())), 0, s) == 0, L.dq_last_error()
        o = capi.ResidualNorm(**both, dh=dh.data_ptr(), dr=dr.data_ptr(), dy=got["y"].data_ptr(), dresidual=got["residual"].data_ptr(), dweight=got["weight"].data_ptr(),
                              dgate=got["gate"].data_ptr() if gate else None)
        n = L.dq_residual_norm_work_floats(ctypes.byref(o))
        work = torch.full((n + 64,), 77.0, device=DEV)
        o.work, o.work_floats = work.data_ptr() + 128, n - 1
        assert L.dq_residual_norm_backward(ctypes.byref(o), 0, s) != 0 and b"too small" in L.dq_last_error()
        o.work_floats = n
        assert L.dq_residual_norm_backward(ctypes.byref(o), 0, s) == 0, L.dq_last_error()
        assert bool((work[:32] == 77).all()) and bool((work[-32:] == 77).all())
        assert torch.equal(h2, h) and torch.equal(r2, r)
        for k in want:
            assert torch.equal(got[k], want[k]), k


def test_wide_graph(act):
    """two graphs of such rows, each with its own workspace, between the program's own work"""
    t = tensors((70, 8300), BF, FP, ALL, 1, gate=(70, 8300))
    dh, dr = normal((70, 8300), BF, 2), normal((70, 8300), FP, 3)

    def work():
        leaf = {k: v.detach().requires_grad_() for k, v in t.items()}
        h, r, c = act.residual_norm(leaf["y"], leaf["residual"], leaf["weight"], leaf["bias"], gate=leaf["gate"], after=True, after_weight=leaf["after_weight"],
                                    after_bias=leaf["after_bias"], checkpoint=True)
        return [h.detach(), r.detach(), c.data] + list(torch.autograd.grad((h, r), list(leaf.values()), (dh, dr)))
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        work()
    torch.cuda.current_stream().wait_stream(side)
    graphs, outs = [torch.cuda.CUDAGraph() for _ in range(2)], []
    for graph in graphs:
        with torch.cuda.graph(graph):
            outs.append(work())
    for k in range(4):
        t["y"].normal_()
        for graph in graphs:
            graph.replay()
        torch.cuda.synchronize()
        want = work()
        for out in outs:
            assert all(torch.equal(p, q) for p, q in zip(out, want)), k
        torch.cuda.synchronize()


def test_forward_mode_is_refused(act):
    """a tangent of any input is not dropped without a word, whoever else wants a gradient"""
    import torch.autograd.forward_ad as forward
    t = tensors((6, 64), BF, FP, ALL, 1, gate=(64,))

    def call(t):
        return act.residual_norm(t["y"], t["residual"], t["weight"], t["bias"], gate=t["gate"], after=True, after_weight=t["after_weight"], after_bias=t["after_bias"])
    with forward.dual_level():
        for name in t:
            for wanted in (False, True):
                mine = {k: v.detach().requires_grad_(wanted) for k, v in t.items()}
                mine[name] = forward.make_dual(t[name], torch.ones_like(t[name]))
                with pytest.raises(RuntimeError, match="forward mode"):
                    call(mine)
                with torch.no_grad(), pytest.raises(RuntimeError, match="forward mode"):
                    call(mine)
        plain = forward.make_dual(t["y"], torch.ones_like(t["y"]))
        with pytest.raises(RuntimeError, match="forward mode"):
            act.residual_norm(plain)
        call(t)


@pytest.mark.parametrize("cols", [90, 513, 4096, 8192, 9000, 16400, 32768])
def test_rows_near_the_largest_sum_of_squares(act, cols):
    """rows whose squares add up to somewhat less than 2^128, at every width, are like others; from there on they are NaN, and their neighbours are not"""
    for dtype, parts, kw in ((FP, ("weight",), {}), (BF, ("weight",), {"center": True}), (FP, ("residual", "weight", "after_weight"), {"after": True})):
        t = tensors((6, cols), dtype, dtype, parts, 1)
        v = t["y"].double()
        # (with a norm after the block it is that one which takes them)
        t["y"] = (v * (0.9 * 2.0 ** 64 / v.square().sum(-1, keepdim=True).sqrt())).to(dtype)
        if "after" not in kw:
            against_definition(act, t, True, False, eps=0.0, **kw)
        else:
            against_definition(act, t, True, True, eps=1e-5, **kw)
        t["y"][2] *= 4
        h = act.residual_norm(t["y"], t.get("residual"), t["weight"], after_weight=t.get("after_weight"), eps=1e-5, **kw)[0]
        assert bool(torch.isnan(h[2]).all()) and bool(torch.isfinite(h[[0, 1, 3, 4, 5]]).all())


@pytest.mark.parametrize("shape,gate", [((40001, 512), (512,)), ((30001, 256), (256,)), ((20000, 768), (768,)), ((5001, 4096), (4096,)), ((4100, 5000), (5000,)), ((1201, 8192), (8192,)),
                                        ((2001, 8200), (8200,)), ((601, 16390), (16390,)), ((4095, 64), (4095, 64)), ((8190, 3, 512), (8190, 1, 512)), ((2730, 3, 512), (2730, 1, 512)),
                                        ((3000, 4, 256), (3000, 1, 256)), ((1001, 5, 512), (1001, 1, 512)), ((90, 3, 8200), (90, 1, 8200)), ((40, 900, 768), (40, 1, 768)),
                                        ((16, 300, 4096), (16, 1, 4096)), ((7, 160, 8200), (7, 1, 8200))])
@pytest.mark.parametrize("eight", [False, True])
@pytest.mark.parametrize("stream", [BF, FP], ids=str)
def test_every_row_counts_once(act, shape, gate, eight, stream):
    """The sums over the rows of numbers that binary32 adds without rounding: a row that is lost, or taken twice, changes them.  Rows of +1 and -1, as many of each, have a mean of 0, a
    mean square of 1 and, with eps 0, are their own norm; what is multiplied with them are whole numbers up to 7, of which 2^24 / 7 add up exactly.  The weight is 0 and its gradient is
    not: nothing but the gradient of r reaches the gate and the norm after the block."""
    cols, flat = shape[-1], (-1, shape[-1])
    rows = math.prod(shape[:-1])
    g = torch.Generator(device=DEV).manual_seed(rows)

    def signs(*size):
        return 1.0 - 2.0 * torch.randint(0, 2, size, generator=g, device=DEV).float()

    def whole():
        return torch.randint(1, 8, shape, generator=g, device=DEV).float()
    # each pair of columns has both signs, which gate and weight change together
    y = torch.stack((signs(*shape[:-1], cols // 2),) * 2, -1).mul_(torch.tensor([1.0, -1.0], device=DEV)).view(shape)
    t = {"y": y.to(BF), "weight": torch.zeros(cols, device=DEV), "bias": torch.zeros(cols, device=DEV), "after_bias": torch.zeros(cols, device=DEV),
         "gate": signs(*gate[:-1], cols // 2).repeat_interleave(2, -1), "after_weight": signs(cols // 2).repeat_interleave(2)}
    dh, dr = whole(), whole()
    per = t["gate"] if len(gate) == 1 else t["gate"].expand(shape)
    after = y * t["after_weight"]
    r = after * per
    want = {"weight": dh * r, "bias": dh, "gate": dr * after, "after_weight": dr * per * y, "after_bias": dr * per}
    for names in (list(want), ["weight", "bias"], ["gate", "after_weight"]):
        # without the norm after the block where nothing of it is wanted
        sandwich = "after_weight" in names
        leaf = {k: v.detach().requires_grad_(k in names) for k, v in t.items()}
        residual = torch.zeros(shape, dtype=stream, device=DEV)
        kw = dict(gate=leaf["gate"], after=True, after_weight=leaf["after_weight"], after_bias=leaf["after_bias"]) if sandwich else {}
        for center in (False, True):
            got = act.residual_norm(leaf["y"], residual, leaf["weight"], leaf["bias"], center=center, eps=0.0, checkpoint=eight, **kw)
            assert torch.equal(got[1].float(), r if sandwich else y)
            grads = dict(zip(names, torch.autograd.grad(got[:2], [leaf[k] for k in names], (dh.to(BF), dr.to(stream)))))
            for k in names:
                v = want[k] if sandwich or k != "weight" else dh * y
                v = v.double().view(shape)
                v = v.sum(1, keepdim=True) if k == "gate" and len(gate) == 3 else v if k == "gate" and len(gate) == len(shape) else v.reshape(flat).sum(0)
                assert torch.equal(grads[k].double(), v), (k, center, names)
