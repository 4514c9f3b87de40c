"""The gradient norm and the AdamW step against their definitions in 64 bits (ref_operators.py)."""
import math

import numpy as np
import pytest
import torch

import ref_operators as R

pytestmark = pytest.mark.gpu
DEV = "cuda:0"
BF, HF, FP = torch.bfloat16, torch.float16, torch.float32


@pytest.fixture(scope="module")
def opt(capi):
    from dynamiq_sigcomm_artifact_amd import optimizer
    return optimizer


def views(sizes, dtype, seed, scale=1.0, offset=0):
    """consecutive views of one buffer, the first `offset` elements into it"""
    g = torch.Generator(device=DEV).manual_seed(seed)
    flat = (torch.randn(offset + sum(sizes), generator=g, device=DEV) * scale).to(dtype)
    out, at = [], offset
    for n in sizes:
        out.append(flat[at:at + n])
        at += n
    return out


# ---- norm ----

@pytest.mark.parametrize("sizes", [[1], [8191], [8192], [8193], [5, 0, 31, 1000003], [17] * 130, [8192 * 3000 + 1]], ids=str)
@pytest.mark.parametrize("dtype", [FP, BF, HF], ids=str)
def test_norm(opt, sizes, dtype):
    grads = views(sizes, dtype, 1, offset=1)
    norm = math.sqrt(sum(float(g.double().square().sum()) for g in grads))
    got = opt.grad_norm(grads, 0.5 * norm).double().tolist()
    # sums in 64 bits, then one rounding each
    assert abs(got[0] - norm) <= norm * (2.0 ** -24 + 1e-12) and abs(got[1] - 0.5 * norm / (norm + 1e-6)) <= 2.0 ** -24 + 1e-12
    assert opt.grad_norm(grads).tolist()[1] == 1.0 and opt.grad_norm(grads, 2 * norm).tolist()[1] == 1.0


def test_norm_of_mixed_types_and_nothing(opt):
    grads = views([1000] * 3, FP, 1) + views([77] * 70, BF, 2) + views([4001], HF, 3) + views([0, 5], FP, 4)
    norm = math.sqrt(sum(float(g.double().square().sum()) for g in grads))
    work = opt.norm_work(DEV)
    first = opt.grad_norm(grads, 1.0, work=work)
    assert abs(float(first[0]) - norm) <= norm * 2.0 ** -23
    assert opt.grad_norm([grads[-2]], 1.0, work=work).tolist() == [0.0, 1.0]
    assert opt.grad_norm(views([0, 0], BF, 1), work=work).tolist() == [0.0, 1.0]
    assert torch.equal(opt.grad_norm(grads, 1.0, work=work), first)          # the same bits, whichever workgroup ends last


def test_norm_of_extreme_values(opt):
    assert opt.grad_norm([torch.full((10000,), 1e30, device=DEV)]).tolist()[0] == pytest.approx(1e32, rel=1e-7)
    assert opt.grad_norm([torch.full((10000,), 1e-30, device=DEV)]).tolist()[0] == pytest.approx(1e-28, rel=1e-7)
    for bad in (float("inf"), -float("inf"), float("nan")):
        x = torch.ones(100001, device=DEV)
        x[100000] = bad
        norm, factor = opt.grad_norm([x[:50000], x[50000:]], 1.0).tolist()
        assert not math.isfinite(norm) and math.isnan(factor)


def test_norm_refusals(opt):
    x = torch.ones(64, device=DEV)
    with pytest.raises(RuntimeError, match="contiguous"):
        opt.grad_norm([x[::2]])
    with pytest.raises(RuntimeError, match="unsupported element dtype"):
        opt.grad_norm([x.double()])
    with pytest.raises(RuntimeError, match="work buffer is too small"):
        opt.grad_norm([x], work=torch.zeros(8, dtype=torch.float64, device=DEV))
    with pytest.raises(RuntimeError, match="work: wrong dtype"):
        opt.grad_norm([x], work=torch.zeros(4096, device=DEV))
    with pytest.raises(RuntimeError, match="max_norm must be positive"):
        opt.grad_norm([x], 0.0)


# ---- AdamW ----

SIZES = [1, 31, 32, 33, 0, 2047, 2048, 2049, 5000, 100003]
HYPER = dict(lr=3e-3, betas=(0.9, 0.99), eps=1e-6, weight_decay=0.05)


def blocks(arrays):
    """list of float64 arrays -> one arena"""
    return np.concatenate([np.pad(a, (0, -len(a) % 32)) for a in arrays])


def host(tensors):
    return [t.detach().double().cpu().numpy() for t in tensors]


def arena_parts(arena, sizes):
    at, out = 0, []
    for n in sizes:
        out.append(arena[at:at + n])
        at += -(-n // 32) * 32
    return out


def close(got, want, rel, of=None):
    """within rel of the larger of |want| and `of`"""
    assert np.all(np.abs(got - want) <= rel * np.maximum(np.abs(want), 0 if of is None else of)), float(np.max(np.abs(got - want)))


def half_step(dtype):
    return torch.finfo(dtype).eps / 2


@pytest.mark.parametrize("pd,gd,master", [(FP, FP, False), (FP, BF, False), (BF, BF, True), (BF, FP, False), (HF, HF, True), (BF, HF, False), (HF, FP, True)], ids=str)
@pytest.mark.parametrize("bits", [32, 8])
def test_steps(opt, pd, gd, master, bits):
    """three steps, each against the definition on the states that the kernel had"""
    params, scale = views(SIZES, pd, 1, 0.5, offset=1), torch.full((1,), 0.25, device=DEV)
    state, weights = opt.adamw_state(params, bits), opt.master_weights(params) if master else None
    for t in (1, 2, 777):
        grads = views(SIZES, gd, 10 + t, 1e-2, offset=3)
        p0 = arena_parts(weights.double().cpu().numpy(), SIZES) if master else host(params)
        if bits == 32:
            m0, v0 = (arena_parts(x.double().cpu().numpy(), SIZES) for x in state)
        else:
            was = [x.cpu().numpy() for x in state]
            m0, r0 = (arena_parts(R.decode8(was[0][k], was[1][k]), SIZES) for k in (0, 1))
            v0 = [r * r for r in r0]
        opt.adamw_step(params, grads, state, t, master=weights, grad_scale=scale, **HYPER)
        want = [R.adamw(p, 0.25 * g, m, v, t, HYPER["lr"], HYPER["betas"], HYPER["eps"], HYPER["weight_decay"])
                for p, g, m, v in zip(p0, host(grads), m0, v0)]
        got_p = arena_parts(weights.double().cpu().numpy(), SIZES) if master else host(params)
        for k, (p, m, v) in enumerate(want):
            # The weight: two products and a difference, three half steps of it at most.  The step: the moment's four roundings (of terms that may cancel: `step` takes
            # their magnitudes), v's seven, halved by the root, whose own is one, the product with the correction and the sum with eps two; then the reciprocal, good to a
            # whole step, two products, and three constants that are rounded themselves.
            step = HYPER["lr"] / (1 - 0.9 ** t) * (0.9 * np.abs(m0[k]) + 0.1 * np.abs(0.25 * host(grads)[k])) / (np.sqrt(v) / math.sqrt(1 - 0.99 ** t) + HYPER["eps"])
            err = (3 * np.abs(p) + (4 + 3.5 + 1 + 2 + 2 + 2 + 3) * step) * 2.0 ** -24
            if not master:
                err = err + half_step(pd) * (np.abs(p) + err) + (2.0 ** -25 if pd == HF else 0)
            assert np.all(np.abs(got_p[k] - p) <= err), (t, k, float(np.max(np.abs(got_p[k] - p) - err)))
        if master:
            for p, w in zip(params, got_p):
                assert torch.equal(p.cpu(), torch.from_numpy(w).float().to(pd))
        m_all, v_all = blocks([w[1] for w in want]), blocks([w[2] for w in want])
        if bits == 32:
            # 0.9 m + 0.1 g with g a product: four roundings of terms that may cancel; v's terms are of one sign
            bound = blocks([0.9 * np.abs(m) + 0.1 * np.abs(0.25 * g) for m, g in zip(m0, host(grads))])
            assert np.all(np.abs(state[0].double().cpu().numpy() - m_all) <= 4 * 2.0 ** -24 * bound + 2.0 ** -149)
            assert np.all(np.abs(state[1].double().cpu().numpy() - v_all) <= 6 * 2.0 ** -24 * v_all + 2.0 ** -148)
        else:
            d = np.concatenate([R.dither(-(-n // 32) * 32, t) for n in SIZES])
            # m is off by four roundings of terms that may cancel; v by seven of terms of one sign (the square of the stored root is one), its root by half of that and one of its own.
            # So a byte, and with the byte given a code, lies between those of the two ends of that interval.  (Ends at a border do occur: sqrt(0.01 (0.25 g)^2) is
            # a multiple of a fortieth of a gradient with eight bits, and 448 / 2^k is one of those.)
            bound = blocks([0.9 * np.abs(m) + 0.1 * np.abs(0.25 * g) for m, g in zip(m0, host(grads))])
            r_all = np.sqrt(v_all)
            for row, x, off, dd in ((0, m_all, 4 * 2.0 ** -24 * bound, d), (1, r_all, 5 * 2.0 ** -24 * r_all, 2 ** 20 - 1 - d)):
                codes, scales = state[0][row].cpu().numpy().astype(np.int64), state[1][row].cpu().numpy()
                low, high = np.maximum(np.abs(x) - off, 0), np.abs(x) + off
                assert np.all((scales >= R.scales8(low)) & (scales <= R.scales8(high)))
                at, least = codes & 127, R.magnitudes8(low, dd, scales)
                if row == 1:
                    least = np.where(low > 0, np.maximum(least, 1), least)
                assert np.all((at >= least) & (at <= np.maximum(R.magnitudes8(high, dd, scales), (high > 0) & (row == 1))))
                assert np.all(((codes >> 7) == (x < 0)) | (np.abs(x) <= off))


@pytest.mark.parametrize("pd,gd,master", [(FP, FP, False), (BF, BF, True)], ids=str)
@pytest.mark.parametrize("bits", [32, 8])
def test_one_large_call_is_many_small_ones(opt, pd, gd, master, bits):
    """beyond the cache, and beyond what one launch takes"""
    sizes = [40_000_001, 31] + [1000 + 7 * k for k in range(300)]
    results = []
    for parts in (1, 2):
        params, grads = views(sizes, pd, 1, 0.1), views(sizes, gd, 2, 1e-2)
        state, weights = opt.adamw_state(params, bits), opt.master_weights(params) if master else None
        total = opt.padded_elements(params)
        if parts == 1:
            opt.adamw_step(params, grads, state, 3, master=weights)
        else:
            at = 0
            for p, g in zip(params, grads):
                n = -(-p.numel() // 32) * 32
                cut = [t[:, s:s + m].contiguous() for t, s, m in ([(state, at, n)] if bits == 32 else [(state[0], at, n), (state[1], at // 32, n // 32)])]
                w = weights[at:at + n].clone() if master else None
                opt.adamw_step([p], [g], cut[0] if bits == 32 else tuple(cut), 3, master=w)
                for t, c, s in zip([state] if bits == 32 else state, cut, (at, at // 32)):
                    t[:, s:s + c.shape[1]] = c
                if master:
                    weights[at:at + n] = w
                at += n
            assert at == total
        results.append([params[0], params[-1], torch.cat(params)] + ([state] if bits == 32 else list(state)) + ([weights] if master else []))
    assert all(torch.equal(a, b) for a, b in zip(*results))


@pytest.mark.parametrize("bits", [32, 8])
def test_zero_gradients_and_padding(opt, bits):
    """nothing moves a weight whose gradients are all zero, whatever lies in the arenas' gaps"""
    params = views([5, 40], FP, 1)
    state = opt.adamw_state(params, bits)
    tensors = [state] if bits == 32 else list(state)
    tensors[0][:, 5:32] = 99
    tensors[0][:, 72:] = 99
    was = [p.clone() for p in params]
    opt.adamw_step(params, [torch.zeros_like(p) for p in params], state, 1, weight_decay=0.0)
    assert all(torch.equal(p, w) for p, w in zip(params, was))
    assert all(int((t != 0).sum()) == 0 for t in tensors)


@pytest.mark.parametrize("size", [1e-30, 1e-20, 1e-10, 1e10, 1e15, 1e19])
@pytest.mark.parametrize("eps", [1e-8, 0.0])
def test_extreme_sizes(opt, size, eps):
    """moments at both ends of binary32, beside ordinary ones and zeros"""
    n, t = 4096, 3
    g = torch.randn(n, device=DEV)
    g[1::2] *= size
    g[::64] = 0
    p, state = torch.randn(n, device=DEV), opt.adamw_state([g])
    p0, g0 = p.double().cpu().numpy(), g.double().cpu().numpy()
    opt.adamw_step([p], [g], state, t, lr=1e-2, eps=eps, weight_decay=0.0)
    m, v = 0.1 * g0, 0.001 * g0 * g0
    got_m, got_v = state.double().cpu().numpy()
    # (1 - beta is rounded; a square below 2^-126 has fewer bits, to a half step of 2^-149, and one of 2^128 and more is infinite in binary32)
    beyond = g0 * g0 >= 2.0 ** 128
    assert np.all(np.abs(got_m - m) <= 4 * 2.0 ** -24 * np.abs(m)) and np.all(np.isinf(got_v[beyond]))
    assert np.all((np.abs(got_v - v) <= 6 * 2.0 ** -24 * v + 2.0 ** -149)[~beyond])
    # the step from the moments as they were stored, which carry the loss of small squares
    under = np.sqrt(got_v / (1 - 0.999 ** t)) + eps
    with np.errstate(all="ignore"):
        step = 1e-2 * (got_m / (1 - 0.9 ** t)) / under
    got = p.double().cpu().numpy()
    fine = np.isfinite(step)
    assert np.all(np.abs(got - (p0 - step))[fine] <= (2 * np.abs(p0) + 14 * np.abs(step))[fine] * 2.0 ** -24)
    assert np.all(np.isfinite(got[fine]))
    assert np.array_equal(np.isnan(got), np.isnan(step))          # 0 / 0 with eps 0


def test_small_roots_do_not_vanish(opt):
    """a root that is 2^-20 of its block's largest keeps the step bounded: |m| / r is at most what it is for the smallest code"""
    p, g = torch.zeros(32, device=DEV), torch.full((32,), 2.0 ** -20, device=DEV)
    g[0] = 1.0
    state = opt.adamw_state([p], 8)
    for t in range(1, 50):
        was = p.clone()
        opt.adamw_step([p], [g if t == 1 else torch.zeros_like(g)], state, t, lr=1.0, weight_decay=0.0)
        # m <= 2^-9 of a scale that is at most 1/448 * 2 of the block's largest, 0.1, or decays; r >= 2^-9 / 448 of 0.0316: their ratio is below 2 * 2 * 3.17, the
        # corrections' ratio sqrt(1 - 0.999^t) / (1 - 0.9^t) below 1
        assert float((p - was).abs().max()) <= 13.0
    assert int((state[0][1] == 0).sum()) == 0


@pytest.mark.parametrize("bits", [32, 8])
def test_skipped_and_missing(opt, bits):
    params, grads = views([100, 50], FP, 1), views([100, 50], FP, 2)
    state = opt.adamw_state(params, bits)
    opt.adamw_step(params, grads, state, 1)
    was = [p.clone() for p in params], [t.clone() for t in (state if bits == 8 else [state])]
    for bad in (float("nan"), float("inf"), -float("inf")):
        opt.adamw_step(params, grads, state, 2, grad_scale=torch.full((1,), bad, device=DEV))
    assert all(torch.equal(p, w) for p, w in zip(params, was[0])) and all(torch.equal(t, w) for t, w in zip(state if bits == 8 else [state], was[1]))
    opt.adamw_step(params, [None, grads[1]], state, 2)
    assert torch.equal(params[0], was[0][0]) and not torch.equal(params[1], was[0][1])
    now = state[0] if bits == 8 else state
    assert torch.equal(now[:, :128], was[1][0][:, :128]) and not torch.equal(now[:, 128:], was[1][0][:, 128:])


def test_gradients_that_are_not_numbers(opt):
    """as in 32 bits they make their weights NaN; in 8 the whole block"""
    for bits, bad in ((32, float("nan")), (8, float("nan")), (8, float("inf"))):
        p, g = torch.ones(96, device=DEV), torch.ones(96, device=DEV)
        g[40] = bad
        state = opt.adamw_state([p], bits)
        opt.adamw_step([p], [g], state, 1)
        opt.adamw_step([p], [torch.ones_like(g)], state, 2)
        gone = torch.isnan(p).nonzero().flatten().tolist()
        assert gone == ([40] if bits == 32 else list(range(32, 64)))


def test_step_refusals(opt):
    p, g = torch.ones(64, device=DEV), torch.ones(64, device=DEV)
    s32, s8 = opt.adamw_state([p]), opt.adamw_state([p], 8)
    for args, kw, text in ((([p], [g, g], s32, 1), {}, "as many gradients"), (([p], [g[:32]], s32, 1), {}, "as many elements"),
                           (([p, p], [g, g], opt.adamw_state([p, p]), 1), {}, "share memory"), (([p, p[32:]], [g, g[32:]], opt.adamw_state([p, p[32:]]), 1), {}, "share memory"),
                           (([p[:10]], [g[:10]], s32, 1), {}, "other parameters"), (([p], [g], s32.to(torch.uint8), 1), {}, "float32"),
                           (([p], [g], (s32, s8[1]), 1), {}, "uint8"), (([p], [g], (s8[0], s8[1][:, :1].contiguous()), 1), {}, "scales"),
                           (([p], [g], s32, 0), {}, "counts from 1"), (([p], [g], s32, 1), dict(betas=(1.0, 0.9)), "beta"), (([p], [g], s32, 1), dict(lr=float("nan")), "lr"),
                           (([p], [g], s32, 1), dict(master=torch.zeros(64, device=DEV)), "16-bit"), (([p.half()], [g], s32, 1), dict(master=torch.zeros(32, device=DEV)), "master"),
                           (([p], [g.double()], s32, 1), {}, "unsupported element dtype"), (([p], [torch.ones(128, device=DEV)[::2]], s32, 1), {}, "contiguous"),
                           (([], [], torch.zeros(2, 0, device=DEV), 1), {}, None)):
        was = p.clone()
        if text is None:
            opt.adamw_step(*args, **kw)
            continue
        with pytest.raises(RuntimeError, match=text):
            opt.adamw_step(*args, **kw)
        assert torch.equal(p, was)


def test_versions_move(opt):
    """autograd notices that a weight it has saved was changed"""
    w, x = torch.ones(3, device=DEV, requires_grad=True), torch.ones(3, device=DEV, requires_grad=True)
    y = (w * x).sum()
    with torch.no_grad():
        opt.adamw_step([w], [torch.ones(3, device=DEV)], opt.adamw_state([w]), 1)
    with pytest.raises(RuntimeError, match="modified by an inplace operation"):
        y.backward()


@pytest.mark.parametrize("bits", [32, 8])
def test_object(opt, bits):
    """the object's steps are the operator's, and go on after load_state_dict()"""
    def model():
        params = [p.clone().requires_grad_() for p in views([1000, 33], FP, 1) + views([257, 64], BF, 2)]
        return params, opt.AdamW([{"params": params[:3]}, {"params": params[3:], "weight_decay": 0.0, "lr": 1e-2}], lr=1e-3, bits=bits)
    params, a = model()
    states = [opt.adamw_state(params[:2], bits), opt.adamw_state(params[2:3], bits), opt.adamw_state(params[3:], bits)]
    mine = [p.detach().clone() for p in params]
    masters = [None, opt.master_weights(mine[2:3]), opt.master_weights(mine[3:])]
    saved = None
    for t in range(1, 5):
        grads = [torch.randn_like(p) for p in params]
        for p, g in zip(params, grads):
            p.grad = g
        if t == 3:
            saved = a.state_dict(), [p.detach().clone() for p in params]
        clip = opt.grad_norm(grads, 1.0, work=a.work)
        a.step(grad_scale=clip[1:])
        for part, (lo, hi, lr, wd) in enumerate(((0, 2, 1e-3, 1e-2), (2, 3, 1e-3, 1e-2), (3, 4, 1e-2, 0.0))):
            opt.adamw_step(mine[lo:hi], grads[lo:hi], states[part], t, lr=lr, weight_decay=wd, master=masters[part], grad_scale=clip[1:])
        assert all(torch.equal(p, q) for p, q in zip(params, mine))
        if t >= 3:
            again = again if t > 3 else model()
            if t == 3:
                again[1].load_state_dict(saved[0])
                for p, q in zip(again[0], saved[1]):
                    p.data.copy_(q)
            for p, g in zip(again[0], grads):
                p.grad = g
            again[1].step(grad_scale=clip[1:])
            assert all(torch.equal(p, q) for p, q in zip(params, again[0]))
    a.zero_grad()
    assert all(p.grad is None for p in params)


@pytest.mark.parametrize("bits", [32, 8])
def test_recorded_steps(opt, bits):
    """a recorded step counts on, reads the learning rate when it runs, and does not count what it skips"""
    sizes = [1000, 77]
    params, mine = ([p.clone() for p in views(sizes, BF, 1)] for _ in range(2))
    grads = views(sizes, BF, 2)
    lr, scale = torch.full((1,), 1e-2, device=DEV), torch.ones(1, device=DEV)
    a = opt.AdamW(params, lr=lr, bits=bits, capturable=True)
    b = opt.AdamW(mine, lr=1e-2, bits=bits)
    work, norm = opt.norm_work(DEV), torch.zeros(2, device=DEV)
    for p, q, g in zip(params, mine, grads):
        p.grad, q.grad = g, g
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        a.step(grad_scale=scale)
    torch.cuda.current_stream().wait_stream(side)
    b.step(grad_scale=scale)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        opt.grad_norm(grads, 1.0, work=work, out=norm)
        a.step(grad_scale=scale)
    for k in range(6):
        for g in grads:
            g.copy_(torch.randn(g.numel(), device=DEV) * (k + 1))
        lr.fill_(1e-2 / (k + 1))
        b.param_groups[0]["lr"] = float(lr)
        scale.fill_(float("nan") if k == 2 else 0.5)
        graph.replay()
        if k != 2:
            b.step(grad_scale=scale)
        torch.cuda.synchronize()
        assert torch.equal(norm, opt.grad_norm(grads, 1.0))
        assert a._steps.tolist() == [b.steps]
        # the device's pow may differ from the host's in the last place of a binary64: the factors are the same binary32 numbers but for a tie
        for p, q in zip(params, mine):
            assert torch.allclose(p.float(), q.float(), rtol=2.0 ** -7, atol=1e-6)
        for x, y in zip(a._parts[0]["state"] if bits == 8 else [a._parts[0]["state"]], b._parts[0]["state"] if bits == 8 else [b._parts[0]["state"]]):
            assert torch.equal(x, y)


def test_other_streams(opt):
    """work goes to the current stream, behind what is on it"""
    params = views([1 << 20], FP, 1)
    want = [p.clone() for p in params]
    grads, state, state2 = [torch.zeros(1 << 20, device=DEV)], opt.adamw_state(params), opt.adamw_state(params)
    new = torch.randn(1 << 20, device=DEV)
    torch.cuda.synchronize()
    side = torch.cuda.Stream()
    with torch.cuda.stream(side):
        torch.cuda._sleep(20_000_000)
        grads[0].copy_(new)
        norm = opt.grad_norm(grads, 1.0)
        opt.adamw_step(params, grads, state, 1, grad_scale=norm[1:])
    torch.cuda.synchronize()
    opt.adamw_step(want, [new], state2, 1, grad_scale=opt.grad_norm([new], 1.0)[1:])
    assert torch.equal(params[0], want[0]) and torch.equal(state, state2)


@pytest.mark.parametrize("bits", [32, 8])
def test_skipped_steps_are_not_counted(opt, bits):
    """a step that its factor makes do nothing leaves the count where it is, recorded or not, with or without factors before it, and across load_state_dict()"""
    def model(**kw):
        params = [p.clone() for p in views([1000, 77], FP, 1) + views([300], BF, 2)]
        return params, opt.AdamW([{"params": params[:2]}, {"params": params[2:], "lr": 1e-2}], lr=1e-3, bits=bits, **kw)
    fine, bad = torch.full((1,), 0.5, device=DEV), torch.full((1,), float("nan"), device=DEV)
    scales = [None, bad, fine, bad, torch.full((1,), float("inf"), device=DEV), None, fine]
    (p, eager), (q, device), (r, only) = model(), model(capturable=True), model()
    done = 0
    for t, scale in enumerate(scales):
        grads = [torch.randn_like(v) for v in p]
        for params in (p, q, r):
            for v, g in zip(params, grads):
                v.grad = g.clone()
        if t == 4:                                    # the count goes with the state
            saved = eager.state_dict()
            again = model()
            for v, u in zip(again[0], p):
                v.copy_(u)
            again[1].load_state_dict(saved)
            for v, g in zip(again[0], grads):
                v.grad = g.clone()
            p, eager = again
        eager.step(grad_scale=scale)
        device.step(grad_scale=scale)
        if scale is None or bool(torch.isfinite(scale)):
            only.step(grad_scale=scale)               # the steps that count, alone
            done += 1
        assert eager.steps == device.steps == only.steps == done
        for a, b, c in zip(p, q, r):
            assert torch.equal(a, c) and torch.equal(b, c)
        for x, y, z in zip(eager._parts, device._parts, only._parts):
            for a, b, c in zip(*((s["state"] if bits == 8 else [s["state"]]) for s in (x, y, z))):
                assert torch.equal(a, c) and torch.equal(b, c)


def test_norm_of_gradients_that_are_missing(opt):
    """None takes no part, and what AdamW.step() takes grad_norm(AdamW.grads()) takes"""
    params = [torch.ones(40, 30, device=DEV), torch.ones(7, device=DEV), torch.ones(64, device=DEV), torch.ones(3, device=DEV)]
    a = opt.AdamW(params, lr=1e-2)
    params[0].grad = torch.randn(30, 40, device=DEV).t()
    params[2].grad = torch.randn(64, device=DEV)
    norm = math.sqrt(float(params[0].grad.double().square().sum() + params[2].grad.double().square().sum()))
    got = opt.grad_norm([None, params[2].grad, None, params[0].grad.contiguous()], 1.0)
    assert abs(float(got[0]) - norm) <= norm * 2.0 ** -23
    clip = opt.grad_norm(a.grads(), 1.0, work=a.work)
    assert abs(float(clip[0]) - norm) <= norm * 2.0 ** -23
    was = [p.clone() for p in params]
    a.step(grad_scale=clip[1:])
    assert [torch.equal(p, w) for p, w in zip(params, was)] == [False, True, False, True]
    a.zero_grad()
    assert opt.grad_norm(a.grads(), 1.0, work=a.work).tolist() == [0.0, 1.0]
    with pytest.raises(RuntimeError, match="no tensors"):
        opt.grad_norm(a.grads(), 1.0)


def test_loaded_learning_rates_are_ones_own(opt):
    """a learning rate on the device that load_state_dict() brings is a copy, on the parameters' device"""
    def model(lr):
        p = torch.ones(10, device=DEV)
        p.grad = torch.ones(10, device=DEV)
        return opt.AdamW([p], lr=lr, capturable=True)
    a = model(torch.full((1,), 0.25, device=DEV))
    saved = a.state_dict()
    for state in (saved, {**saved, "groups": [{**saved["groups"][0], "lr": saved["groups"][0]["lr"].cpu()}]}):
        b, c = model(0.1), model(0.1)
        b.load_state_dict(state)
        c.load_state_dict(state)
        b.param_groups[0]["lr"].fill_(7.0)
        c.step()
        assert float(c.param_groups[0]["lr"]) == 0.25 and float(state["groups"][0]["lr"]) == 0.25
