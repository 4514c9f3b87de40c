"""4-bit microscaled matrices against their definition (ref_operators.py): bytes to the bit, products in 64 bits."""
import math

import numpy as np
import pytest
import torch

import ref_operators as R

pytestmark = pytest.mark.gpu
DEV = "cuda:0"
BF, HF, FP = torch.bfloat16, torch.float16, torch.float32


@pytest.fixture(scope="module")
def ms(capi):
    from dynamiq_sigcomm_artifact_amd import microscale
    return microscale


def matrix(r, c, dtype, seed=0, spread=3.0):
    g = torch.Generator(device=DEV).manual_seed(seed)
    x = torch.randn(r, c, generator=g, device=DEV) * torch.exp(spread * torch.randn(r, c, generator=g, device=DEV))
    return x.clamp(-6e4, 6e4).to(dtype)


def signs(capi, n, seed):
    bits = torch.empty(-(-n // 256) * 8, dtype=torch.int32, device=DEV)
    capi.rand_diag_bits(bits, bits.numel() * 32, seed)
    s = 1.0 - 2.0 * ((bits.cpu().numpy().view(np.uint32)[:, None] >> np.arange(32)) & 1).reshape(-1)
    return bits, s


def pool(rows, n, dtype, seed=5):
    g = torch.Generator(device=DEV).manual_seed(seed)
    return torch.rand(rows, -(-n // 256) * 256, generator=g, device=DEV).mul_(0.99).to(dtype)


def same(q, values, scales):
    assert np.array_equal(q.scales.cpu().numpy(), scales)
    live = np.repeat(scales, 32, axis=1) != 255
    got = R.unpack4(q.codes.cpu().numpy(), scales)
    assert np.array_equal(got[live], values[live])


SHAPES = [(1, 1), (1, 32), (3, 31), (5, 33), (7, 256), (130, 257), (129, 300), (257, 131), (64, 1000)]


@pytest.mark.parametrize("r,c", SHAPES)
@pytest.mark.parametrize("columns", [False, True])
@pytest.mark.parametrize("dtype", [FP, BF, HF], ids=str)
def test_nearest(ms, r, c, columns, dtype):
    x = matrix(r, c, dtype, r + c)
    q = ms.quantize(x, columns=columns)
    assert q.shape == ((c, r) if columns else (r, c))
    v = x.float().cpu().numpy()
    values, scales = R.quantize4(v.T if columns else v)
    same(q, values, scales)
    for out in (FP, BF, HF):
        got = ms.dequantize(q, out)
        want = torch.from_numpy(values[:, :q.cols]).to(out)          # one rounding, of a value with two significant bits
        assert torch.equal(got.cpu(), want)


@pytest.mark.parametrize("r,c", [(3, 31), (130, 257), (257, 131)])
@pytest.mark.parametrize("columns", [False, True])
@pytest.mark.parametrize("rotate", [False, True])
@pytest.mark.parametrize("source", [FP, BF, HF, "philox"], ids=str)
def test_stochastic_and_rotated(ms, capi, r, c, columns, rotate, source):
    dtype = BF if rotate else FP
    x = matrix(r, c, dtype, 7)
    rows, n = (c, r) if columns else (r, c)
    bits, s = signs(capi, n, 11) if rotate else (None, None)
    if source == "philox":
        q = ms.quantize(x, columns, bits, seed=123, step=9)
        u = torch.empty(rows * (-(-n // 256) * 256), dtype=FP, device=DEV)
        capi.philox_uniform(u, 123, 9)
    else:
        u = pool(rows, n, source)
        q = ms.quantize(x, columns, bits, rand_pool=u)
    v = x.float().cpu().numpy()
    same(q, *R.quantize4(v.T if columns else v, s, u.float().cpu().numpy()))


@pytest.mark.parametrize("columns", [False, True])
def test_rotation_to_nearest(ms, capi, columns):
    x = matrix(100, 300, FP, 3, spread=1.0)
    n = 100 if columns else 300
    bits, s = signs(capi, n, 4)
    v = x.cpu().numpy()
    same(ms.quantize(x, columns, bits), *R.quantize4(v.T if columns else v, s))


@pytest.mark.parametrize("columns", [False, True])
def test_borders(ms, columns):
    """ties, saturation, subnormal numbers, the largest and smallest scales, blocks of zeros"""
    halves = np.concatenate([np.arange(0, 33) / 4.0, -np.arange(0, 33) / 4.0, np.nextafter(np.float32([0.25, 0.75, 1.25, 1.75, 2.5, 3.5, 5.0]), np.float32(9)),
                             np.nextafter(np.float32([0.25, 0.75, 1.25, 1.75, 2.5, 3.5, 5.0]), np.float32(0))]).astype(np.float32)
    rows = []
    for k in (0, 1, -1, 100, -100, 124, -126, -130, -140, -149):
        for top in (4.0, 6.0, 7.999, 7.0):
            with np.errstate(all="ignore"):
                for at in range(0, len(halves), 31):
                    b = np.zeros(32, np.float32)
                    part = halves[at:at + 31]
                    b[:len(part)] = np.clip(part, -top, top)
                    b[31] = top
                    rows.append(np.ldexp(b, k).astype(np.float32))
    rows.append(np.zeros(32, np.float32))
    rows.append(np.full(32, 1e-45, np.float32))
    rows.append(np.full(32, np.finfo(np.float32).max))
    x = np.concatenate(rows).reshape(1, -1)
    x[~np.isfinite(x)] = 1.0
    t = torch.from_numpy(x).to(DEV)
    q = ms.quantize(t.t().contiguous() if columns else t, columns)
    same(q, *R.quantize4(x))
    u = np.full((1, -(-x.shape[1] // 256) * 256), 0.5, np.float32)
    q = ms.quantize(t.t().contiguous() if columns else t, columns, rand_pool=torch.from_numpy(u).to(DEV))
    same(q, *R.quantize4(x, None, u))


@pytest.mark.parametrize("columns", [False, True])
@pytest.mark.parametrize("bad", [float("inf"), -float("inf"), float("nan")])
def test_what_is_not_finite(ms, columns, bad):
    """its block is NaN, and so is every product with it, and nothing else"""
    x = torch.ones(70, 300, device=DEV)
    x[33, 40] = bad
    for kw in (dict(), dict(seed=1)):
        q = ms.quantize(x, columns, **kw)
        rows, n = q.shape
        row, at = (40, 33) if columns else (33, 40)
        values = ms.dequantize(q)
        nan = torch.zeros(rows, n, dtype=torch.bool, device=DEV)
        nan[row, at // 32 * 32:min(n, at // 32 * 32 + 32)] = True
        assert torch.equal(torch.isnan(values), nan)
        y = ms.product(q, ms.quantize(torch.zeros(5, n, device=DEV)), FP)
        assert torch.isnan(y[row]).all() and int(torch.isnan(y).sum()) == 5
        y = ms.product(ms.quantize(torch.ones(40, n, device=DEV)), q, FP)
        assert torch.isnan(y[:, row]).all() and int(torch.isnan(y).sum()) == 40


def test_views(ms):
    """rows apart, and elements at any address"""
    big = matrix(40, 1001, BF, 1)
    for x in (big[:, 3:600], big[5:6, 1:], big[::2, 7:8], big[3:, :]):
        for columns in (False, True):
            q, w = ms.quantize(x, columns), ms.quantize(x.clone(memory_format=torch.contiguous_format), columns)
            assert torch.equal(q.codes, w.codes) and torch.equal(q.scales, w.scales)
    with pytest.raises(RuntimeError, match="consecutive"):
        ms.quantize(big.t())
    with pytest.raises(RuntimeError, match="consecutive"):
        ms.quantize(big[:1].expand(4, 1001))
    with pytest.raises(RuntimeError, match="a matrix is required"):
        ms.quantize(big[0])


def test_refusals(ms, capi):
    x = matrix(4, 300, BF)
    with pytest.raises(RuntimeError, match="unsupported element dtype"):
        ms.quantize(x.double())
    with pytest.raises(RuntimeError, match="sign: wrong dtype or too few"):
        ms.quantize(x, sign=torch.zeros(15, dtype=torch.int32, device=DEV))
    with pytest.raises(RuntimeError, match="rand_pool has one value"):
        ms.quantize(x, rand_pool=torch.zeros(4, 300, device=DEV))
    with pytest.raises(RuntimeError, match="not both"):
        ms.quantize(x, rand_pool=torch.zeros(4, 512, device=DEV), seed=1)
    with pytest.raises(RuntimeError, match="unsupported element dtype"):
        ms.quantize(x, rand_pool=torch.zeros(4, 512, dtype=torch.uint8, device=DEV))
    q = ms.quantize(x)
    with pytest.raises(RuntimeError, match="do not belong"):
        ms.dequantize(ms.Microscaled(q.codes, q.scales, 4, 700))
    with pytest.raises(RuntimeError, match="do not belong"):
        ms.product(q, ms.Microscaled(q.codes, q.scales, 5, 300))
    with pytest.raises(RuntimeError, match="uint8"):
        ms.dequantize(ms.Microscaled(q.codes.int(), q.scales, 4, 300))
    with pytest.raises(RuntimeError, match="contiguous"):
        ms.dequantize(ms.Microscaled(torch.zeros(4, 512, dtype=torch.uint8, device=DEV)[:, ::2], q.scales, 4, 300))


def test_empty(ms):
    x = torch.ones(3, 40, device=DEV)
    none = ms.quantize(x[:0])
    assert none.shape == (0, 40) and ms.dequantize(none).shape == (0, 40)
    assert ms.product(none, ms.quantize(x)).shape == (0, 3) and ms.product(ms.quantize(x), none).shape == (3, 0)
    flat = ms.quantize(x[:, :0])
    assert torch.equal(ms.product(flat, flat, FP), torch.zeros(3, 3, device=DEV))


# ---- products ----

def packed(ms, r, n, seed):
    """a matrix of all codes and many scales, and its values"""
    rng = np.random.default_rng(seed)
    values, scales = R.quantize4(rng.standard_normal((r, n)) * np.exp(rng.standard_normal((r, n))))
    return ms.Microscaled(torch.from_numpy(R.pack4(values, scales)).to(DEV), torch.from_numpy(scales).to(DEV), r, n), values[:, :n]


PRODUCTS = [(1, 1, 1), (1, 16, 256), (1, 1000, 4096), (2, 33, 31), (3, 17, 4000), (15, 64, 512), (16, 100, 768), (17, 48, 300), (31, 129, 1024), (33, 255, 513), (64, 64, 64),
            (65, 130, 2048), (100, 1, 777), (127, 129, 255), (128, 128, 1024), (129, 257, 2304), (256, 256, 256), (300, 500, 4100), (513, 1030, 1500), (1025, 777, 300),
            # every kernel that sizes choose: few rows and columns of each kind, tiles of 128 and of 256, their last rows and columns
            (5, 3100, 600), (16, 12300, 257), (20, 13000, 300), (33, 5000, 520), (40, 20000, 260), (1000, 40, 300), (3000, 70, 1111), (20000, 9, 300), (129, 12801, 300),
            (1, 12400, 300), (8, 6200, 520), (9, 3100, 300), (1300, 1281, 900), (2000, 2049, 513), (4097, 3300, 256), (4100, 3200, 1025), (2049, 7000, 100),
            # scales come for four superchunks at a time, and of odd numbers of them the last row's end early: one to nine of them, in tiles of 128 and of 256
            (700, 900, 200), (701, 899, 700), (702, 898, 1100), (703, 897, 1281), (640, 1000, 1793), (641, 1001, 2049), (2900, 3000, 250), (2901, 2999, 512), (2817, 3001, 600),
            (2818, 2990, 1280), (2819, 3011, 1537),
            # a last round that is cut, along either side
            (4100, 4200, 2049), (4400, 4090, 1900)]


@pytest.mark.parametrize("m,n,k", PRODUCTS)
def test_product(ms, m, n, k):
    a, x = packed(ms, m, k, m + k)
    b, y = packed(ms, n, k, n)
    want, size = x @ y.T, np.abs(x) @ np.abs(y).T
    # products of two E2M1 numbers and two powers of two are exact; k additions in binary32, in whatever order, are off by k half steps of the sum of magnitudes at most
    # (the matrix core may cut instead of rounding: a whole step each)
    bound = k * 2.0 ** -23 * size
    for dtype in (FP, BF, HF):
        got = ms.product(a, b, dtype).double().cpu().numpy()
        err = bound + (torch.finfo(dtype).eps / 2 * (np.abs(want) + bound) + (2.0 ** -25 if dtype == HF else 0) if dtype != FP else 0)
        assert np.all(np.abs(got - want) <= err), float(np.max(np.abs(got - want) - err))


def test_exact_sums(ms):
    """small whole numbers: every sum is exact, so every element must be right to the bit"""
    for m, n, k in ((1, 300, 1000), (20, 70, 512), (140, 300, 1111), (600, 520, 256)):
        rng = np.random.default_rng(k)
        x, y = rng.integers(-4, 5, (m, k)).astype(np.float32), rng.integers(-4, 5, (n, k)).astype(np.float32)
        x[:, ::32], y[:, ::32] = 4, 4                       # no block's largest below 4: scale 1
        got = ms.product(ms.quantize(torch.from_numpy(x).to(DEV)), ms.quantize(torch.from_numpy(y).to(DEV)), FP)
        assert np.array_equal(got.cpu().numpy(), x @ y.T)


def test_scales_of_the_product(ms):
    """the extreme scales, and each of a row's"""
    x = torch.ones(40, 512, device=DEV) * torch.exp2(torch.arange(16, device=DEV).repeat_interleave(32).float() - 8)
    y = torch.ones(24, 512, device=DEV) * torch.exp2(-2.0 * torch.arange(16, device=DEV).repeat_interleave(32).float() + 3)
    got = ms.product(ms.quantize(x), ms.quantize(y), FP)
    assert torch.equal(got, (x.double() @ y.double().t()).float())
    # (2^-149 is below a quarter of the smallest scale, 2^-127: a zero; 2^-128 is half of it)
    for a, b, want in ((2.0 ** 120, 2.0 ** -120, 256.0), (2.0 ** -126, 2.0 ** 100, 2.0 ** -18), (2.0 ** -128, 2.0 ** 126, 64.0), (2.0 ** -149, 2.0 ** 126, 0.0)):
        got = ms.product(ms.quantize(torch.full((33, 256), a, device=DEV)), ms.quantize(torch.full((20, 256), b, device=DEV)), FP)
        assert torch.equal(got, torch.full_like(got, want))


def test_order_does_not_change(ms):
    a, _ = packed(ms, 100, 3000, 1)
    b, _ = packed(ms, 200, 3000, 2)
    first = ms.product(a, b, FP)
    assert all(torch.equal(ms.product(a, b, FP), first) for _ in range(5))


# ---- the layer ----

def plain_linear(x, w, dy, sn, sm, pr, pc):
    q = lambda t, s=None, u=None: R.quantize4(t, s, u)[0]          # noqa: E731
    f = lambda t: t.float().cpu().numpy()                          # noqa: E731
    k, n, m = x.shape[1], w.shape[0], x.shape[0]
    y = q(f(x)) @ q(f(w)).T
    dx = q(f(dy), sn, None if pr is None else f(pr)) @ q(f(w).T, sn).T
    dw = q(f(dy).T, sm, None if pc is None else f(pc)) @ q(f(x).T, sm).T
    return y, dx[:, :k], dw[:, :k]


@pytest.mark.parametrize("m,n,k", [(1, 40, 64), (70, 33, 300), (300, 257, 96)])
@pytest.mark.parametrize("rotate,rounding", [(False, "nearest"), (True, "pool"), (True, "philox")])
@pytest.mark.parametrize("dtype", [BF, FP], ids=str)
def test_linear(ms, capi, m, n, k, rotate, rounding, dtype):
    x, w, dy = matrix(m, k, dtype, 1, 1.0).requires_grad_(), matrix(n, k, dtype, 2, 1.0).requires_grad_(), matrix(m, n, dtype, 3, 1.0)
    (bn, sn), (bm, sm) = (signs(capi, n, 5), signs(capi, m, 6)) if rotate else ((None, None),) * 2
    pools = (pool(m, n, BF, 1), pool(n, m, BF, 2)) if rounding == "pool" else None
    kw = dict(seed=77, step=3) if rounding == "philox" else {}
    y = ms.linear(x, w, sign=(bn, bm) if rotate else None, rand_pool=pools, **kw)
    y.backward(dy)
    if rounding == "philox":
        pools = tuple(torch.empty(r, -(-c // 256) * 256, device=DEV) for r, c in ((m, n), (n, m)))
        capi.philox_uniform(pools[0], 77, 3)
        capi.philox_uniform(pools[1], 77, 3 + (1 << 63))
    want = plain_linear(x.detach(), w.detach(), dy, sn, sm, *(pools or (None, None)))
    for got, t, length in ((y, want[0], k), (x.grad, want[1], n), (w.grad, want[2], m)):
        assert got.dtype == dtype
        g = got.detach().double().cpu().numpy()
        # as in test_product, with the operands' magnitudes bounded by their norms
        size = np.abs(t).max() * 4 + 1e-30
        assert np.all(np.abs(g - t) <= torch.finfo(dtype).eps / 2 * np.abs(t) + length * 2.0 ** -23 * size * 8)


def test_linear_shapes_and_partial_gradients(ms):
    x, w = matrix(12, 64, BF, 1).view(3, 4, 64), matrix(10, 64, BF, 2)
    y = ms.linear(x, w)
    assert y.shape == (3, 4, 10) and torch.equal(y.view(12, 10), ms.product(ms.quantize(x.view(12, 64)), ms.quantize(w)))
    wg = w.clone().requires_grad_()
    ms.linear(x, wg).sum().backward()                       # an expanded gradient
    assert wg.grad.shape == (10, 64)
    xg = x.clone().requires_grad_()
    ms.linear(xg, w, seed=1).float().square().sum().backward()
    assert xg.grad.shape == x.shape
    assert ms.linear(x.transpose(0, 1), w).shape == (4, 3, 10)


def test_linear_refusals_and_empty(ms):
    x, w = matrix(6, 64, BF, 1), matrix(10, 64, BF, 2)
    for args, kw, text in (((x, w[:, :32]), {}, "weight"), ((x, w[0]), {}, "weight"), ((x.double(), w), {}, "unsupported element dtype"), ((x.cpu(), w), {}, "live on the GPU"),
                           ((x, w.cpu()), {}, "different devices"), ((x, None), {}, "a tensor argument"), ((x, w), dict(rand_pool=(pool(6, 10, BF), pool(10, 6, BF)), seed=1), "not both")):
        with pytest.raises(RuntimeError, match=text):
            ms.linear(*args, **kw)
    xg = x.clone().requires_grad_()
    for kw, text in ((dict(sign=(torch.zeros(4, dtype=torch.int32, device=DEV), None)), "signs are int32"), (dict(rand_pool=(torch.zeros(6, 10, device=DEV), None)), "rand_pool has one value")):
        with pytest.raises(RuntimeError, match=text):
            ms.linear(xg, w, **kw).sum().backward()
    y = ms.linear(xg, w)
    with pytest.raises(RuntimeError, match="cannot be differentiated again"):
        torch.autograd.grad(y.sum(), xg, create_graph=True)
    for shape in ((0, 64), (2, 0, 64)):
        e, v = torch.zeros(shape, dtype=BF, device=DEV, requires_grad=True), w.clone().requires_grad_()
        y = ms.linear(e, v)
        assert y.shape == shape[:-1] + (10,)
        y.sum().backward()
        assert e.grad.shape == shape and int((v.grad != 0).sum()) == 0
    assert ms.linear(x[0], w).shape == (10,)
    y = ms.linear(torch.zeros(3, 0, device=DEV), torch.zeros(5, 0, device=DEV))
    assert y.shape == (3, 5) and int((y != 0).sum()) == 0
    big = matrix(6, 128, BF, 3)                              # rows apart, and a transposed weight
    assert torch.equal(ms.linear(big[:, :64], w.t().contiguous().t()), ms.linear(big[:, :64].contiguous(), w))


def test_gradients_against_differences(ms):
    """with operands that 4 bits hold exactly, the layer is the plain product, and its gradients are its differences"""
    rng = np.random.default_rng(0)
    x0, w0 = (rng.integers(-2, 3, s).astype(np.float32) for s in ((8, 64), (32, 64)))
    c = rng.integers(-4, 5, (8, 32)).astype(np.float32)
    for t in (x0, w0, c):
        t[:, 0] = 4
    x0[0], w0[0], c[0] = 4, 4, 4
    x, w = (torch.from_numpy(t).to(DEV).requires_grad_() for t in (x0, w0))
    dy = torch.from_numpy(c).to(DEV)
    (ms.linear(x, w) * dy).sum().backward()
    value = lambda a, b: float((ms.linear(a, b) * dy).sum())       # noqa: E731
    with torch.no_grad():
        for i, j in ((1, 3), (7, 60), (2, 2), (5, 33)):
            a, b = x.clone(), w.clone()
            a[i, j], b[i, j] = 0, 0
            assert value(x, w) - value(a, w) == float(x[i, j] * x.grad[i, j])
            assert value(x, w) - value(x, b) == float(w[i, j] * w.grad[i, j])


def test_rounding_has_no_bias(ms):
    """the mean of many stochastic roundings is the value: 4096 draws, six standard deviations of half a step at most"""
    x = matrix(1, 256, FP, 1, 1.0)
    mean = sum(ms.dequantize(ms.quantize(x, seed=s)).double() for s in range(4096)) / 4096
    step = torch.exp2(ms.quantize(x, seed=0).scales.double().repeat_interleave(32, 1) - 127) * 2
    # a uniform value is a multiple of 1/256: half of that is the bias of one rounding at most
    assert torch.all((mean - x.double()).abs() <= step * (6 * 0.5 / 64 + 1 / 256))


def test_graph_and_streams(ms, capi):
    x, w = matrix(70, 512, BF, 1), matrix(300, 512, BF, 2)
    bits, _ = signs(capi, 70, 3)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        torch.cuda._sleep(5_000_000)
        x.mul_(2)
        y = ms.product(ms.quantize(x), ms.quantize(w))
    torch.cuda.current_stream().wait_stream(side)
    assert torch.equal(y, ms.product(ms.quantize(x), ms.quantize(w)))
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        q = ms.quantize(x, True, bits, seed=5, step=1)
        z = ms.product(ms.quantize(x), ms.quantize(w))
        values = ms.dequantize(q, BF)
    for k in range(4):
        x.copy_(matrix(70, 512, BF, 10 + k))
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(z, ms.product(ms.quantize(x), ms.quantize(w)))
        assert torch.equal(values, ms.dequantize(ms.quantize(x, True, bits, seed=5, step=1), BF))


def test_layer_in_a_graph(ms, capi):
    """forward and backward recorded together"""
    x0, w0, dy = matrix(40, 96, BF, 1, 1.0), matrix(50, 96, BF, 2, 1.0), matrix(40, 50, BF, 3, 1.0)
    x, w = x0.clone().requires_grad_(), w0.clone().requires_grad_()
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        torch.autograd.grad(ms.linear(x, w, seed=1, step=2), (x, w), dy)
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        y = ms.linear(x, w, seed=1, step=2)
        dx, dw = torch.autograd.grad(y, (x, w), dy)
    for k in range(3):
        with torch.no_grad():
            x.copy_(x0 * (k + 1))
        graph.replay()
        torch.cuda.synchronize()
        a, b = (x0 * (k + 1)).requires_grad_(), w0.clone().requires_grad_()
        e = ms.linear(a, b, seed=1, step=2)
        assert torch.equal(y, e) and all(torch.equal(s, t) for s, t in zip((dx, dw), torch.autograd.grad(e, (a, b), dy)))


def test_step_on_the_device(ms):
    """the random stream of a step in device memory is that of the number, also in a graph that is replayed with another one"""
    x, w, dy = matrix(40, 96, BF, 1, 1.0).requires_grad_(), matrix(50, 96, BF, 2, 1.0).requires_grad_(), matrix(40, 50, BF, 3, 1.0)
    step = torch.tensor([7], device=DEV)

    def layer(t):
        return torch.autograd.grad(ms.linear(x, w, seed=1, step=t), (x, w), dy)

    def same(a, b):
        return all(torch.equal(s, t) for s, t in zip(a, b))
    for columns in (False, True):
        assert torch.equal(ms.quantize(dy, columns, seed=3, step=step).codes, ms.quantize(dy, columns, seed=3, step=7).codes)
    assert same(layer(step), layer(7)) and not same(layer(7), layer(8))
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        layer(step)
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got = layer(step)
        step.add_(1)
    for t in (7, 8, 9):
        graph.replay()
        torch.cuda.synchronize()
        assert same(got, layer(t))
    y = ms.linear(x, w, seed=1, step=step)
    step.add_(1)                                            # the backward pass would draw other numbers than those of its step
    with pytest.raises(RuntimeError, match="modified by an inplace operation"):
        y.sum().backward()
    for bad in (torch.zeros(1, device=DEV), torch.zeros(1, dtype=torch.int64), torch.zeros(0, dtype=torch.int64, device=DEV)):
        with pytest.raises(RuntimeError):
            ms.linear(x, w, seed=1, step=bad)
        with pytest.raises(RuntimeError):
            ms.quantize(dy, seed=1, step=bad)


def test_list_is_one_after_the_other(ms, capi):
    """every kind of matrix in a list, in runs of one type and alternating, too large to share a launch, and the same matrix twice"""
    kinds = [(rows, columns, rotate, source) for rows in ((70, 300), (257, 513)) for columns in (False, True) for rotate in (False, True)
             for source in (None, "philox", FP, BF, HF)]
    entries = [(matrix(*kinds[k][0], dtype, k),) + kinds[k][1:] for dtype in (BF, FP, HF) for k in range(len(kinds))]
    entries += [(matrix(9000, 2100, BF, 1), True, False, None), (matrix(30000, 2100, HF, 2), False, False, None), (matrix(50, 40, HF, 3), False, False, None)]
    entries += [entries[0], entries[-1], entries[0], entries[7], entries[50], entries[3], entries[90]]
    step = torch.tensor([5], device=DEV)
    jobs, wants, held = [], [], []
    codes = {torch.float16: 0, torch.bfloat16: 1, torch.float32: 2}
    for k, (x, columns, rotate, source) in enumerate(entries):
        rows, length = (x.shape[1], x.shape[0]) if columns else x.shape
        sign = signs(capi, length, k)[0] if rotate else None
        drawn = pool(rows, length, source, k) if source not in (None, "philox") else None
        want = ms.quantize(x, columns, sign, drawn, **(dict(seed=k, step=5 + k) if source == "philox" else {}))
        out = torch.full_like(want.codes, 77), torch.full_like(want.scales, 77)
        jobs.append(capi.Mx4Matrix(x.data_ptr(), x.shape[0], x.shape[1], x.shape[1], None if sign is None else sign.data_ptr(), None if drawn is None else drawn.data_ptr(), k, k,
                                   step.data_ptr() if source == "philox" else None, out[0].data_ptr(), out[1].data_ptr(), codes[x.dtype], int(columns),
                                   int(source is not None), 0 if drawn is None else codes[drawn.dtype]))
        wants.append((want, out))
        held.append((x, sign, drawn))
    stream = torch.cuda.current_stream().cuda_stream
    assert capi.lib().dq_mx4_quantize_list((capi.Mx4Matrix * len(jobs))(*jobs), len(jobs), 0, stream) == 0
    for k, (want, out) in enumerate(wants):
        assert torch.equal(out[0], want.codes) and torch.equal(out[1], want.scales), (k, entries[k][1:], entries[k][0].shape)
    assert capi.lib().dq_mx4_quantize_list(None, 0, 0, stream) == 0


def test_recording_beside_a_living_graph_is_refused(ms):
    x, w, dy = matrix(40, 96, BF, 1, 1.0).requires_grad_(), matrix(50, 96, BF, 2, 1.0).requires_grad_(), matrix(40, 50, BF, 3, 1.0)
    side, graph = torch.cuda.Stream(), torch.cuda.CUDAGraph()

    def record():
        with torch.cuda.graph(graph, stream=side):
            return torch.autograd.grad(ms.linear(x, w, seed=1, step=2), (x, w), dy)
    alive = ms.linear(x, w)
    with pytest.raises(RuntimeError, match="still alive"):
        record()
    torch.cuda.synchronize()
    with torch.no_grad(), torch.cuda.graph(torch.cuda.CUDAGraph(), stream=side):
        ms.linear(x, w)                                     # no backward pass, nothing to refuse
    del alive
    graph = torch.cuda.CUDAGraph()
    got = record()
    for _ in range(2):
        graph.replay()
        torch.cuda.synchronize()
        want = torch.autograd.grad(ms.linear(x, w, seed=1, step=2), (x, w), dy)
        assert all(torch.equal(s, t) for s, t in zip(got, want))
        del want


# ---- what lies at the ends of a rotation, of a draw and of the layer's arguments ----

@pytest.mark.parametrize("columns", [False, True])
@pytest.mark.parametrize("dtype", [BF, FP], ids=str)
@pytest.mark.parametrize("rounding", ["nearest", "pool", "philox"])
def test_rotation_of_the_largest_numbers(ms, capi, columns, dtype, rounding):
    """a power of two in front of a matrix is one in its scales, also where the sums of 32 pass binary32's range; only beyond the largest scale is a block NaN"""
    top = 1.9921875 * 2.0 ** 9                            # the largest number of bf16, over 2^118
    x = matrix(70, 300, dtype, 5, spread=1.0).clamp(-top, top)
    x[:, 64:96] *= 2.0 ** -3
    x[:8] = torch.where(x[:8] < 0, -top, top).to(dtype)
    x[32:64, 128:160] = 0
    x[64:, 0:2] = 0
    rows, n = (300, 70) if columns else (70, 300)
    bits, s = signs(capi, n, 4)
    at = x.t() if columns else x
    at[0, :64] = torch.from_numpy(s[:64]).to(DEV).to(dtype) * top                             # 32 top / sqrt(32) is above 2^130 over 2^118: more than the largest scale holds
    at[1, :32] = torch.from_numpy(s[:32]).to(DEV).to(dtype) * 2.0 ** 9
    kw = dict(rand_pool=pool(rows, n, BF)) if rounding == "pool" else dict(seed=3, step=4) if rounding == "philox" else {}
    small, far = ms.quantize(x, columns, bits, **kw), ms.quantize(x * 2.0 ** 118, columns, bits, **kw)
    assert torch.isfinite(x * 2.0 ** 118).all()
    want = small.scales.int() + 118
    empty = ms.quantize(x, columns, bits).scales == 0
    want = torch.where(empty, 0, torch.where(want > 254, 255, want))
    assert (want[0, :2] == 255).all() and int(want[1, 0]) == 254
    assert torch.equal(far.scales.int(), want)
    live = (want != 255).repeat_interleave(16, 1)
    assert torch.equal(far.codes[live], small.codes[live])
    # and what a product makes of them: the same sums, 2^118 times
    one = ms.quantize(torch.full((3, n), 2.0 ** -100, device=DEV))
    a, b = ms.product(small, one, FP), ms.product(far, one, FP)
    gone = (want == 255).any(1)
    assert torch.equal(b[~gone], a[~gone] * 2.0 ** 118) and torch.isnan(b[gone]).all()


@pytest.mark.parametrize("bad", [float("inf"), float("nan")])
def test_rotation_beside_what_is_not_finite(ms, capi, bad):
    """in one row: a block with an infinity or NaN, a block of the largest numbers and ordinary ones"""
    x = matrix(6, 256, BF, 2, 1.0)
    bits, _ = signs(capi, 256, 4)
    want = ms.quantize(x, sign=bits)
    x[2, 40] = bad
    x[2, 64:96] *= 2.0 ** 100
    x[2, 70] = -2.0 ** 126
    got = ms.quantize(x, sign=bits)
    same_block = torch.ones(6, 8, dtype=torch.bool, device=DEV)
    same_block[2, 1:3] = False
    assert torch.equal(got.scales[same_block], want.scales[same_block]) and int(got.scales[2, 1]) == 255 and 245 <= int(got.scales[2, 2]) <= 254


def test_linear_refuses_before_its_backward_pass(ms):
    """what the backward pass would refuse is refused with the call, and only what it would take"""
    x, w = matrix(6, 64, BF, 1), matrix(10, 64, BF, 2)
    xg, wg = x.clone().requires_grad_(), w.clone().requires_grad_()
    short, good = torch.zeros(4, dtype=torch.int32, device=DEV), torch.zeros(8, dtype=torch.int32, device=DEV)
    rows, columns = torch.zeros(6, 256, device=DEV), torch.zeros(10, 256, device=DEV)
    for kw, text in ((dict(sign=(short, None)), "signs are int32"), (dict(sign=(good.float(), None)), "signs are int32"), (dict(sign=(good.cpu(), None)), "signs are int32"),
                     (dict(rand_pool=(rows[:, :10].contiguous(), None)), "rand_pool has one value"), (dict(rand_pool=(rows.cpu(), None)), "rand_pool has one value"),
                     (dict(rand_pool=(rows.double(), None)), "unsupported element dtype")):
        with pytest.raises(RuntimeError, match=text):
            ms.linear(xg, w, **kw)
        flip = {k: v[::-1] for k, v in kw.items()}
        if "rand_pool" in kw:
            flip = dict(rand_pool=(None, columns.cpu() if kw["rand_pool"][0].device.type == "cpu" else columns.double() if kw["rand_pool"][0].dtype == torch.float64 else rows))
        with pytest.raises(RuntimeError, match=text):
            ms.linear(x, wg, **flip)
        # the other operand's gradient does not take them, nor does a call without gradients
        ms.linear(x, wg, **kw).sum().backward()
        ms.linear(xg, w, **flip).sum().backward()
        with torch.no_grad():
            ms.linear(xg, wg, **kw)
        ms.linear(x, w, **kw)
    ms.linear(xg, wg, sign=(good, good), rand_pool=(rows, columns)).sum().backward()


def accumulator(t):
    """the node that a leaf's gradient goes through, as a reducer or a hook holds it"""
    return t.view_as(t).grad_fn.next_functions[0][0]


def test_recording_beside_held_accumulators(ms):
    """nodes that were made on a stream which can take part in a recording do not keep a layer from being recorded; nodes of the default stream, which cannot, do"""
    x, w, dy = matrix(40, 96, BF, 1, 1.0).requires_grad_(), matrix(50, 96, BF, 2, 1.0).requires_grad_(), matrix(40, 50, BF, 3, 1.0)
    made, recorder = torch.cuda.Stream(), torch.cuda.Stream()

    def record():
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=recorder):
            return graph, torch.autograd.grad(ms.linear(x, w, seed=1, step=2), (x, w), dy)
    held = [accumulator(t) for t in (x, w)]
    with pytest.raises(RuntimeError, match="default stream"):
        record()
    torch.cuda.synchronize()
    del held
    made.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(made):
        held = [accumulator(t) for t in (x, w)]
        eager = torch.autograd.grad(ms.linear(x, w, seed=1, step=2), (x, w), dy)
    torch.cuda.current_stream().wait_stream(made)
    torch.cuda.synchronize()
    graph, got = record()
    for _ in range(3):
        for t in got:
            t.zero_()
        graph.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(s, t) for s, t in zip(got, eager))
    # gradients that are added up where they lie, as a reducer's are
    x.grad, w.grad = torch.zeros_like(x), torch.zeros_like(w)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=recorder):
        ms.linear(x, w, seed=1, step=2).backward(dy)
    for t in (x, w):
        t.grad.zero_()
    for _ in range(3):
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(x.grad, eager[0]) and torch.equal(w.grad, eager[1])
        for t in (x, w):
            t.grad.zero_()
    assert len(held) == 2


@pytest.mark.parametrize("columns", [False, True])
def test_resolution_of_the_draws(ms, columns):
    """The in-kernel stream's uniform values are the 128 odd multiples of 1/256: a draw goes up with the nearest probability that they have, and never from a share of the way of
    1/256 or less (always from 255/256); a pool of float32 has no such limits."""
    share = torch.tensor([1 / 4096, 1 / 512, 1 / 256, 3 / 512, 1 / 64, 0.1, 0.25, 1 / 3, 0.5, 0.7, 254.9 / 256, 255.5 / 256], device=DEV)
    low = torch.tensor([0.0, 0.5, 1.0, 2.0, 4.0], device=DEV)
    step = torch.tensor([0.5, 0.5, 0.5, 1.0, 2.0], device=DEV)
    values = (low[:, None] + step[:, None] * share).flatten()                      # 60 values, in two blocks whose largest is 6
    x = torch.zeros(64, device=DEV)
    x[:30], x[32:62], x[31], x[63] = values[:30], values[30:], 6.0, 6.0
    draws = 16384
    many = x.repeat(draws, 1)
    many = many.t().contiguous() if columns else many

    def ups(**kw):
        v = ms.dequantize(ms.quantize(many, columns, **kw)).double()
        v = torch.cat([v[:, :30], v[:, 32:62]], 1)
        up = (v - low.double().repeat_interleave(12)) / step.double().repeat_interleave(12)
        assert torch.all((up == 0) | (up == 1))
        return up.mean(0).view(5, 12)
    p = share.double().expand(5, 12)
    # odd multiples of 1/256 below the share; six standard deviations of a mean of 16384 draws.  (low + step * share is rounded, by 2^-22 of a step at most, and no share lies that near
    # to a multiple that it is not.)
    q = torch.ceil((256 * p - 1) / 2) / 128
    assert torch.all((q - p).abs() <= 1 / 256) and torch.all(q[:, share <= 1 / 256] == 0) and torch.all(q[:, share > 255 / 256] == 1)
    assert torch.all((ups(seed=11, step=2) - q).abs() <= 6 * (q * (1 - q) / draws).sqrt())
    fine = ups(rand_pool=torch.rand(draws, 256, generator=torch.Generator(device=DEV).manual_seed(1), device=DEV))
    assert torch.all((fine - p).abs() <= 6 * (p * (1 - p) / draws).sqrt() + 2.0 ** -21)


@pytest.mark.parametrize("dtype", [BF, FP], ids=str)
def test_gradients_of_the_largest_numbers(ms, capi, dtype):
    """a power of two in front of a layer's gradient is one in front of what it makes of it, also where a rotation's sums pass binary32's range: 2^127 is the largest here"""
    x, w = ((matrix(r, 96, dtype, r, 1.0) * 2.0 ** -20).requires_grad_() for r in (70, 300))
    dy = matrix(70, 300, dtype, 3, 1.0).clamp(-2.0 ** 9, 2.0 ** 9)
    dy[:20] = torch.where(dy[:20] < 0, -2.0 ** 9, 2.0 ** 9).to(dtype)
    (bn, _), (bm, _) = signs(capi, 300, 5), signs(capi, 70, 6)
    for kw in (dict(seed=1, step=2), dict(rand_pool=(pool(70, 300, BF), pool(300, 70, BF))), dict()):
        small, far = (torch.autograd.grad(ms.linear(x, w, sign=(bn, bm), **kw), (x, w), dy * f) for f in (1.0, 2.0 ** 118))
        for a, b in zip(small, far):
            assert torch.isfinite(b).all() and torch.equal(b, a * 2.0 ** 118)
