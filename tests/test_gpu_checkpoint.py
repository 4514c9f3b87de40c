"""8-bit activation checkpoints against their definition (ref_activations.py): to the bit, and through the 4-bit layers that read them."""
import math

import numpy as np
import pytest
import torch

import ref_activations as A
import ref_operators as R

pytestmark = pytest.mark.gpu
DEV = "cuda:0"
BF, HF, FP = torch.bfloat16, torch.float16, torch.float32
NAME = {BF: "bfloat16", HF: "float16", FP: "float32"}


@pytest.fixture(scope="module")
def act(capi):
    from dynamiq_sigcomm_artifact_amd import activations
    return activations


@pytest.fixture(scope="module")
def ms(capi):
    from dynamiq_sigcomm_artifact_amd import microscale
    return microscale


def matrix(r, c, dtype, seed=0, spread=3.0):
    g = torch.Generator(device=DEV).manual_seed(seed)
    x = torch.randn(r, c, generator=g, device=DEV) * torch.exp(spread * torch.randn(r, c, generator=g, device=DEV))
    return x.clamp(-6e4, 6e4).to(dtype)


def f64(t):
    return t.detach().double().cpu().numpy()


def signs(capi, n, seed):
    bits = torch.empty(-(-n // 256) * 8, dtype=torch.int32, device=DEV)
    capi.rand_diag_bits(bits, bits.numel() * 32, seed)
    return bits


def same(c, x):
    """c is the checkpoint of x to the bit, but for the codes of blocks that are not numbers"""
    codes, scales, values = A.compress(f64(x).reshape(-1, x.shape[-1]), NAME[x.dtype])
    assert np.array_equal(c.scales.cpu().numpy(), scales)
    live = np.repeat(scales, 32, axis=1) != 255
    assert np.array_equal(c.codes.cpu().numpy()[live], codes[live])
    return values[:, :x.shape[-1]]


SHAPES = [(1, 1), (1, 32), (3, 31), (5, 33), (7, 256), (130, 257), (64, 1000), (2, 4099)]


@pytest.mark.parametrize("r,c", SHAPES)
@pytest.mark.parametrize("dtype", [FP, BF, HF], ids=str)
def test_to_the_bit(act, r, c, dtype):
    x = matrix(r, c, dtype, r + c)
    k = act.compress(x)
    assert k.shape == (r, c) and k.data.numel() == r * -(-c // 32) * 33
    values = same(k, x)
    for out in (FP, BF, HF):
        # one rounding, of a value with four significant bits
        assert torch.equal(act.restore(k, out).cpu(), torch.from_numpy(values).to(out))


def test_borders(act):
    """ties, the largest of a block on either side of a border, subnormal codes, negative zero"""
    rows = []
    for e in (-140, -130, -126, -20, 0, 60, 118):
        for top in (448.0, 448.5, 464.0, 479.9, 448.0 - 2 ** -10, 256.0, 240.0, 224.0, 447.0):
            for v in (0.0, 2 ** -10, 1.5 * 2 ** -9, 2 ** -9 * 2.5, 1.0625, 1.1875, 17.0, 19.0, -27.0, 300.0, -0.0, 2 ** -11):
                row = np.zeros(32)
                row[0], row[1:] = top, v
                rows.append(np.ldexp(row, e - 8))
    x = torch.from_numpy(np.array(rows)).to(FP).to(DEV)
    values = same(act.compress(x), x)
    assert torch.equal(act.restore(act.compress(x)).cpu(), torch.from_numpy(values).to(FP))


@pytest.mark.parametrize("dtype", [FP, BF, HF], ids=str)
def test_largest_and_smallest(act, dtype):
    """finite values stay finite in their type, and the smallest keep the least scale"""
    top = torch.finfo(dtype).max
    x = torch.zeros(6, 64, device=DEV, dtype=FP)
    for i, v in enumerate((top, -top, top * (1 - 2.0 ** -4), top / 2, torch.finfo(dtype).tiny, torch.finfo(dtype).smallest_normal * 2.0 ** -3)):
        x[i, 0], x[i, 40] = v, v
        x[i, 1] = v / 3
    x = x.to(dtype)
    k = act.compress(x)
    same(k, x)
    back = act.restore(k, dtype)
    assert torch.isfinite(back).all() and torch.equal(torch.sign(back[:4]), torch.sign(x[:4]))


@pytest.mark.parametrize("bad", [math.nan, math.inf, -math.inf])
def test_what_is_not_finite(act, ms, bad):
    x = matrix(40, 100, BF, 3)
    x[7, 40] = bad
    k = act.compress(x)
    same(k, x)
    back = act.restore(k, BF)
    hit = torch.zeros(40, 100, dtype=torch.bool, device=DEV)
    hit[7, 32:64] = True
    assert torch.equal(torch.isnan(back), hit)
    for columns in (False, True):
        v = ms.dequantize(ms.quantize(k, columns=columns))
        # a row's block is NaN as one; a column's takes the 32 tokens around it along
        want = hit.clone()
        if columns:
            want[:32, 32:64] = True
        assert torch.equal(torch.isnan(v.t() if columns else v), want)


def test_views_and_shapes(act):
    big = matrix(50, 400, BF, 4)
    for x in (big[:, 8:300], big[3:, 1:34], big[::2, :257], big.t(), big.t()[::3], big[:1], big[:, :1]):
        same(act.compress(x), x.contiguous())
    x = matrix(24, 70, HF, 5).view(2, 3, 4, 70)
    k = act.compress(x)
    assert k.shape == (24, 70)
    same(k, x)
    x = matrix(1, 70, FP, 6)[0]
    assert act.compress(x).shape == (1, 70)
    odd = torch.empty(1001, dtype=BF, device=DEV).normal_()[1:]          # an address that is aligned to an element only
    same(act.compress(odd.view(10, 100)), odd.view(10, 100))
    for shape in ((0, 5), (5, 0), (0, 0)):
        k = act.compress(torch.empty(shape, device=DEV))
        assert k.shape == shape and act.restore(k).shape == shape


def test_behind_the_buffer(act):
    """nothing is written outside the result"""
    for r, c in ((3, 33), (1, 1), (257, 100)):
        x = matrix(r, c, BF, 8)
        from dynamiq_sigcomm_artifact_amd import capi
        n = capi.lib().dq_checkpoint_bytes(r, c)
        room = torch.full((n + 64,), 77, dtype=torch.uint8, device=DEV)
        s = torch.cuda.current_stream().cuda_stream
        assert capi.lib().dq_checkpoint_compress(x.data_ptr(), 1, r, c, c, room.data_ptr() + 32, 0, s) == 0
        assert bool((room[:32] == 77).all()) and bool((room[32 + n:] == 77).all())
        assert torch.equal(room[32:32 + n], act.compress(x).data)
        out = torch.full((r * c + 16,), 5.0, dtype=BF, device=DEV)
        assert capi.lib().dq_checkpoint_restore(room.data_ptr() + 32, out.data_ptr() + 16, 1, r, c, 0, s) == 0
        assert bool((out[:8] == 5).all()) and bool((out[8 + r * c:] == 5).all())
        assert torch.equal(out[8:8 + r * c].view(r, c), act.restore(act.compress(x), BF))


@pytest.mark.parametrize("r,c", [(1, 1), (3, 31), (33, 5), (130, 257), (257, 131), (513, 1000), (64, 128)])
@pytest.mark.parametrize("columns", [False, True])
@pytest.mark.parametrize("rotate", [False, True])
def test_in_four_bits(act, ms, capi, r, c, columns, rotate):
    """a checkpoint in 4 bits is that of its values in float32"""
    k = act.compress(matrix(r, c, BF, 9))
    sign = signs(capi, r if columns else c, 4) if rotate else None
    q, want = ms.quantize(k, columns=columns, sign=sign), ms.quantize(act.restore(k), columns=columns, sign=sign)
    assert torch.equal(q.codes, want.codes) and torch.equal(q.scales, want.scales) and q.shape == want.shape


@pytest.mark.parametrize("r,c", [(2100, 8200), (256 * 16, 4096), (65, 70001), (70001, 65)])
@pytest.mark.parametrize("rotate", [False, True])
def test_in_four_bits_of_many(act, ms, capi, r, c, rotate):
    """sizes that fill the chip: wide tiles, ragged at both ends"""
    x = matrix(r, c, BF, 12)
    x[r // 2, c // 3], x[r - 1, c - 1], x[r - 1, 0] = math.inf, math.nan, torch.finfo(BF).max
    k = act.compress(x)
    sign = signs(capi, r, 4) if rotate else None
    q, want = ms.quantize(k, columns=True, sign=sign), ms.quantize(act.restore(k), columns=True, sign=sign)
    live = torch.repeat_interleave(want.scales != 255, 16, 1)
    assert torch.equal(q.scales, want.scales) and torch.equal(q.codes[live], want.codes[live]) and bool((want.scales == 255).any())


def test_hinted_loads(act):
    """what is beyond the cache, whose loads carry a hint, against parts of it that are not"""
    x = matrix(9001, 8192, BF, 13)
    whole = act.compress(x)
    for part, codes, scales in zip(x.split(3000), whole.codes.split(3000), whole.scales.split(3000)):
        c = act.compress(part)
        assert torch.equal(c.codes, codes) and torch.equal(c.scales, scales)


def test_in_four_bits_of_the_largest_numbers(act, ms, capi):
    """sums beyond 2^128 in the rotation, next to what is not finite"""
    x = matrix(300, 200, FP, 10, 0.5)
    x[32:64] = torch.finfo(FP).max * torch.where(torch.rand(32, 200, device=DEV) < 0.5, -1.0, 1.0)
    x[64:96, 7] = 2.0 ** 126
    x[150, 3] = math.inf
    k = act.compress(x)
    for columns in (False, True):
        sign = signs(capi, 300 if columns else 200, 4)
        q, want = ms.quantize(k, columns=columns, sign=sign), ms.quantize(act.restore(k), columns=columns, sign=sign)
        live = torch.repeat_interleave(want.scales != 255, 16, 1)
        assert torch.equal(q.scales, want.scales) and torch.equal(q.codes[live], want.codes[live])


def test_rows_ignore_what_lies_in_the_padding(act, ms):
    k = act.compress(matrix(5, 40, BF, 11))
    want = ms.quantize(k)
    k.codes[:, 40:] = 126
    got = ms.quantize(k)
    assert torch.equal(got.codes, want.codes) and torch.equal(got.scales, want.scales)


@pytest.mark.parametrize("m,n,k", [(1, 40, 64), (70, 33, 300), (300, 257, 96)])
@pytest.mark.parametrize("dtype", [BF, HF, FP], ids=str)
@pytest.mark.parametrize("made", ["here", "given"])
def test_linear(act, ms, capi, m, n, k, dtype, made):
    """the layer's results and dx are those without a checkpoint, dw is that of x restored"""
    x, w, dy = matrix(m, k, dtype, 1, 1.0), matrix(n, k, dtype, 2, 1.0), matrix(m, n, dtype, 3, 1.0)
    kw = dict(sign=(signs(capi, n, 5), signs(capi, m, 6)), seed=77, step=3)
    x1, w1 = x.clone().requires_grad_(), w.clone().requires_grad_()
    c = act.compress(x)
    y1 = ms.linear(x1, w1, checkpoint=True if made == "here" else c, **kw)
    y1.backward(dy)
    x2, w2 = x.clone().requires_grad_(), w.clone().requires_grad_()
    y2 = ms.linear(x2, w2, **kw)
    y2.backward(dy)
    assert torch.equal(y1, y2) and torch.equal(x1.grad, x2.grad) and w1.grad.dtype == dtype
    pools = torch.empty(n, -(-m // 256) * 256, device=DEV)
    capi.philox_uniform(pools, 77, 3 + (1 << 63))
    a = ms.quantize(dy, columns=True, sign=kw["sign"][1], rand_pool=pools)
    b = ms.quantize(act.restore(c), columns=True, sign=kw["sign"][1])
    assert torch.equal(w1.grad, ms.product(a, b, dtype))


def test_linear_shares_and_partial_gradients(act, ms):
    x, w1, w2 = matrix(60, 96, BF, 1, 1.0).view(3, 20, 96), matrix(40, 96, BF, 2, 1.0), matrix(50, 96, BF, 3, 1.0)
    c = act.compress(x)
    dy1, dy2 = matrix(60, 40, BF, 4).view(3, 20, 40), matrix(60, 50, BF, 5).view(3, 20, 50)
    w1.requires_grad_(), w2.requires_grad_()
    torch.autograd.backward((ms.linear(x, w1, checkpoint=c), ms.linear(x, w2, checkpoint=c)), (dy1, dy2))
    for w, dy in ((w1, dy1), (w2, dy2)):
        q = ms.product(ms.quantize(dy.view(60, -1), columns=True), ms.quantize(c, columns=True), BF)
        assert torch.equal(w.grad, q)
    x.requires_grad_()
    fixed = w1.detach()
    dx, = torch.autograd.grad(ms.linear(x, fixed, checkpoint=True), x, dy1)
    want, = torch.autograd.grad(ms.linear(x, fixed), x, dy1)
    assert torch.equal(dx, want)
    with torch.no_grad():
        assert torch.equal(ms.linear(x, w1, checkpoint=True), ms.linear(x, w1))
    empty = torch.empty(0, 96, dtype=BF, device=DEV)
    y = ms.linear(empty, w1, checkpoint=True)
    dw, = torch.autograd.grad(y, w1, torch.empty_like(y))
    assert not dw.any()


def test_linear_lets_go_of_x(act, ms):
    """what the layer holds between the passes is a byte an element"""
    x, w = matrix(4096, 1024, BF, 1, 1.0), matrix(32, 1024, BF, 2, 1.0).requires_grad_()
    torch.cuda.synchronize()
    before = torch.cuda.memory_allocated()
    y = ms.linear(x.clone(), w, checkpoint=True)
    held = torch.cuda.memory_allocated() - before - y.numel() * 2
    assert held <= 4096 * 1024 * 33 // 32 + 4096
    del y


def test_refusals(act, ms):
    x = matrix(10, 64, BF, 1)
    c = act.compress(x)
    w = matrix(8, 64, BF, 2)
    for call, text in ((lambda: act.compress(x.double()), "element dtype"), (lambda: act.compress(x.cpu()), "must live on the GPU"), (lambda: act.compress(x[0, 0]), "rows are required"),
                       (lambda: act.compress([1.0]), "a tensor argument"), (lambda: act.restore(c, torch.float64), "element dtype"),
                       (lambda: act.restore(act.Checkpoint(c.data, 11, 64)), "does not belong"), (lambda: act.restore(act.Checkpoint(c.data.cpu(), 10, 64)), "must live on the GPU"),
                       (lambda: act.restore(act.Checkpoint(c.data.float(), 10, 64)), "does not belong"),
                       (lambda: ms.quantize(c, rand_pool=x), "to nearest"), (lambda: ms.quantize(c, seed=1), "to nearest"),
                       (lambda: ms.quantize(c, sign=torch.zeros(7, dtype=torch.int32, device=DEV)), "sign"),
                       (lambda: ms.quantize(act.Checkpoint(c.data[:-1], 10, 64)), "does not belong"),
                       (lambda: ms.linear(x, w, checkpoint=act.compress(x[:5])), "does not belong"), (lambda: ms.linear(x, w, checkpoint=act.Checkpoint(c.data, 20, 32)), "32 columns"),
                       (lambda: ms.linear(x, w, checkpoint=act.Checkpoint(c.data.cpu(), 10, 64)), "must live on the GPU")):
        with pytest.raises(RuntimeError, match=text):
            call()


def test_graph_and_streams(act, ms, capi):
    """recorded and replayed, a whole step of a layer with a checkpoint, between eager work"""
    x, w, dy = matrix(300, 128, BF, 1, 1.0), matrix(64, 128, BF, 2, 1.0).requires_grad_(), matrix(300, 64, BF, 3, 1.0)
    count = torch.zeros(1, dtype=torch.int64, device=DEV)
    sign = (signs(capi, 64, 5), signs(capi, 300, 6))

    def step(step):
        c = act.compress(x)
        y = ms.linear(x, w, sign=sign, seed=9, step=step, checkpoint=c)
        dw, = torch.autograd.grad(y, w, dy)
        return c.data, act.restore(c, BF), y.detach(), dw
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step(count)
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = step(count)
    for k in range(4):
        count.fill_(k)
        x.normal_()
        graph.replay()
        torch.cuda.synchronize()
        want = step(k)
        assert all(torch.equal(a, b) for a, b in zip(out, want)), k
        torch.cuda.synchronize()


def test_views_of_a_batch_are_read_in_place(act):
    """views with consecutive rows of more dimensions than two: right, and nothing of their size is made beside the result"""
    big = matrix(24, 400, BF, 4).view(2, 3, 4, 400)
    for x in (big[..., 8:300], big[..., :257], big[:, :, ::2], big.transpose(0, 1)[..., 3:90], big[..., ::3], big[:1, :1, :1, :33], big[:, :1].expand(2, 3, 4, 400)):
        same(act.compress(x), x.contiguous())
    x = matrix(2048, 4096, BF, 5).view(8, 256, 4096)[..., :2048]
    torch.cuda.synchronize()
    torch.cuda.reset_peak_memory_stats()
    before = torch.cuda.memory_allocated()
    c = act.compress(x)
    assert torch.cuda.max_memory_allocated() - before <= c.data.numel() + 65536
