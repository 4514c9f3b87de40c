"""The optimizer's and the 4-bit operators beyond 2^31 elements: what the last rows come out as on their own."""
import pytest
import torch

pytestmark = pytest.mark.gpu
DEV = "cuda:0"
BF = torch.bfloat16
ROWS, COLS = 66000, 33000  # 2,178,000,000 elements


@pytest.fixture(scope="module")
def ops():
    if not torch.cuda.is_available():
        pytest.skip("needs a GPU")
    if torch.cuda.get_device_properties(0).total_memory < 100 << 30:
        pytest.skip("needs 100 GB of device memory")
    from dynamiq_sigcomm_artifact_amd import microscale, optimizer
    yield microscale, optimizer
    torch.cuda.empty_cache()


def big(rows, cols, seed):
    """random elements, in pieces (torch draws a few billion at a time)"""
    g = torch.Generator(device=DEV).manual_seed(seed)
    out = torch.empty(rows, cols, dtype=BF, device=DEV)
    for part in out.split(8192):
        part.copy_(torch.randn(part.shape, generator=g, device=DEV))
    return out


def same(a, b):
    return torch.equal(a.codes, b.codes) and torch.equal(a.scales, b.scales)


def part(ms, q, lo):
    return ms.Microscaled(q.codes[lo:], q.scales[lo:], q.rows - lo, q.cols)


def test_rows_and_columns(ops):
    ms = ops[0]
    x = big(ROWS, COLS, 1)
    q = ms.quantize(x)
    assert same(part(ms, q, ROWS - 40), ms.quantize(x[-40:]))
    assert torch.equal(ms.dequantize(q, BF)[-40:], ms.dequantize(ms.quantize(x[-40:]), BF))
    del q
    q = ms.quantize(x, columns=True)
    assert same(part(ms, q, COLS - 40), ms.quantize(x[:, -40:].contiguous(), columns=True))
    del q
    pool = torch.empty(ROWS, -(-COLS // 256) * 256, dtype=BF, device=DEV)
    for p in pool.split(8192):
        p.copy_(torch.rand(p.shape, device=DEV) * 0.99)
    assert same(part(ms, ms.quantize(x, rand_pool=pool), ROWS - 40), ms.quantize(x[-40:], rand_pool=pool[-40:].contiguous()))
    del pool
    # the in-kernel stream's chunks count over the whole result, padding included: 2^27 of them and more
    from dynamiq_sigcomm_artifact_amd import capi
    words = torch.empty(ROWS * (-(-COLS // 256) * 256), dtype=torch.float32, device=DEV)
    capi.philox_uniform(words, 9, 4)
    assert same(part(ms, ms.quantize(x, seed=9, step=4), ROWS - 40), ms.quantize(x[-40:], rand_pool=words.view(ROWS, -1)[-40:].contiguous()))


def test_rows_far_apart(ops):
    """rows of a view whose offsets pass 2^31 elements and 2^32 bytes"""
    ms = ops[0]
    x = big(40, 64, 2)
    far = torch.empty(39 * (1 << 26) + 64, dtype=BF, device=DEV).as_strided((40, 64), (1 << 26, 1))
    far.copy_(x)
    for columns in (False, True):
        assert same(ms.quantize(far, columns), ms.quantize(x, columns))


def test_product(ops):
    """small integers: E2M1 has them, and their sums are exact"""
    ms = ops[0]
    g = torch.Generator(device=DEV).manual_seed(3)
    a, b = (torch.randint(-4, 5, (r, 300), generator=g, device=DEV).to(BF) for r in (ROWS, COLS))
    # (a scale that every block shares, so that no element is rounded)
    a[:, ::32], b[:, ::32] = 4, 4
    out = ms.product(ms.quantize(a), ms.quantize(b))
    want = (a[-70:].float() @ b.float().t()).to(BF)
    assert torch.equal(out[-70:], want)
    assert torch.equal(out[:, -70:].float(), (a.float() @ b[-70:].float().t()).to(BF).float())


def test_norm_and_step(ops):
    opt = ops[1]
    n = (1 << 31) + 1234
    g = big(1, 1 << 20, 4).view(-1).repeat(n // (1 << 20) + 1)[:n]
    once = g[:1 << 20].double().square().sum()
    want = float(torch.sqrt(once * (n // (1 << 20)) + g[n - n % (1 << 20):].double().square().sum()))
    assert abs(float(opt.grad_norm([g])[0]) - want) <= want * (2.0 ** -24 + 1e-11)
    p = torch.empty(n, dtype=torch.float32, device=DEV)
    p.fill_(0.5)
    for bits in (32, 8):
        tail = [p[-1000:].clone()]
        state, small = opt.adamw_state([p], bits), opt.adamw_state(tail, bits)
        opt.adamw_step([p], [g], state, 1)
        opt.adamw_step(tail, [g[-1000:]], small, 1)
        # (a first step takes the moments from the gradient alone, whatever the 8-bit states become: the dither counts from the tensor's beginning)
        assert torch.equal(p[-1000:], tail[0])
        if bits == 32:
            lo = n - 1000
            assert torch.equal(state[:, lo:lo + 1000], small[:, :1000])
        del state


def test_states_in_8_bits(ops):
    """What the last elements' states become, and what the next step makes of them.  The dither of element i at step t is a function of i C + t D mod 2^32 with D odd: it is that
    of element i - lo at the step t + lo C / D, which a small call is given.  (The moments do not depend on the step's number otherwise; the weights do.)"""
    opt = ops[1]
    n = (1 << 31) + 1234
    lo = (n - 1000) // 32 * 32
    shift = lo * 0x9E3779B9 * pow(0xB504F333, -1, 1 << 32) % (1 << 32)
    p = torch.full((n,), 0.5, dtype=torch.float32, device=DEV)
    state = opt.adamw_state([p], 8)
    tail, small = p[lo:].clone(), opt.adamw_state([p[lo:]], 8)
    g = torch.empty(n, dtype=BF, device=DEV)
    for t in (1, 2, 3):
        g.copy_(big(1, 1 << 20, 10 + t).view(-1).repeat(n // (1 << 20) + 1)[:n])
        now = tuple(s.clone() for s in small)
        opt.adamw_step([p], [g], state, t)
        opt.adamw_step([tail], [g[lo:]], now, t)                               # the weights, from the states before
        opt.adamw_step([torch.zeros_like(tail)], [g[lo:]], small, t + shift)   # the states behind
        assert torch.equal(p[lo:], tail)
        for whole, part, unit in zip(state, small, (1, 32)):
            assert torch.equal(whole[:, lo // unit:], part)
        assert int((state[0][:, lo:] != 0).sum()) > 1900                       # (both moments of nearly all 1000 elements)
