"""The operators between the linear layers beyond 2^31 elements and 2^32 bytes: offsets in 64 bits, on rows at both ends and in the middle."""
import pytest
import torch

pytestmark = pytest.mark.gpu
DEV = "cuda:0"
BF = torch.bfloat16


@pytest.fixture(scope="module")
def ops(capi):
    if torch.cuda.get_device_properties(0).total_memory < 100 << 30:
        pytest.skip("needs 100 GB")
    from dynamiq_sigcomm_artifact_amd import activations, microscale
    yield activations, microscale
    torch.cuda.empty_cache()


def filled(rows, cols, seed, dtype=BF):
    x = torch.empty(rows, cols, dtype=dtype, device=DEV)
    g = torch.Generator(device=DEV).manual_seed(seed)
    for part in x.split(8192):
        part.normal_(generator=g)
    return x


def some(rows):
    """rows at the ends, and around 2^31 and 2^32 elements of 32768 columns"""
    return torch.tensor(sorted({k for at in (0, 1 << 16, 1 << 17, rows) for k in range(at - 3, at + 3) if 0 <= k < rows}), device=DEV)


ROWS, COLS = (1 << 17) + 40, 32768          # 4.3e9 elements, 8.6 GB in 16 bits


def test_checkpoint(ops):
    act, ms = ops
    x = filled(ROWS, COLS, 1)
    c = act.compress(x)
    at = some(ROWS)
    want = act.compress(x[at])
    assert torch.equal(c.codes[at], want.codes) and torch.equal(c.scales[at], want.scales)
    back = act.restore(c, BF)
    assert torch.equal(back[at], act.restore(want, BF))
    del x, back
    q = ms.quantize(c, columns=True)
    for k in (0, 1 << 16, ROWS - 256 - ROWS % 256):
        k -= k % 256
        part = act.Checkpoint(torch.cat((c.codes[k:k + 256].reshape(-1), c.scales[k:k + 256].reshape(-1))), min(256, ROWS - k), COLS)
        w = ms.quantize(part, columns=True)
        assert torch.equal(q.codes[:, k // 2:k // 2 + 128], w.codes) and torch.equal(q.scales[:, k // 32:k // 32 + 8], w.scales)


def test_gated(ops):
    act, _ = ops
    x = filled(ROWS // 2, COLS, 2).requires_grad_()          # rows of 2 * 16384
    out, c = act.gated(x, checkpoint=True)
    da = filled(ROWS // 2, COLS // 2, 3)
    dx, = torch.autograd.grad(out, x, da)
    at = some(ROWS // 2)
    y = x.detach()[at].requires_grad_()
    want, wc = act.gated(y, checkpoint=True)
    assert torch.equal(out[at], want) and torch.equal(c.codes[at], wc.codes)
    assert torch.equal(dx[at], torch.autograd.grad(want, y, da[at])[0])


@pytest.mark.parametrize("cols", [8192, 32768])
@pytest.mark.parametrize("eight", [False, True])
def test_residual_norm(ops, cols, eight):
    act, _ = ops
    rows = ((1 << 31) + (1 << 20)) // cols + 40
    y, x = filled(rows, cols, 4), filled(rows, cols, 5)
    w = torch.randn(cols, device=DEV).to(BF)
    at = torch.tensor(sorted({k for b in (0, rows // 2, (1 << 31) // cols, rows) for k in range(b - 3, b + 3) if 0 <= k < rows}), device=DEV)

    def run(y, x, dh, dr):
        y, x = y.requires_grad_(), x.requires_grad_()
        got = act.residual_norm(y, x, w, gate=w, checkpoint=eight)
        return got, torch.autograd.grad(got[:2], (y, x), (dh, dr))
    dh, dr = filled(rows, cols, 6), filled(rows, cols, 7)
    got, grads = run(y, x, dh, dr)
    want, wants = run(y.detach()[at], x.detach()[at], dh[at], dr[at])
    assert all(torch.equal(a[at], b) for a, b in zip(got[:2], want[:2])) and all(torch.equal(a[at], b) for a, b in zip(grads, wants))
    if eight:
        assert torch.equal(got[2].codes[at], want[2].codes) and torch.equal(got[2].scales[at], want[2].scales)
