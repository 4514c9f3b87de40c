"""What the entry points of activations refuse, before any device work, and the host side of their objects."""
import ctypes

import numpy as np
import pytest
import torch

import ref_activations as A

P, N, S = ctypes.c_void_p(0x1000), ctypes.c_void_p(0), ctypes.c_void_p(0)


@pytest.fixture(scope="module")
def L():
    from dynamiq_sigcomm_artifact_amd import capi
    return capi.lib()


def refused(L, rc, text):
    assert rc != 0 and text in L.dq_last_error().decode(), (rc, L.dq_last_error().decode())


def test_checkpoints_refuse(L):
    assert L.dq_checkpoint_bytes(3, 33) == 3 * 2 * 33 and L.dq_checkpoint_bytes(1, 1) == 33 and L.dq_checkpoint_bytes(0, 5) == 0
    odd = ctypes.c_void_p(0x1008)

    def compress(x=P, dtype=1, r=10, c=300, stride=300, data=P):
        return L.dq_checkpoint_compress(x, dtype, r, c, stride, data, 0, S)

    def restore(data=P, out=P, dtype=1, r=10, c=300):
        return L.dq_checkpoint_restore(data, out, dtype, r, c, 0, S)
    for kw, text in ((dict(dtype=3), "dtype"), (dict(r=0), "positive"), (dict(c=0), "positive"), (dict(r=1 << 31, c=1), "2^31"), (dict(c=1 << 31, stride=1 << 31), "2^31"),
                     (dict(r=1 << 30, c=32), "2^35"), (dict(stride=299), "stride"), (dict(stride=1 << 40), "stride"), (dict(x=N), "null"), (dict(data=N), "null"), (dict(data=odd), "aligned")):
        refused(L, compress(**kw), text)
    for kw, text in ((dict(dtype=3), "dtype"), (dict(r=-1), "positive"), (dict(c=0), "positive"), (dict(r=1 << 30, c=32), "2^35"), (dict(data=N), "null"), (dict(out=N), "null"),
                     (dict(data=odd), "aligned")):
        refused(L, restore(**kw), text)


def test_checkpoints_as_matrices_refuse(L):
    Z = ctypes.c_uint64(0)

    def quantize(x=P, r=10, c=300, stride=320, stochastic=0, pool=N, codes=P, scales=P):
        return L.dq_mx4_quantize(x, 3, r, c, stride, 1, N, stochastic, pool, 1, Z, Z, N, codes, scales, 0, S)
    for kw, text in ((dict(stride=300), "padded columns"), (dict(stride=352), "padded columns"), (dict(x=ctypes.c_void_p(0x1008)), "aligned"), (dict(stochastic=1), "to nearest"),
                     (dict(stochastic=1, pool=P), "to nearest"), (dict(r=0), "positive"), (dict(x=N), "null"), (dict(codes=N), "null")):
        refused(L, quantize(**kw), text)


def test_modules_refuse_host_tensors():
    from dynamiq_sigcomm_artifact_amd import activations, microscale
    x = torch.zeros(4, 32)
    c = activations.Checkpoint(torch.zeros(4 * 33, dtype=torch.uint8), 4, 32)
    assert c.shape == (4, 32) and c.codes.shape == (4, 32) and c.scales.shape == (4, 1) and "4 x 32" in repr(c)
    for call in (lambda: activations.compress(x), lambda: activations.restore(c), lambda: microscale.quantize(c), lambda: microscale.linear(x, x, checkpoint=True)):
        with pytest.raises(RuntimeError, match="must live on the GPU"):
            call()
    with pytest.raises(RuntimeError, match="element dtype"):
        activations.restore(c, torch.float64)
    with pytest.raises(RuntimeError, match="to nearest"):
        microscale.quantize(c, seed=1)
    with pytest.raises(RuntimeError, match="columns"):
        microscale.linear(torch.zeros(4, 33), x, checkpoint=c)


def test_definition_against_the_cast():
    """the definition's codes are those of torch's cast to E4M3 of the scaled values"""
    x = np.random.default_rng(1).standard_normal((40, 100)) * np.exp(np.random.default_rng(2).standard_normal((40, 100)) * 4)
    x = torch.from_numpy(x).bfloat16().double().numpy()
    codes, scales, values = A.compress(x, "bfloat16")
    padded = np.zeros((40, 128))
    padded[:, :100] = x
    y = torch.from_numpy(padded.reshape(40, 4, 32) / 2.0 ** (scales.astype(np.float64) - 127)[:, :, None]).float()
    assert float(y.abs().max()) <= 448 and np.array_equal(y.to(torch.float8_e4m3fn).view(torch.uint8).reshape(40, 128).numpy(), codes)
    assert np.abs(values[:, :100] - x).max() <= np.abs(x).max() * 2.0 ** -4
