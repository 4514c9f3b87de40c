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


def test_gated_refuses(L):
    from dynamiq_sigcomm_artifact_amd import capi
    good = dict(gate=0x1000, up=0x1000, gate_stride=20, up_stride=20, out=0x1000, rows=4, cols=10, dtype=1, kind=0)
    back = dict(good, dgate=0x1000, dup=0x1000, dgate_stride=20, dup_stride=20)
    for fn, base in ((L.dq_gated_forward, good), (L.dq_gated_backward, back)):
        refused(L, fn(None, 0, S), "null")
        for kw, text in ((dict(dtype=3), "dtype"), (dict(kind=2), "activation"), (dict(rows=0), "positive"), (dict(cols=-1), "positive"), (dict(rows=1 << 31), "2^31"),
                         (dict(rows=1 << 30, cols=32, gate_stride=32, up_stride=32, dgate_stride=32, dup_stride=32), "2^35"), (dict(gate=None), "null"), (dict(up=None), "null"),
                         (dict(out=None), "null"), (dict(gate_stride=9), "stride"), (dict(up_stride=1 << 40), "stride"), (dict(gate8=0x1004, up8=0x1000), "aligned")):
            refused(L, fn(ctypes.byref(capi.Gated(**{**base, **kw})), 0, S), text)
    refused(L, L.dq_gated_forward(ctypes.byref(capi.Gated(**good, out8=0x1008)), 0, S), "aligned")
    refused(L, L.dq_gated_backward(ctypes.byref(capi.Gated(**back, gate8=0x1000)), 0, S), "or neither")
    refused(L, L.dq_gated_backward(ctypes.byref(capi.Gated(**{**back, "dup_stride": 5})), 0, S), "stride")


def test_gradients_of_the_definitions_against_differences():
    """the formulas of the reference itself, in 64 bits: central differences with a step of 1e-5 are off by some 1e-10 of the third derivative and 1e-11 of the value"""
    rng = np.random.default_rng(3)
    step = 1e-5
    for kind in ("silu", "gelu_tanh"):
        g = rng.standard_normal(200) * 3
        slope = (A.act(g + step, kind)[0] - A.act(g - step, kind)[0]) / (2 * step)
        assert np.abs(slope - A.act(g, kind)[1]).max() < 1e-8
    rows, cols = 3, 11
    for case in range(24):
        center, after, gated, residual, before = case & 1, case >> 1 & 1, case >> 2 & 1, case >> 3 & 1, case < 16
        v = {k: rng.standard_normal((rows, cols)) for k in ("y", "residual", "gate")}
        p = {k: rng.standard_normal(cols) for k in ("weight", "bias", "after_weight", "after_bias")}
        dh, dr = rng.standard_normal((rows, cols)), rng.standard_normal((rows, cols))

        def settings(p):
            return {**p, "center": center, "after": after, "before": before, "eps": 1e-3, "residual_scale": 0.7, "block_scale": 1.3,
                    **({} if before else {"weight": None, "bias": None}), **({} if after else {"after_weight": None, "after_bias": None})}

        def loss(v, p):
            h, r, _, _ = A.block(v["y"], v["residual"] if residual else None, v["gate"] if gated else None, settings(p))
            return (r * dr).sum() + ((h * dh).sum() if before else 0.0)
        _, r, st_r, st_y = A.block(v["y"], v["residual"] if residual else None, v["gate"] if gated else None, settings(p))
        got = A.block_gradients(v["y"], r, st_r, st_y, v["gate"] if gated else None, settings(p), dh if before else None, dr)
        names = ["y"] + ["residual"] * residual + ["gate"] * gated + ["weight", "bias"] * before + ["after_weight", "after_bias"] * after
        for name in names:
            where = v if name in v else p
            direction = rng.standard_normal(where[name].shape)
            ends = [loss(*[{**d, name: d[name] + sign * step * direction} if d is where else d for d in (v, p)]) for sign in (1, -1)]
            want = (ends[0] - ends[1]) / (2 * step)
            mine = (got[name] * direction).sum()
            assert abs(want - mine) <= 1e-6 * max(1.0, abs(want)), (case, name, want, mine)


def test_residual_norm_refuses(L):
    from dynamiq_sigcomm_artifact_amd import capi
    inf = float("inf")
    forward = dict(y=0x1000, residual=0x1000, h=0x1000, r=0x1000, rows=6, cols=40, eps=1e-5, residual_scale=1.0, block_scale=1.0, dtype=1, stream_dtype=1, before=1)
    backward = dict(forward, stats=0x1000, dh=0x1000, dr=0x1000, dy=0x1000, dweight=0x1000, work=0x1000, work_floats=1 << 20)

    def call(fn, base, **kw):
        return fn(ctypes.byref(capi.ResidualNorm(**{**base, **kw})), 0, S)
    for fn, base in ((L.dq_residual_norm_forward, forward), (L.dq_residual_norm_backward, backward)):
        refused(L, fn(None, 0, S), "null")
        for kw, text in ((dict(dtype=3), "dtype"), (dict(stream_dtype=0), "dtype"), (dict(rows=0), "rows must"), (dict(rows=1 << 31), "rows must"), (dict(cols=7), "cols"), (dict(cols=32769), "cols"),
                         (dict(gate=0x1000, rows_per_gate=4), "divide"), (dict(gate=0x1000, rows_per_gate=0), "divide"), (dict(eps=-1.0), "eps"), (dict(eps=inf), "eps"),
                         (dict(residual_scale=inf), "scales"), (dict(block_scale=float("nan")), "scales"), (dict(keep_r=1), "null"), (dict(kept=0x1008), "aligned"), (dict(stats=0x1008), "aligned"),
                         (dict(h8=0x1004), "aligned")):
            refused(L, call(fn, base, **kw), text)
    for kw, text in ((dict(y=None), "null"), (dict(h=None), "null"), (dict(r=None), "null"), (dict(before=0), "before"), (dict(residual=None, stream_dtype=2), "stream")):
        refused(L, call(L.dq_residual_norm_forward, forward, **kw), text)
    for kw, text in ((dict(stats=None), "null"), (dict(dh=None, dr=None), "null"), (dict(before=0), "before"), (dict(dh=None), "took no part"), (dict(dgate=0x1000), "took no part"),
                     (dict(dafter_weight=0x1000), "took no part"), (dict(r=None), "checkpoints"), (dict(after=1, y=None), "checkpoints"), (dict(work=None), "null"), (dict(work_floats=39), "too small"),
                     (dict(after=1, keep_y=1, kept=0x1000), "both in 8 bits")):
        refused(L, call(L.dq_residual_norm_backward, backward, **kw), text)

    def room(**kw):
        return L.dq_residual_norm_work_floats(ctypes.byref(capi.ResidualNorm(**{**backward, **kw})))
    assert 40 <= room() <= 6 * 40 and room(dweight=None) == 0 and room(dbias=0x1000) == 2 * room() and room(cols=7) == -1
    assert room(gate=0x1000, dgate=0x1000, rows_per_gate=1) == room(gate=0x1000, rows_per_gate=1)
    # runs of rows: as many partial sums as workgroups, and a gate's rows with none but their own
    assert room(rows=1 << 20, dbias=0x1000) % (2 * 40) == 0 and room(rows=1 << 20) // 40 <= 2048
    assert room(rows=1 << 20, gate=0x1000, dgate=0x1000, rows_per_gate=1 << 19) // 40 <= 4096
    for rows in (1, 2, 1000, 4097, 100003):
        for per in (1, rows):
            assert 0 < room(rows=rows, gate=0x1000, dgate=0x1000, rows_per_gate=per) <= 2 * 40 * min(rows, 2048)


def test_residual_norm_refuses_checkpoints_beyond_their_size(L):
    """one of 2^35 elements, which no reader of a checkpoint takes; what keeps nothing in 8 bits has no such limit"""
    from dynamiq_sigcomm_artifact_amd import capi
    both = dict(y=0x1000, residual=0x1000, r=0x1000, rows=1 << 20, cols=32768, eps=1e-5, residual_scale=1.0, block_scale=1.0, dtype=1, stream_dtype=1, before=1)
    forward = dict(both, h=0x1000)
    backward = dict(both, stats=0x1000, dh=0x1000, dr=0x1000, dy=0x1000, dweight=0x1000, work=0x1000, work_floats=1 << 40)

    def call(fn, base, **kw):
        return fn(ctypes.byref(capi.ResidualNorm(**{**base, **kw})), 0, S)
    for kw in (dict(h8=0x1000), dict(keep_r=1, kept=0x1000), dict(after=1, keep_y=1, kept=0x1000), dict(after=1, keep_r=1, keep_y=1, kept=0x1000)):
        refused(L, call(L.dq_residual_norm_forward, forward, **kw), "2^35")
        if "kept" in kw:
            refused(L, call(L.dq_residual_norm_backward, backward, **kw), "2^35")
            assert L.dq_residual_norm_work_floats(ctypes.byref(capi.ResidualNorm(**{**backward, **kw}))) == -1
    assert L.dq_residual_norm_work_floats(ctypes.byref(capi.ResidualNorm(**backward))) > 0
    small = dict(backward, rows=(1 << 20) - 1, after=1, keep_r=1, keep_y=1, kept=0x1000)
    assert L.dq_residual_norm_work_floats(ctypes.byref(capi.ResidualNorm(**small))) > 0


def test_residual_norm_shares_its_rows_out(L):
    """A gate with somewhat more rows than a team would take makes no more workgroups, and partial sums of theirs, than others do: two a CU, in wide rows for all of their tiles together,
    and twice as many where runs of whole gates are shorter than the others, by less than half"""
    from dynamiq_sigcomm_artifact_amd import capi
    for cols, rows, pers in ((512, 8190, (1, 2, 3)), (512, 8192, (4,)), (256, 12288, (1, 2, 3, 4, 6)), (64, 30000, (1, 6, 8, 12)), (1024, 2048, (1, 2)), (14336, 4096, (1, 16, 32)), (32768, 984, (8, 24))):
        for per in pers:
            o = capi.ResidualNorm(y=0x1000, residual=0x1000, gate=0x1000, h=0x1000, r=0x1000, rows=rows, cols=cols, rows_per_gate=per, eps=1e-5, residual_scale=1.0, block_scale=1.0, dtype=1,
                                  stream_dtype=1, before=1, stats=0x1000, dh=0x1000, dweight=0x1000)
            workgroups = (L.dq_residual_norm_work_floats(ctypes.byref(o)) - (4 * rows if cols > 8192 else 0)) / cols
            assert workgroups <= 2 * (512 if cols <= 8192 else 512 // -(-cols // 512)), (cols, rows, per, workgroups)
