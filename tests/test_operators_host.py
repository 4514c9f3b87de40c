"""What the optimizer's and the microscaled entry points refuse, before any device work, and the host side of their objects."""
import ctypes

import numpy as np
import pytest
import torch

import ref_operators as R

P, N, S = ctypes.c_void_p(0x1000), ctypes.c_void_p(0), ctypes.c_void_p(0)
NAN = float("nan")


@pytest.fixture(scope="module")
def L():
    from dynamiq_sigcomm_artifact_amd import capi
    return capi.lib()


def refused(L, rc, text):
    assert rc != 0 and text in L.dq_last_error().decode(), (rc, L.dq_last_error().decode())


def test_norm_refuses(L):
    from dynamiq_sigcomm_artifact_amd import capi
    room = L.dq_grad_norm_work_doubles()
    assert room <= 4096                               # callers may count on this much
    one = (capi.Span * 1)(capi.Span(0x1000, 10, capi.F32, 0))

    def call(spans=one, count=1, most=1.0, work=P, doubles=room, out=P):
        return L.dq_grad_norm(spans, count, most, work, doubles, out, 0, S)
    refused(L, call(count=-1), "count")
    refused(L, call(work=N), "null pointer")
    refused(L, call(out=N), "null pointer")
    refused(L, call(most=0.0), "max_norm")
    refused(L, call(most=NAN), "max_norm")
    refused(L, call(doubles=room - 1), "work buffer is too small")
    for bad, text in ((capi.Span(0x1000, 10, 7, 0), "element dtype"), (capi.Span(0x1000, -1, capi.F32, 0), "2^40"),
                      (capi.Span(0x1000, 1 << 40, capi.F32, 0), "2^40"), (capi.Span(None, 10, capi.F32, 0), "null pointer")):
        refused(L, call(spans=(capi.Span * 1)(bad)), text)


def test_step_refuses(L):
    from dynamiq_sigcomm_artifact_amd import capi
    good = dict(state=0x1000, scales=None, master=None, total=64, bits=32, reserved=0, lr=1e-3, beta1=0.9, beta2=0.999, eps=1e-8, weight_decay=0.0,
                step=1, grad_scale=None, coefficients=None)
    tensor = dict(param=0x1000, grad=0x1000, n=40, start=0, param_dtype=capi.F32, grad_dtype=capi.F32)

    def call(t=(), **kw):
        x = (capi.AdamwTensor * 1)(capi.AdamwTensor(**{**tensor, **dict(t)}))
        return L.dq_adamw_step(ctypes.byref(capi.Adamw(**{**good, **kw})), x, 1, 0, S)
    for kw, text in ((dict(bits=16), "32 or in 8"), (dict(total=63), "multiple of 32"), (dict(total=-32), "multiple of 32"), (dict(total=1 << 37), "2^37"),
                     (dict(state=None), "null pointer"), (dict(bits=8), "null pointer"), (dict(state=0x1008), "16-byte"), (dict(master=0x1004), "16-byte"),
                     (dict(beta1=1.0), "beta"), (dict(beta2=-0.1), "beta"), (dict(beta1=NAN), "beta"), (dict(eps=-1.0), "eps"), (dict(eps=NAN), "eps"),
                     (dict(step=0), "counts from 1"), (dict(lr=NAN), "lr"), (dict(weight_decay=float("inf")), "weight_decay"), (dict(total=32), "room"),
                     (dict(master=0x1000), "16-bit")):
        refused(L, call(**kw), text)
    for t, text in ((dict(n=-1), "n must"), (dict(n=1 << 36), "n must"), (dict(start=16), "start"), (dict(start=-32), "start"), (dict(start=32), "room"),
                    (dict(param=None), "null"), (dict(grad=None), "null"), (dict(param_dtype=3), "dtype"), (dict(grad_dtype=-1), "dtype")):
        refused(L, call(t=t), text)
    refused(L, L.dq_adamw_step(None, None, 0, 0, S), "null pointer")
    refused(L, L.dq_adamw_step(ctypes.byref(capi.Adamw(**good)), None, -1, 0, S), "count")


def test_coefficients_refuse(L):
    refused(L, L.dq_adamw_coefficients(N, 1e-3, N, 0.9, 0.999, 0.0, N, P, 0, S), "null pointer")
    refused(L, L.dq_adamw_coefficients(P, 1e-3, N, 0.9, 0.999, 0.0, N, N, 0, S), "null pointer")
    refused(L, L.dq_adamw_coefficients(P, 1e-3, N, 0.9, 1.0, 0.0, N, P, 0, S), "beta")
    refused(L, L.dq_adamw_coefficients(P, NAN, N, 0.9, 0.999, 0.0, N, P, 0, S), "lr")


def test_matrices_refuse(L):
    Z = ctypes.c_uint64(0)

    def quantize(x=P, dtype=1, r=10, c=300, stride=300, columns=0, sign=N, stochastic=0, pool=N, pool_dtype=1, counter=N, codes=P, scales=P):
        return L.dq_mx4_quantize(x, dtype, r, c, stride, columns, sign, stochastic, pool, pool_dtype, Z, Z, counter, codes, scales, 0, S)
    odd, four = ctypes.c_void_p(0x1008), ctypes.c_void_p(0x1004)
    for kw, text in ((dict(dtype=5), "dtype"), (dict(pool=P, stochastic=1, pool_dtype=4), "dtype"), (dict(r=0), "positive"), (dict(c=0), "positive"),
                     (dict(r=1 << 27, c=256), "2^35"), (dict(r=256, c=1 << 27, columns=1, stride=1 << 27), "2^35"),
                     (dict(r=(1 << 27) - 15, c=256), "2^35"), (dict(r=1 << 31, c=1, columns=1), "2^31"), (dict(r=1, c=1 << 31, stride=1 << 31), "2^31"), (dict(stride=299), "stride"), (dict(pool=P), "stochastic"), (dict(counter=P), "step_dev"), (dict(counter=P, pool=P, stochastic=1), "step_dev"),
                     (dict(x=N), "null"), (dict(codes=N), "null"), (dict(scales=N), "null"), (dict(codes=odd), "aligned"), (dict(scales=four), "aligned")):
        refused(L, quantize(**kw), text)
    from dynamiq_sigcomm_artifact_amd.capi import Mx4Matrix
    good = dict(x=0x1000, x_rows=10, x_cols=300, stride=300, codes=0x1000, scales=0x1000, dtype=1)
    for kw, text in ((dict(dtype=5), "dtype"), (dict(x_rows=0), "positive"), (dict(stride=299), "stride"), (dict(rand_pool=0x1000), "stochastic"), (dict(codes=0x1008), "aligned"),
                     (dict(x=None), "null")):
        refused(L, L.dq_mx4_quantize_list((Mx4Matrix * 2)(Mx4Matrix(**good), Mx4Matrix(**{**good, **kw})), 2, 0, S), text)
    refused(L, L.dq_mx4_quantize_list(None, 1, 0, S), "null")
    refused(L, L.dq_mx4_quantize_list(None, -1, 0, S), "count")
    refused(L, L.dq_mx4_dequantize(P, P, P, 9, 1, 1, 0, S), "dtype")
    refused(L, L.dq_mx4_dequantize(P, P, P, 1, 1, 0, 0, S), "positive")
    refused(L, L.dq_mx4_dequantize(P, P, N, 1, 1, 1, 0, S), "null")
    refused(L, L.dq_mx4_dequantize(odd, P, P, 1, 1, 1, 0, S), "aligned")
    refused(L, L.dq_mx4_product(P, P, P, P, P, 9, 1, 1, 1, 0, S), "dtype")
    for m, n, k in ((0, 1, 1), (1, 0, 1), (1, 1, 0), (1 << 27, 1, 1), (1 << 20, 1 << 20, 1)):
        refused(L, L.dq_mx4_product(P, P, P, P, P, 1, m, n, k, 0, S), "positive")
    refused(L, L.dq_mx4_product(P, P, P, P, P, 1, 1, 1, (1 << 24) + 1, 0, S), "2^24")
    refused(L, L.dq_mx4_product(P, P, N, P, P, 1, 1, 1, 1, 0, S), "null")
    refused(L, L.dq_mx4_product(P, P, odd, P, P, 1, 1, 1, 1, 0, S), "aligned")


def test_modules_refuse_host_tensors():
    from dynamiq_sigcomm_artifact_amd import microscale, optimizer
    x = torch.zeros(4, 4)
    with pytest.raises(RuntimeError, match="must live on the GPU"):
        microscale.quantize(x)
    with pytest.raises(RuntimeError, match="must live on the GPU"):
        optimizer.grad_norm([x], work=torch.zeros(4096, dtype=torch.float64), out=torch.zeros(2))
    with pytest.raises(RuntimeError, match="must live on the GPU"):
        optimizer.adamw_step([x], [x], torch.zeros(2, 32), 1)
    with pytest.raises(RuntimeError, match="a tensor argument is required"):
        microscale.quantize(None)
    with pytest.raises(RuntimeError, match="no tensors"):
        optimizer.grad_norm([])
    with pytest.raises(RuntimeError, match="32 or in 8"):
        optimizer.adamw_state([x], 16)
    for call in (lambda: optimizer.grad_norm(x), lambda: optimizer.adamw_state(x), lambda: optimizer.master_weights(x), lambda: optimizer.AdamW(x),
                 lambda: optimizer.AdamW([{"params": x}]), lambda: optimizer.adamw_step(x, [x], x, 1), lambda: optimizer.adamw_step([x], x, x, 1)):
        with pytest.raises(RuntimeError, match="of tensors"):
            call()
    for call in (lambda: optimizer.adamw_state([]), lambda: optimizer.master_weights([])):
        with pytest.raises(RuntimeError, match="no parameters"):
            call()
    assert optimizer.adamw_state(iter([x, x]), 8)[0].shape == (2, 64)
    a, b = microscale.Microscaled(None, None, 2, 5), microscale.Microscaled(None, None, 2, 6)
    with pytest.raises(RuntimeError, match="vectors of 5 and of 6"):
        microscale.product(a, b)
    with pytest.raises(RuntimeError, match="unsupported element dtype"):
        microscale.product(a, a, torch.float64)


def test_optimizer_object_lays_out_its_states():
    from dynamiq_sigcomm_artifact_amd import optimizer
    a, b, c = torch.zeros(5, 7, dtype=torch.bfloat16), torch.zeros(64), torch.ones(1, dtype=torch.float16)
    opt = optimizer.AdamW([{"params": [a, b], "lr": 0.5}, {"params": [c], "weight_decay": 0.0}], lr=0.1, bits=8)
    assert [g["lr"] for g in opt.param_groups] == [0.5, 0.1] and opt.param_groups[1]["weight_decay"] == 0.0
    assert [(p["group"], p["master"] is None, p["state"][0].shape[1], p["state"][1].shape[1]) for p in opt._parts] == [(0, True, 64, 2), (0, False, 64, 2), (1, False, 32, 1)]
    assert opt._parts[2]["master"][:2].tolist() == [1.0, 0.0]
    with pytest.raises(RuntimeError, match="appears twice"):
        optimizer.AdamW([a, a])
    with pytest.raises(RuntimeError, match="no parameters"):
        optimizer.AdamW([])
    other = optimizer.AdamW([a, b], bits=32)
    with pytest.raises(RuntimeError, match="other parameters"):
        other.load_state_dict(opt.state_dict())


def test_reference_codes_and_dither():
    """the tables are torch's float8, and the dither's mean over many steps is that of a uniform number"""
    codes = torch.arange(256, dtype=torch.uint8)
    want = codes.view(torch.float8_e4m3fn).double().numpy()
    got = R.decode8(codes.numpy(), np.full(8, 127, np.uint8))
    assert np.array_equal(got, want, equal_nan=True)
    # one code's way: rounded over 4096 steps, a value comes out as itself to a code's distance / 4096 (one step more or less)
    x = np.full(32, 3.3e-3)
    x[0] = 1.0
    mean = np.zeros(32)
    for t in range(1, 4097):
        c, s = R.encode8(x, R.dither(32, t), False)
        mean += R.decode8(c, s) / 4096
    assert np.all(np.abs(mean - x) <= 2.0 ** -8 * 2 ** -3 * 16 / 4096)


def test_inline_assembly_names_what_it_writes():
    """an assembly statement that writes a register of its own choosing says so, or the compiler may keep a value there"""
    import glob
    import os
    import re
    root = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "dynamiq_sigcomm_artifact_amd", "csrc")
    seen = 0
    for path in sorted(glob.glob(os.path.join(root, "*.hip")) + glob.glob(os.path.join(root, "*.cuh"))):
        for text in re.findall(r"asm volatile\((.*?)\);", open(path).read(), re.S):
            if re.search(r"s_mov_b32 m0\b", text):
                seen += 1
                assert re.search(r':\s*"m0"|,\s*"m0"', text), (os.path.basename(path), text)
    assert seen >= 1


def test_norm_of_nothing_is_refused():
    """None takes no part; a list of nothing else needs a buffer that says where"""
    from dynamiq_sigcomm_artifact_amd import optimizer
    for grads in ([None], [None, None], iter([None])):
        with pytest.raises(RuntimeError, match="no tensors"):
            optimizer.grad_norm(grads)
    with pytest.raises(RuntimeError, match="must live on the GPU"):
        optimizer.grad_norm([None], out=torch.zeros(2))
    p = torch.zeros(4, 6)
    opt = optimizer.AdamW([p, torch.zeros(3)])
    p.grad = torch.ones(6, 4).t()
    got = opt.grads()
    assert got[1] is None and got[0].is_contiguous() and torch.equal(got[0], p.grad)


def test_loaded_hyperparameters_are_copies():
    """what one object does to a value that it has loaded changes neither the saved state nor another object"""
    from dynamiq_sigcomm_artifact_amd import optimizer
    saved = optimizer.AdamW([torch.zeros(5)], lr=torch.full((1,), 0.25)).state_dict()
    a, b = optimizer.AdamW([torch.zeros(5)], lr=0.1), optimizer.AdamW([torch.zeros(5)], lr=0.1)
    a.load_state_dict(saved)
    b.load_state_dict(saved)
    a.param_groups[0]["lr"].fill_(7.0)
    assert float(b.param_groups[0]["lr"]) == 0.25 and float(saved["groups"][0]["lr"]) == 0.25
