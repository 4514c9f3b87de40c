"""What lies between the linear layers of a training step, and what their backward passes keep: norms around a block fused with its gate and
residual, the gated activation, and activations held in 8 bits.

A case is a dict of plain values; ``op`` names the operator and the other keys size it:

  checkpoint  an activation cut to 8 bits and brought back
  columns     the columns of such a checkpoint in 4-bit microscaled blocks, what a weight's gradient takes
  linear      a linear layer's training step in 4 bits that keeps its input in 8: output and both gradients
  norm        r = residual + gate * norm(y), h = norm(r); with ``train`` the gradients, with ``eight`` what they take of r and y in 8 bits
  gated       act(g) * u of rows [g, u]; ``train`` and ``eight`` as above

The formats.  8 bits: blocks of 32 along a row share a power of two 2^k (a byte k + 127), the least that holds the block's largest below 448;
elements are E4M3, rounded to nearest, ties to even.  One buffer: the codes of all rows, each padded with zeros to whole blocks, then the bytes.
4 bits: blocks of 32 along the contraction, k = floor(log2 max) - 2, elements E2M1 (0, 0.5, 1, 1.5, 2, 3, 4, 6 and a sign) to nearest, ties to even,
saturating; stochastic rounding takes the least k with max <= 6 2^k.  With signs s a block x becomes H(s x) / sqrt(32) before, H the
Walsh-Hadamard matrix.
A norm is v / sqrt(mean(v^2) + eps) * w, with ``center`` (v - mean) / sqrt(var + eps) * w + b.  r is rounded to the residual stream's type, h to y's;
a checkpoint is that of the rounded values.
"""
import math

import torch
from torch.nn.functional import pad

own = False

DEVICE = "cuda:0"
DTYPES = {"fp32": torch.float32, "bf16": torch.bfloat16, "fp16": torch.float16}
EPS = 1e-5


# ---- cases --------------------------------------------------------------------------------------------------------

def listed():
    return [
        # a short, odd batch's activations; and the hidden ones of 8192 tokens in an 8B model's block
        {"name": "checkpoint odd", "op": "checkpoint", "dtype": "fp16", "rows": 333, "cols": 1000},
        {"name": "checkpoint hidden", "op": "checkpoint", "dtype": "bf16", "rows": 8192, "cols": 14336},
        # what the weights' gradients of the two widths take of them
        {"name": "columns odd", "op": "columns", "rows": 333, "cols": 1000, "rotate": False},
        {"name": "columns hidden", "op": "columns", "rows": 8192, "cols": 14336, "rotate": True},
        # training steps of a linear layer: a small odd one, and one of an 8B model's
        {"name": "linear odd", "op": "linear", "dtype": "fp16", "m": 333, "n": 776, "k": 1000},
        {"name": "linear layer", "op": "linear", "dtype": "bf16", "m": 4096, "n": 14336, "k": 4096},
        # one token: latency
        {"name": "norm token", "op": "norm", "dtype": "bf16", "stream": "bf16", "rows": 1, "cols": 4096, "center": False, "after": False, "groups": 0, "train": False, "eight": False},
        # a 124M-parameter model's width, centred norms with biases, a gate that is learnt per channel, the residual stream in 32 bits, an odd number of tokens
        {"name": "norm centred", "op": "norm", "dtype": "bf16", "stream": "fp32", "rows": 4095, "cols": 768, "center": True, "after": False, "groups": 1, "train": True, "eight": False},
        # an 8B model's training step: the residual added, the next block's norm, what the backward pass takes in 8 bits
        {"name": "norm layer", "op": "norm", "dtype": "bf16", "stream": "bf16", "rows": 8192, "cols": 4096, "center": False, "after": False, "groups": 0, "train": True, "eight": True},
        # norms on both sides of the residual, a gate for each of 16 sequences
        {"name": "norm sandwich", "op": "norm", "dtype": "bf16", "stream": "bf16", "rows": 8192, "cols": 4096, "center": False, "after": True, "groups": 16, "train": True, "eight": False},
        # one token, and a training step that keeps its inputs in 8 bits
        {"name": "gated token", "op": "gated", "dtype": "bf16", "kind": "silu", "rows": 1, "cols": 14336, "train": False, "eight": False},
        {"name": "gated hidden", "op": "gated", "dtype": "bf16", "kind": "silu", "rows": 8192, "cols": 14336, "train": True, "eight": True},
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    op = rng.choice(("checkpoint", "columns", "linear", "norm", "norm", "gated"))
    dtype = rng.choice(("fp32", "bf16", "fp16"))
    if op == "checkpoint":
        return {"op": op, "dtype": dtype, "rows": _log(rng, 1, 8192), "cols": _log(rng, 16, 14336)}
    if op == "columns":
        return {"op": op, "rows": _log(rng, 1, 8192), "cols": _log(rng, 16, 14336), "rotate": rng.random() < 0.5}
    if op == "linear":
        return {"op": op, "dtype": rng.choice(("bf16", "fp16")), "m": _log(rng, 16, 4096), "n": _log(rng, 128, 8192), "k": _log(rng, 128, 4096)}
    train = rng.random() < 0.7
    if op == "gated":
        return {"op": op, "dtype": dtype, "kind": rng.choice(("silu", "gelu_tanh")), "rows": _log(rng, 1, 4096), "cols": _log(rng, 64, 14336), "train": train,
                "eight": train and rng.random() < 0.5}
    after = rng.random() < 0.5
    each = rng.choice((0, 0, 1, 2, 3))
    rows, groups = _log(rng, 1, 4096), 0
    if each == 1:
        groups = 1
    elif each == 2:     # a gate for every token
        groups = rows
    elif each == 3:     # ... for every sequence
        groups = _log(rng, 1, min(rows, 64))
        rows = rows // groups * groups
    return {"op": op, "dtype": dtype, "stream": rng.choice((dtype, dtype, "fp32", "none")), "rows": rows, "cols": _log(rng, 128, 8192), "center": rng.random() < 0.5,
            "after": after, "groups": groups, "train": train, "eight": train and dtype != "fp32" and rng.random() < 0.5}


def _padded(n, to):
    return -(-n // to) * to


# ---- inputs -------------------------------------------------------------------------------------------------------

def _matrix(rows, cols, g, dtype):
    """activations: columns of different scales, a few of them large"""
    scale = torch.exp(torch.randn(cols, generator=g, device=DEVICE))
    return torch.randn(rows, cols, generator=g, device=DEVICE).mul_(scale).to(dtype)


def _gradient(rows, cols, g, dtype):
    """heavy-tailed"""
    return torch.randn(rows, cols, generator=g, device=DEVICE).mul_(torch.exp(torch.randn(rows, cols, generator=g, device=DEVICE))).mul_(1e-3).to(dtype)


def _signs(n, g):
    """+-1 per place, and the same as one bit each, set where negative"""
    negative = torch.rand(_padded(n, 256), generator=g, device=DEVICE) < 0.5
    words = (negative.view(-1, 32).long() << torch.arange(32, device=DEVICE)).sum(1)
    return 1.0 - 2.0 * negative.float(), words.to(torch.int32)


def _pool(rows, n, g):
    """uniform in [0, 1), in 16 bits as the codec's pools are; multiples of 1/256, so that none is rounded to 1"""
    return torch.randint(0, 256, (rows, _padded(n, 256)), generator=g, device=DEVICE, dtype=torch.uint8).float().mul_(1 / 256).to(torch.bfloat16)


def _prepare_checkpoint(case, g):
    return {"x": _matrix(case["rows"], case["cols"], g, DTYPES[case["dtype"]])}


def _prepare_columns(case, g):
    codes, scales = _encode8(_matrix(case["rows"], case["cols"], g, torch.bfloat16))
    return {"data": torch.cat((codes.view(-1), scales.view(-1))), "signs": _signs(case["rows"], g) if case["rotate"] else (None, None)}


def _prepare_linear(case, g):
    m, n, k, dtype = case["m"], case["n"], case["k"], DTYPES[case["dtype"]]
    return {"x": _matrix(m, k, g, dtype), "w": torch.randn(n, k, generator=g, device=DEVICE).mul_(0.02).to(dtype),
            "dy": _gradient(m, n, g, dtype), "signs": (_signs(n, g), _signs(m, g)), "pools": (_pool(m, n, g), _pool(n, m, g))}


def _prepare_norm(case, g):
    rows, cols, dtype = case["rows"], case["cols"], DTYPES[case["dtype"]]
    stream = dtype if case["stream"] == "none" else DTYPES[case["stream"]]

    def weights(mean, spread):
        return torch.randn(cols, generator=g, device=DEVICE).mul_(spread).add_(mean).to(dtype)
    s = {"y": _matrix(rows, cols, g, dtype), "residual": None if case["stream"] == "none" else _matrix(rows, cols, g, stream), "weight": weights(1.0, 0.1),
         "bias": weights(0.0, 0.1) if case["center"] else None, "after_weight": weights(1.0, 0.1) if case["after"] else None,
         "after_bias": weights(0.0, 0.1) if case["center"] and case["after"] else None, "gate": None}
    if case["groups"]:
        s["gate"] = torch.randn(case["groups"], cols, generator=g, device=DEVICE).mul_(0.2).add_(0.5).to(dtype)
    if case["train"]:
        s["dh"], s["dr"] = _gradient(rows, cols, g, dtype), _gradient(rows, cols, g, stream)
    return s


def _prepare_gated(case, g):
    dtype = DTYPES[case["dtype"]]
    # (what a linear layer with both halves of the weight gives)
    s = {"x": torch.randn(case["rows"], 2 * case["cols"], generator=g, device=DEVICE).mul_(1.5).to(dtype)}
    if case["train"]:
        s["da"] = _gradient(case["rows"], case["cols"], g, dtype)
    return s


# ---- the plain forms ----------------------------------------------------------------------------------------------

def _shared(largest, top, lift):
    """the byte k + 127 of a block: k = floor(log2 largest) - top, one more where the mantissa in [1, 2) is above `lift`"""
    mantissa, exponent = torch.frexp(largest)
    k = exponent - (1 + top) + (2.0 * mantissa > lift).int()
    return torch.where(largest > 0, (k + 127).clamp(0, 254), 0)


def _down(code):
    """2^-k, exact"""
    return ((254 - code) << 23).view(torch.float32)


def _up(code):
    """2^k, exact"""
    return torch.where(code > 0, (code << 23).view(torch.float32), 2.0 ** -127)


def _encode8(x):
    """codes [rows, 32 b] and scale bytes [rows, b]"""
    x = pad(x.float(), (0, -x.shape[1] % 32))
    rows, n = x.shape
    x = x.reshape(rows, n // 32, 32)
    code = _shared(x.abs().amax(2), 8, 1.75)
    return (x * _down(code)[:, :, None]).to(torch.float8_e4m3fn).view(rows, n).view(torch.uint8), code.to(torch.uint8)


def _decode8(codes, scales, cols):
    y = codes.view(torch.float8_e4m3fn).float().view(codes.shape[0], -1, 32) * _up(scales.int())[:, :, None]
    return y.view(codes.shape)[:, :cols]


def _parts8(data, rows, cols):
    """codes and scale bytes of a checkpoint's buffer"""
    n = rows * _padded(cols, 32)
    return data[:n].view(rows, -1), data[n:].view(rows, -1)


def _as_values(codes, scales):
    return {"codes": codes.view(torch.float8_e4m3fn), "scales": scales.view(torch.float8_e8m0fnu)}


def _butterfly(x, h):
    a, b = x.view(-1, 16 // h, 2, h).unbind(2)
    return torch.stack((a + b, a - b), 2)


def _blocks4(x, sign, uniform):
    """the values of the rows of x in 4-bit blocks, padded to superchunks"""
    x = pad(x.float(), (0, -x.shape[1] % 256)).contiguous()
    rows, n = x.shape
    if sign is not None:
        x = _butterfly(_butterfly(_butterfly(_butterfly(_butterfly(x * sign, 1), 2), 4), 8), 16) * (1 / math.sqrt(32))
    x = x.reshape(rows, n // 32, 32)
    y = x.abs()
    code = _shared(y.amax(2), 2, 2.0 if uniform is None else 1.5)
    y = y * _down(code)[:, :, None]
    step = torch.where(y < 2, 0.5, torch.where(y < 4, 1.0, 2.0))
    if uniform is None:
        q = ((y / step).round() * step).clamp(max=6)
    else:
        low = (y / step).floor()
        q = (low + (uniform.float().view(rows, n // 32, 32) < y / step - low).float()) * step
    return (torch.where(x < 0, -q, q) * _up(code)[:, :, None]).view(rows, n)


def _plain_checkpoint(s):
    codes, scales = _encode8(s["x"])
    return {**_as_values(codes, scales), "values": _decode8(codes, scales, s["x"].shape[1]).to(s["x"].dtype)}


def _plain_columns(s, rows, cols):
    x = _decode8(*_parts8(s["data"], rows, cols), cols)
    return _blocks4(x.t(), s["signs"][0], None)[:, :rows].to(torch.bfloat16)


def _plain_linear(s):
    x, w, dy = s["x"], s["w"], s["dy"]
    (sn, _), (sm, _) = s["signs"]
    y = _blocks4(x, None, None) @ _blocks4(w, None, None).t()
    kept = _decode8(*_encode8(x), x.shape[1])
    dx = _blocks4(dy, sn, s["pools"][0]) @ _blocks4(w.t(), sn, None).t()
    dw = _blocks4(dy.t(), sm, s["pools"][1]) @ _blocks4(kept.t(), sm, None).t()
    return {"y": y.to(x.dtype), "dx": dx.to(x.dtype), "dw": dw.to(w.dtype)}


def _statistics(x, center):
    mean = x.mean(1, keepdim=True) if center else 0.0
    return mean, torch.rsqrt((x - mean).square().mean(1, keepdim=True) + EPS)


def _affine(x, weight, bias):
    return x * weight.float() if bias is None else x * weight.float() + bias.float()


def _through_norm(g, xhat, rs, center):
    """the gradient of what was normalised, from that of xhat"""
    inner = g - xhat * (g * xhat).mean(1, keepdim=True)
    return rs * (inner - g.mean(1, keepdim=True) if center else inner)


def _plain_norm(s, case):
    y, residual, center = s["y"].float(), s["residual"], case["center"]
    dtype, stream, rows, cols = s["y"].dtype, s["y"].dtype if residual is None else residual.dtype, case["rows"], case["cols"]
    gate = None if s["gate"] is None else s["gate"].float().repeat_interleave(rows // case["groups"], 0)

    def block(y, mean, rs):
        yhat = (y - mean) * rs
        return yhat, _affine(yhat, s["after_weight"], s["after_bias"]) if case["after"] else y
    y_mean, y_rs = _statistics(y, center) if case["after"] else (0.0, 1.0)
    z = block(y, y_mean, y_rs)[1]
    r = z if gate is None else z * gate
    if residual is not None:
        r = residual.float() + r
    mean, rs = _statistics(r, center)
    h = _affine((r - mean) * rs, s["weight"], s["bias"]).to(dtype)
    r = r.to(stream)
    out = {"h": h, "r": r}
    if case["eight"]:
        out.update(_as_values(*_encode8(h)))
    if not case["train"]:
        return out
    kept = _decode8(*_encode8(r), cols) if case["eight"] else r.float()
    kept_y = _decode8(*_encode8(s["y"]), cols) if case["eight"] else y
    dh, xhat = s["dh"].float(), (kept - mean) * rs
    dr = _through_norm(dh * s["weight"].float(), xhat, rs, center) + s["dr"].float()
    if residual is not None:
        out["dresidual"] = dr.to(stream)
    out["dweight"] = (dh * xhat).sum(0).to(dtype)
    if center:
        out["dbias"] = dh.sum(0).to(dtype)
    yhat, z = block(kept_y, y_mean, y_rs)
    if gate is not None:
        out["dgate"] = (dr * z).view(case["groups"], -1, cols).sum(1).to(dtype)
        dr = dr * gate
    if case["after"]:
        out["dafter_weight"] = (dr * yhat).sum(0).to(dtype)
        if center:
            out["dafter_bias"] = dr.sum(0).to(dtype)
        dr = _through_norm(dr * s["after_weight"].float(), yhat, y_rs, center)
    out["dy"] = dr.to(dtype)
    return out


def _slope(g, kind):
    """q and its derivative, of act(g) = g sigmoid(q(g))"""
    if kind == "silu":
        return g, 1.0
    c = 2 * math.sqrt(2 / math.pi)
    return c * (g + 0.044715 * g * g * g), c * (1 + 3 * 0.044715 * g * g)


def _plain_gated(s, case):
    x, cols = s["x"], case["cols"]
    g, u = x[:, :cols].float(), x[:, cols:].float()
    a = (g * torch.sigmoid(_slope(g, case["kind"])[0]) * u).to(x.dtype)
    out = {"a": a}
    if case["eight"]:
        out.update(_as_values(*_encode8(a)))
        g, u = _decode8(*_encode8(g), cols), _decode8(*_encode8(u), cols)
    if case["train"]:
        da = s["da"].float()
        q, dq = _slope(g, case["kind"])
        p = torch.sigmoid(q)
        out["dx"] = torch.cat((da * u * (p + g * dq * (p * torch.sigmoid(-q))), da * g * p), 1).to(x.dtype)
    return out


# ---- one pass -----------------------------------------------------------------------------------------------------

_PREPARE = {"checkpoint": _prepare_checkpoint, "columns": _prepare_columns, "linear": _prepare_linear, "norm": _prepare_norm, "gated": _prepare_gated}


def prepare(case, seed):
    return {"case": case, **_PREPARE[case["op"]](case, torch.Generator(device=DEVICE).manual_seed(seed))}


def run(state):
    case, op = state["case"], state["case"]["op"]
    if own:
        return _own(case, op, state)
    if op == "checkpoint":
        return _plain_checkpoint(state)
    if op == "columns":
        return _plain_columns(state, case["rows"], case["cols"])
    if op == "linear":
        return _plain_linear(state)
    return _plain_norm(state, case) if op == "norm" else _plain_gated(state, case)


def _own(case, op, s):
    from dynamiq_sigcomm_artifact_amd import activations, microscale
    if op == "checkpoint":
        c = activations.compress(s["x"])
        return {**_as_values(c.codes, c.scales), "values": activations.restore(c, s["x"].dtype)}
    if op == "columns":
        c = activations.Checkpoint(s["data"], case["rows"], case["cols"])
        return microscale.dequantize(microscale.quantize(c, columns=True, sign=s["signs"][1]), torch.bfloat16)
    if op == "linear":
        x, w = s["x"].detach().requires_grad_(), s["w"].detach().requires_grad_()
        y = microscale.linear(x, w, sign=(s["signs"][0][1], s["signs"][1][1]), rand_pool=s["pools"], checkpoint=True)
        dx, dw = torch.autograd.grad(y, (x, w), s["dy"])
        return {"y": y.detach(), "dx": dx, "dw": dw}
    if op == "gated":
        x = s["x"].detach().requires_grad_(case["train"])
        a = activations.gated(x, kind=case["kind"], checkpoint=case["eight"])
        a, c = a if case["eight"] else (a, None)
        out = {"a": a.detach()}
        if c is not None:
            out.update(_as_values(c.codes, c.scales))
        if case["train"]:
            out["dx"], = torch.autograd.grad(a, x, s["da"])
        return out
    names = [k for k in ("residual", "weight", "bias", "gate", "after_weight", "after_bias", "y") if s[k] is not None]
    leaf = dict.fromkeys(("residual", "weight", "bias", "gate", "after_weight", "after_bias", "y"))
    leaf.update({k: s[k].detach().requires_grad_(case["train"]) for k in names})
    gate = leaf["gate"] if case["groups"] <= 1 or case["groups"] == case["rows"] else leaf["gate"].view(case["groups"], 1, -1)
    shape = (case["groups"], -1, case["cols"]) if gate is not None and gate.dim() == 3 else (case["rows"], case["cols"])
    got = activations.residual_norm(leaf["y"].view(shape), None if leaf["residual"] is None else leaf["residual"].view(shape), leaf["weight"], leaf["bias"],
                                    gate=gate, after=case["after"], after_weight=leaf["after_weight"], after_bias=leaf["after_bias"], center=case["center"],
                                    eps=EPS, checkpoint=case["eight"])
    h, r = got[0], got[1]
    flat = (case["rows"], case["cols"])
    out = {"h": h.detach().view(flat), "r": r.detach().view(flat)}
    if case["eight"]:
        out.update(_as_values(got[2].codes, got[2].scales))
    if case["train"]:
        grads = torch.autograd.grad((h, r), [leaf[k] for k in names], (s["dh"].view(shape), s["dr"].view(shape)))
        out.update({"d" + k: v for k, v in zip(names, grads)})
    return out


# ---- what a pass cannot do without ------------------------------------------------------------------------------------

def work(case):
    """a backward pass comes long after its forward one: what the one has kept the other reads"""
    op, eight = case["op"], 33 / 32
    if op == "columns":
        n = case["rows"] * case["cols"]
        return {"bytes": (eight + 2) * n, "flops": (4 + 6 * case["rotate"]) * n}
    size = DTYPES[case["dtype"]].itemsize
    if op == "linear":
        m, n, k = case["m"], case["n"], case["k"]
        return {"bytes": size * (2 * m * k + 2 * n * k + 2 * m * n) + 4 * m * n + 2 * eight * m * k, "flops": 6 * m * n * k}
    n = case["rows"] * case["cols"]
    if op == "checkpoint":
        return {"bytes": (2 * size + 2 * eight) * n, "flops": 6 * n}
    if op == "gated":
        moved = 3 * size + (3 * size if case["train"] else 0)
        if case["train"]:
            moved += 5 * eight if case["eight"] else 2 * size
        return {"bytes": moved * n, "flops": (10 + 20 * case["train"]) * n}
    residual = 0 if case["stream"] == "none" else DTYPES[case["stream"]].itemsize
    stream, gates = residual or size, size * case["cols"] * case["groups"]
    moved = 2 * size + residual + stream
    if case["train"]:
        needs_y = case["after"] or case["groups"] > 0
        # dh, dr -> dy, dresidual (which are the same where nothing lies between); r and y
        moved += size + stream + size + (residual if needs_y or residual != size else 0)
        moved += (eight * (3 + 2 * needs_y) if case["eight"] else stream + size * needs_y)
        gates *= 3
    return {"bytes": moved * n + gates, "flops": (8 + 24 * case["train"]) * n}


# ---- the definitions in 64 bits -----------------------------------------------------------------------------------------

_E2M1 = (0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0)
_E4M3 = tuple((c & 7) / 512 if c < 8 else (1 + (c & 7) / 8) * 2.0 ** ((c >> 3) - 7) for c in range(127))


def _power(k):
    """2^k, exact (a device's power function need not be)"""
    return (k.long() + 1023 << 52).view(torch.float64)


def _exact_exponent(largest, limit):
    """the least k >= -127 with largest <= limit 2^k, and the exponent of the byte 0 for an empty block"""
    k = torch.ceil(torch.log2(torch.where(largest > 0, largest, 1.0) / limit))
    k = torch.where(largest > limit * _power(k), k + 1, torch.where(largest <= limit * _power(k - 1), k - 1, k))
    return torch.where(largest > 0, k.clamp(min=-127.0), -127.0)


def _exact_nearest(y, table):
    """the nearest of the table's values, of the even index where two are as near"""
    grid = torch.tensor(table, dtype=torch.float64, device=DEVICE)
    at = (torch.searchsorted(grid, y.contiguous(), right=True) - 1).clamp(max=len(table) - 2)
    below, above = y - grid[at], grid[at + 1] - y
    return grid[torch.where((above < below) | ((above == below) & (at % 2 == 1)), at + 1, at)]


def _exact8(x):
    """values in units of the scale [rows, padded], the scales [rows, b], and the values [rows, cols]"""
    cols = x.shape[1]
    x = pad(x.double(), (0, -cols % 32))
    y = x.abs().view(x.shape[0], -1, 32)
    k = _exact_exponent(y.amax(2), 448.0)
    q = _exact_nearest(y / _power(k)[:, :, None], _E4M3).view(x.shape)
    q = torch.where(x < 0, -q, q)
    return q, _power(k), (q.view(y.shape) * _power(k)[:, :, None]).view(x.shape)[:, :cols]


def _exact4(x, sign, uniform):
    x = pad(x.double(), (0, -x.shape[1] % 256)).contiguous()
    rows, n = x.shape
    x = x.reshape(rows, -1, 32)
    if sign is not None:
        i = torch.arange(32, device=DEVICE)
        both = i[:, None] & i[None, :]
        odd = (both ^ both >> 1 ^ both >> 2 ^ both >> 3 ^ both >> 4) & 1
        x = ((x * sign.double().view(-1, 32)) @ (1.0 - 2.0 * odd.double())) / math.sqrt(32.0)
    y = x.abs()
    largest = y.amax(2)
    if uniform is None:
        k = torch.where(largest > 0, torch.frexp(largest)[1].double() - 3.0, -127.0)
        q = _exact_nearest((y / _power(k)[:, :, None]).clamp(max=6.0), _E2M1)
    else:
        k = _exact_exponent(largest, 6.0)
        y = y / _power(k)[:, :, None]
        grid = torch.tensor(_E2M1, dtype=torch.float64, device=DEVICE)
        at = (torch.searchsorted(grid, y.contiguous(), right=True) - 1).clamp(max=6)
        share = (y - grid[at]) / (grid[at + 1] - grid[at])
        q = grid[torch.where(uniform.double().view(rows, -1, 32) < share, at + 1, at)]
    q = q * _power(k)[:, :, None]
    return torch.where(x < 0, -q, q).view(rows, n)


def _exact_norm(case, s):
    y, residual, rows, cols, center = s["y"].double(), s["residual"], case["rows"], case["cols"], case["center"]
    dtype, stream = s["y"].dtype, s["y"].dtype if residual is None else residual.dtype
    per = torch.arange(rows, device=DEVICE) // (rows // case["groups"]) if case["groups"] else None

    def moments(x):
        mean = x.sum(1, keepdim=True) / cols if center else torch.zeros(rows, 1, dtype=torch.float64, device=DEVICE)
        return mean, 1.0 / torch.sqrt((x - mean).pow(2).sum(1, keepdim=True) / cols + EPS)

    def scaled(xhat, weight, bias):
        v = xhat * weight.double()
        return v if bias is None else v + bias.double()
    y_of, r_of = moments(y) if case["after"] else None, None
    z = scaled((y - y_of[0]) * y_of[1], s["after_weight"], s["after_bias"]) if case["after"] else y
    r = z if per is None else s["gate"].double()[per] * z
    r = r if residual is None else r + residual.double()
    r_of = moments(r)
    h = scaled((r - r_of[0]) * r_of[1], s["weight"], s["bias"])
    out = {"h": h, "r": r}
    kept, kept_y = r.to(stream).double(), y
    if case["eight"]:
        out["codes"], out["scales"], _ = _exact8(h.to(dtype))
        kept, kept_y = _exact8(kept)[2], _exact8(y)[2]
    if not case["train"]:
        return out

    def back(g, xhat, rs):
        inner = g - xhat * (g * xhat).sum(1, keepdim=True) / cols
        return (inner - g.sum(1, keepdim=True) / cols if center else inner) * rs
    dh, xhat = s["dh"].double(), (kept - r_of[0]) * r_of[1]
    dr = s["dr"].double() + back(dh * s["weight"].double(), xhat, r_of[1])
    if residual is not None:
        out["dresidual"] = dr
    out["dweight"] = (dh * xhat).sum(0)
    if center:
        out["dbias"] = dh.sum(0)
    yhat = (kept_y - y_of[0]) * y_of[1] if case["after"] else kept_y
    z = scaled(yhat, s["after_weight"], s["after_bias"]) if case["after"] else yhat
    if per is not None:
        out["dgate"] = torch.zeros(case["groups"], cols, dtype=torch.float64, device=DEVICE).index_add_(0, per, dr * z)
        dr = dr * s["gate"].double()[per]
    if case["after"]:
        out["dafter_weight"] = (dr * yhat).sum(0)
        if center:
            out["dafter_bias"] = dr.sum(0)
        dr = back(dr * s["after_weight"].double(), yhat, y_of[1])
    out["dy"] = dr
    return out


def _exact_gated(case, s):
    cols, x = case["cols"], s["x"].double()

    def act(g):
        """the activation and its derivative, from the hyperbolic tangent"""
        if case["kind"] == "silu":
            t = torch.tanh(g / 2)
            return g * (1 + t) / 2, (1 + t) / 2 + g * (1 - t) * (1 + t) / 4
        k = math.sqrt(2 / math.pi)
        t = torch.tanh(k * (g + 0.044715 * g.pow(3)))
        return g * (1 + t) / 2, (1 + t) / 2 + g * (1 - t) * (1 + t) / 2 * k * (1 + 3 * 0.044715 * g.pow(2))
    g, u = x[:, :cols], x[:, cols:]
    a = act(g)[0] * u
    out = {"a": a}
    if case["eight"]:
        out["codes"], out["scales"], _ = _exact8(a.to(s["x"].dtype))
        g, u = _exact8(g)[2], _exact8(u)[2]
    if case["train"]:
        value, slope = act(g)
        da = s["da"].double()
        out["dx"] = torch.cat((da * u * slope, da * value), 1)
    return out


def exact(case, seed):
    s = prepare(case, seed)
    op = case["op"]
    if op == "checkpoint":
        codes, scales, values = _exact8(s["x"])
        return {"codes": codes, "scales": scales, "values": values}
    if op == "columns":
        n = case["rows"] * _padded(case["cols"], 32)
        grid = torch.tensor(_E4M3 + (math.nan,) + tuple(-v for v in _E4M3) + (math.nan,), dtype=torch.float64, device=DEVICE)
        x = grid[s["data"][:n].long()].view(case["rows"], -1, 32) * _power(s["data"][n:].view(case["rows"], -1, 1).long() - 127)
        return _exact4(x.view(case["rows"], -1)[:, :case["cols"]].t(), s["signs"][0], None)[:, :case["rows"]]
    if op == "norm":
        return _exact_norm(case, s)
    if op == "gated":
        return _exact_gated(case, s)
    (sn, _), (sm, _) = s["signs"]
    x, w, dy = s["x"], s["w"], s["dy"]
    return {"y": _exact4(x, None, None) @ _exact4(w, None, None).t(),
            "dx": (_exact4(dy, sn, s["pools"][0]) @ _exact4(w.t(), sn, None).t())[:, :case["k"]],
            "dw": (_exact4(dy.t(), sm, s["pools"][1]) @ _exact4(_exact8(x)[2].t(), sm, None).t())[:, :case["k"]]}
