"""The definitions of the operators between the linear layers in 64 bits, on numpy arrays (TEST INFRASTRUCTURE ONLY)."""
import numpy as np

import ref_operators as R

LAST = {"float16": 127 + 8, "bfloat16": 127 + 120, "float32": 127 + 120}


def compress(x, name):
    """rows of float values -> codes uint8 [rows, 32 b], scale bytes [rows, b] and values [rows, 32 b]; NaN where a block is not finite"""
    rows, cols = x.shape
    b = -(-cols // 32)
    padded = np.zeros((rows, 32 * b))
    padded[:, :cols] = x
    scales = R.scales8(padded.reshape(-1)).reshape(rows, b) if padded.size else np.zeros((rows, b), np.uint8)
    up = np.where(scales == 255, np.nan, 2.0 ** (scales.astype(np.float64) - 127))[:, :, None]
    most = np.where(scales == LAST[name], 240.0, 448.0)[:, :, None]
    with np.errstate(invalid="ignore"):
        y = np.minimum(np.abs(padded.reshape(rows, b, 32)) / up, most)
    at = np.clip(np.searchsorted(R.E4M3, y, side="right") - 1, 0, 125)
    below, above = y - R.E4M3[at], R.E4M3[at + 1] - y
    at = np.where((above < below) | ((above == below) & (at % 2 == 1)), at + 1, at)
    sign = np.signbit(padded.reshape(rows, b, 32))
    values = np.where(sign, -1.0, 1.0) * R.E4M3[at] * up
    return (at | sign * 128).astype(np.uint8).reshape(rows, -1), scales, values.reshape(rows, -1)


def restored(x, name):
    return compress(x, name)[2][:, :x.shape[1]]


def statistics(x, center, eps):
    mean = x.mean(1, keepdims=True) if center else np.zeros((x.shape[0], 1))
    return mean, 1.0 / np.sqrt(((x - mean) ** 2).mean(1, keepdims=True) + eps)


def _times(x, weight, bias):
    x = x if weight is None else x * weight
    return x if bias is None else x + bias


def block(y, residual, gate, s, kept=None):
    """r = residual_scale residual + block_scale gate z, h = norm(r), with what the backward pass takes.  gate: one row for each of y's (or None); s: the settings;
    kept: (r, y) as a backward pass finds them, for its formulas"""
    st_y = statistics(y, s["center"], s["eps"]) if s["after"] else None
    yhat = (y - st_y[0]) * st_y[1] if s["after"] else y
    z = _times(yhat, s["after_weight"], s["after_bias"]) if s["after"] else y
    r = s["block_scale"] * (z if gate is None else gate * z)
    if residual is not None:
        r = r + s["residual_scale"] * residual
    st_r = statistics(r, s["center"], s["eps"])
    h = _times((r - st_r[0]) * st_r[1], s["weight"], s["bias"]) if s["before"] else None
    return h, r, st_r, st_y


def _back(g, xhat, rs, center):
    inner = g - xhat * (g * xhat).mean(1, keepdims=True)
    return rs * (inner - g.mean(1, keepdims=True) if center else inner)


def block_gradients(kept_y, kept_r, st_r, st_y, gate, s, dh, dr_in):
    """dict of the gradients; dgate row by row"""
    out = {}
    dr = np.zeros_like(kept_y) if dr_in is None else dr_in.copy()
    if s["before"] and dh is not None:
        xhat = (kept_r - st_r[0]) * st_r[1]
        out["weight"], out["bias"] = dh * xhat, dh
        dr = dr + _back(dh if s["weight"] is None else dh * s["weight"], xhat, st_r[1], s["center"])
    out["residual"] = s["residual_scale"] * dr
    t = s["block_scale"] * dr
    yhat = (kept_y - st_y[0]) * st_y[1] if s["after"] else kept_y
    z = _times(yhat, s["after_weight"], s["after_bias"]) if s["after"] else kept_y
    if gate is not None:
        out["gate"] = t * z
        t = t * gate
    if s["after"]:
        out["after_weight"], out["after_bias"] = t * yhat, t
        t = _back(t if s["after_weight"] is None else t * s["after_weight"], yhat, st_y[1], s["center"])
    out["y"] = t
    return out


def act(g, kind):
    """the activation and its derivative (the sigmoid as a quotient: from the hyperbolic tangent, 1 + tanh cancels where the sigmoid is small)"""
    with np.errstate(over="ignore"):
        q = g if kind == "silu" else 2 * np.sqrt(2 / np.pi) * (g + 0.044715 * g ** 3)
        s, rest = 1 / (1 + np.exp(-q)), 1 / (1 + np.exp(q))
        dq = 1.0 if kind == "silu" else 2 * np.sqrt(2 / np.pi) * (1 + 3 * 0.044715 * g ** 2)
        return g * s, s + g * s * rest * dq
