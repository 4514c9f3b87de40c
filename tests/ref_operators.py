"""The definitions of the optimizer's and the microscaled operators in 64 bits, on numpy arrays (TEST INFRASTRUCTURE ONLY).

Written from the formats' definitions: values come from tables, neighbours from a search in them."""
import numpy as np

E2M1 = np.array([0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0])
E4M3 = np.array([m / 512.0 if e == 0 else (1 + m / 8.0) * 2.0 ** (e - 7) for e in range(16) for m in range(8)][:127])


def scale_byte(largest, limit, floor_rule=False):
    """byte k + 127: least k with largest <= limit * 2^k, or (floor_rule) floor(log2 largest) - 2"""
    if not np.isfinite(largest):
        return 255
    if largest == 0:
        return 0
    if floor_rule:
        k = int(np.frexp(largest)[1]) - 1 - 2
    else:
        k = int(np.ceil(np.log2(largest / limit))) - 2
        while largest > limit * 2.0 ** k:
            k += 1
    return max(k + 127, 0)


def hadamard32():
    h = np.array([[1.0]])
    for _ in range(5):
        h = np.block([[h, h], [h, -h]])
    return h


def rotate32(blocks, sign):
    """float32 butterflies, stride 1 first, as the format defines them; blocks [..., 32], sign [..., 32] of +-1"""
    x = (blocks * sign).astype(np.float32)
    h = 1
    while h < 32:
        x = x.reshape(x.shape[:-1] + (32 // (2 * h), 2, h)) if x.ndim else x
        a, b = x[..., 0, :], x[..., 1, :]
        x = np.stack((a + b, a - b), axis=-2)
        x = x.reshape(x.shape[:-3] + (32,))
        h *= 2
    return x * np.float32(1 / np.sqrt(32.0))


def quantize4(vectors, sign=None, uniform=None):
    """vectors [rows, n] (any float type) -> values float64 [rows, padded], bytes [rows, blocks]; NaN where a block is not finite"""
    rows, n = vectors.shape
    padded = -(-n // 256) * 256
    x = np.zeros((rows, padded), np.float32)
    x[:, :n] = vectors
    blocks = x.reshape(rows, -1, 32)
    if sign is not None:
        with np.errstate(all="ignore"):
            blocks = rotate32(blocks, np.asarray(sign, np.float32).reshape(1, -1, 32))
    out = np.zeros(blocks.shape)
    scales = np.zeros(blocks.shape[:2], np.uint8)
    u = None if uniform is None else np.asarray(uniform, np.float64).reshape(blocks.shape)
    for r in range(rows):
        for b in range(blocks.shape[1]):
            v = blocks[r, b].astype(np.float64)
            largest = np.max(np.abs(v)) if np.isfinite(v).all() else np.inf
            byte = scale_byte(largest, 6.0, uniform is None)
            scales[r, b] = byte
            if byte == 255:
                out[r, b] = np.nan
                continue
            y = np.abs(v) / 2.0 ** (byte - 127)
            if uniform is None:
                y = np.minimum(y, 6.0)
            at = np.minimum(np.searchsorted(E2M1, y, side="right") - 1, 6)
            share = (y - E2M1[at]) / (E2M1[at + 1] - E2M1[at])
            if uniform is None:
                up = (share > 0.5) | ((share == 0.5) & (at % 2 == 1))
            else:
                up = u[r, b] < share
            out[r, b] = np.copysign(E2M1[at + up], v) * 2.0 ** (byte - 127)
    return out.reshape(rows, padded), scales


def pack4(values, scales):
    """the codes of quantize4's values"""
    rows, padded = values.shape
    y = np.abs(values.reshape(rows, -1, 32)) / 2.0 ** (scales.astype(np.float64) - 127)[:, :, None]
    c = np.searchsorted(E2M1, y.reshape(rows, padded)).astype(np.uint8) | (np.signbit(values).astype(np.uint8) << 3)
    return c[:, 0::2] | (c[:, 1::2] << 4)


def unpack4(codes, scales):
    c = np.stack((codes & 15, codes >> 4), axis=2).reshape(codes.shape[0], -1)
    v = E2M1[c & 7] * np.where(c & 8, -1.0, 1.0)
    up = np.where(scales == 255, np.nan, 2.0 ** (scales.astype(np.float64) - 127))
    return (v.reshape(codes.shape[0], -1, 32) * up[:, :, None]).reshape(v.shape)


def decode8(codes, scales):
    """one row of 8-bit states"""
    c = codes.astype(np.int64)
    v = np.where((c & 127) == 127, np.nan, E4M3[np.minimum(c & 127, 126)]) * np.where(c & 128, -1.0, 1.0)
    up = np.where(scales == 255, np.nan, 2.0 ** (scales.astype(np.float64) - 127))
    return (v.reshape(-1, 32) * up[:, None]).reshape(-1)


def dither(n, step):
    i = np.arange(n, dtype=np.uint64)
    return ((i * np.uint64(0x9E3779B9) + np.uint64(step * 0xB504F333 % 2 ** 32)) % np.uint64(2 ** 32)) >> np.uint64(12)


def scales8(x):
    blocks = x.reshape(-1, 32)
    return np.array([scale_byte(np.max(np.abs(b)) if np.isfinite(b).all() else np.inf, 448.0) for b in blocks], np.uint8)


def magnitudes8(x, d, scales):
    """codes without their sign of magnitudes x, with the blocks' bytes given; above 448 the largest"""
    y = np.minimum(x.reshape(-1, 32) / 2.0 ** (scales.astype(np.float64) - 127)[:, None], 448.0)
    at = np.minimum(np.searchsorted(E4M3, y.reshape(-1), side="right") - 1, 125)
    share = (y.reshape(-1) - E4M3[at]) / (E4M3[at + 1] - E4M3[at])
    return at + (np.floor(share * 2 ** 20) + d >= 2 ** 20)


def encode8(x, d, root):
    """one tensor's moment, padded to blocks: codes and bytes"""
    scales = scales8(x)
    at = magnitudes8(np.abs(x), d, scales)
    if root:
        at = np.where((x > 0) & (at == 0), 1, at)
    return (at | np.where(x < 0, 128, 0)).astype(np.uint8), scales


def adamw(p, g, m, v, t, lr, betas, eps, decay):
    """float64 arrays -> p, m, v"""
    m = betas[0] * m + (1 - betas[0]) * g
    v = betas[1] * v + (1 - betas[1]) * g * g
    p = p * (1 - lr * decay) - lr * (m / (1 - betas[0] ** t)) / (np.sqrt(v / (1 - betas[1] ** t)) + eps)
    return p, m, v
