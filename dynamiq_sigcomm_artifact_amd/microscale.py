"""4-bit microscaled matrices (E2M1 elements, a power of two per block of 32): quantisation, values, products, and a linear layer
whose forward and backward products are in 4 bits.

The quantiser is the codec's kind applied to the operands of a product: blocks along the axis that the product contracts, an
optional randomized Hadamard transform of each block in front, rounding to nearest or stochastic, from a pool or from the
in-kernel Philox stream.  ``include/dynamiq_eden.h`` (dq_mx4_*) has the format and the rounding to the bit.

Everything runs on the current stream of the tensors' device, returns new tensors and can be recorded into a graph.  A replay draws the random
numbers of the recording, unless step is an int64 tensor [1] on the device, which is read when the kernel runs."""
import torch

from . import capi

_DTYPES = (torch.float16, torch.bfloat16, torch.float32)


def _superchunks(length):
    return -(-length // 256)


class Microscaled(object):
    """``rows`` vectors of ``cols`` elements each: ``codes`` uint8 [rows, 128 s], two elements a byte (the first in the low half), and
    ``scales`` uint8 [rows, 8 s], a byte k + 127 for the factor 2^k of every 32 elements (255: NaN), with s = ceil(cols / 256) and zeros
    behind the cols-th element.  ``cols`` is the axis that products contract."""
    __slots__ = ("codes", "scales", "rows", "cols")

    def __init__(self, codes, scales, rows, cols):
        self.codes, self.scales, self.rows, self.cols = codes, scales, int(rows), int(cols)

    @property
    def shape(self):
        return (self.rows, self.cols)

    def __repr__(self):
        return "Microscaled(%d x %d)" % (self.rows, self.cols)


def quantize(x, columns=False, sign=None, rand_pool=None, seed=None, step=0):
    """x [r, c] (fp16, bf16 or fp32; the elements of a row consecutive) -> Microscaled: its rows, or with ``columns`` its columns, as vectors.

    sign: int32 [>= 8 s], the packed signs of capi.pack_signs or capi.rand_diag_bits, one per element of a vector: every block of 32 is rotated,
    H (s x) / sqrt(32).  The product of two matrices that are rotated with the same signs is that of the matrices.
    rand_pool: uniform values in [0, 1), [vectors, 256 s], for stochastic rounding; or seed (and step, a number or an int64 tensor [1]) for the
    in-kernel stream, the codec's, whose values are the 128 odd multiples of 1/256: elements up to 2^k / 512, k of their block, become 0 in every draw,
    and the mean of the draws of another is off by up to 1/256 of the distance between its neighbours (a float32 pool has 24 bits);
    neither: to nearest, ties to even.  Nothing here but linear() is differentiated."""
    codes, scales = capi.host().mx4_quantize(x, columns, sign, rand_pool, seed, step)
    r, c = x.shape
    return Microscaled(codes, scales, c if columns else r, r if columns else c)


def _like(dtype):
    if dtype not in _DTYPES:
        raise RuntimeError("unsupported element dtype %s" % dtype)
    return _EMPTY[dtype]


_EMPTY = {dtype: torch.empty(0, dtype=dtype) for dtype in _DTYPES}


def dequantize(q, dtype=torch.float32):
    """the values of a Microscaled, [rows, cols]"""
    return capi.host().mx4_dequantize(q.codes, q.scales, q.rows, q.cols, _like(dtype))


def product(a, b, dtype=torch.bfloat16):
    """[a.rows, b.rows]: every vector of a times every vector of b, summed in float32"""
    if a.cols != b.cols:
        raise RuntimeError("product: vectors of %d and of %d elements" % (a.cols, b.cols))
    return capi.host().mx4_product(a.codes, a.scales, b.codes, b.scales, a.rows, b.rows, a.cols, _like(dtype))


def linear(x, weight, sign=None, rand_pool=None, seed=None, step=0):
    """y = x weight^T for x [..., k] and weight [n, k], all three products of a training step in 4 bits:

      y  = Q(x) Q(weight)^T             along k, to nearest
      dx = S(dy R) (Q(weight^T R))^T    along n
      dw = S(dy^T R) (Q(x^T R))^T       along the tokens

    Q rounds to nearest (and what it makes of x and weight is off by that), S stochastically, so that the rounding of dy has no bias but for the resolution
    of the random numbers (quantize), R is the rotation of every block of 32 with the given signs, which spreads outliers over their block and cancels in the product.

    sign: (signs of n, signs of the tokens), packed; None leaves R out.  rand_pool: (pool [tokens, n padded to 256], pool [n, tokens padded to
    256]), checked here where their gradient is wanted, or seed and step: then every call needs a step of its own, below 2^63 (the gradient's rows draw at step, its columns at step + 2^63).
    With neither the gradients are rounded to nearest, too.  A step on the device stays as it is until the backward pass has run.  The gradients
    cannot be differentiated again."""
    signs, pools = sign or (None, None), rand_pool or (None, None)
    return capi.host().mx4_linear(x, weight, signs[0], signs[1], pools[0], pools[1], seed, step)
