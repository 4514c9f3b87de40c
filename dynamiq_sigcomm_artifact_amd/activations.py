"""What lies between a training step's linear layers, and what their backward passes keep: activations in 8 bits.

A backward pass needs what its forward pass has seen: in 16 bits that is most of a training step's memory.  A Checkpoint holds it in E4M3 with a power of two for
every 32 elements, 33/32 byte an element, and the layers here and in ``microscale`` read it there; ``include/dynamiq_eden.h`` (dq_checkpoint_*) has the format to the bit.

Everything runs on the current stream of the tensors' device, returns new tensors and can be recorded into a graph."""
import torch

from . import capi

_EMPTY = {dtype: torch.empty(0, dtype=dtype) for dtype in (torch.float16, torch.bfloat16, torch.float32)}


class Checkpoint(object):
    """``rows`` x ``cols`` elements in ``data``, uint8 [rows * 33 b] with b = ceil(cols / 32): the codes of all rows, each padded to whole blocks of 32, and behind them
    a byte k + 127 for every block's factor 2^k (255: NaN)."""
    __slots__ = ("data", "rows", "cols")

    def __init__(self, data, rows, cols):
        self.data, self.rows, self.cols = data, int(rows), int(cols)

    @property
    def shape(self):
        return (self.rows, self.cols)

    @property
    def codes(self):
        """uint8 [rows, 32 b], E4M3"""
        b = -(-self.cols // 32)
        return self.data.as_strided((self.rows, 32 * b), (32 * b, 1), self.data.storage_offset())

    @property
    def scales(self):
        """uint8 [rows, b]"""
        b = -(-self.cols // 32)
        return self.data.as_strided((self.rows, b), (b, 1), self.data.storage_offset() + self.rows * 32 * b)

    def __repr__(self):
        return "Checkpoint(%d x %d)" % (self.rows, self.cols)


def _rows(x):
    n = 1
    for k in x.shape[:-1]:
        n *= k
    return n


def compress(x):
    """x [..., cols] (fp16, bf16 or fp32) -> Checkpoint of its rows, rounded to nearest, ties to even.  A block of 32 with an infinity or NaN is NaN as a whole; finite
    values stay finite in x's type.  Not differentiated: it is what a backward pass keeps."""
    data = capi.host().checkpoint_compress(x)
    return Checkpoint(data, _rows(x), x.shape[-1])


def restore(c, dtype=torch.float32):
    """the values of a Checkpoint, [rows, cols]"""
    if dtype not in _EMPTY:
        raise RuntimeError("unsupported element dtype %s" % dtype)
    return capi.host().checkpoint_restore(c.data, c.rows, c.cols, _EMPTY[dtype])


def residual_norm(y, residual=None, weight=None, bias=None, gate=None, residual_scale=1.0, block_scale=1.0, after=False, after_weight=None, after_bias=None, before=True,
                  center=False, eps=1e-6, checkpoint=False):
    """what lies between a block's last linear layer and the next block's first, in one pass over y [..., cols], the block's output:

      z = norm(y) * after_weight + after_bias     the norm after the block, with ``after``; otherwise y
      r = residual_scale * residual + block_scale * gate * z
      h = norm(r) * weight + bias                 the norm before the next block, unless ``before`` is False

    norm(x) = x / sqrt(mean(x^2) + eps), or with ``center`` (x - mean(x)) / sqrt(variance(x) + eps), in float32: a row whose squares add up to 2^128 or more
    gives NaN (10^17 in every element of the widest row, 6 10^18 in the narrowest).  Everything but y may be missing.

    residual: of y's shape; its type, y's or float32, is r's.  gate: [cols], or of y's shape with ones in place of the last dimensions that share it: [batch, 1, cols] is a gate
    for each sequence.  weights, biases, gate: of y's type or float32, and so are their gradients.  cols: 8 to 32768.

    -> (h, r), r being y itself where nothing is added to it or done with it; r alone without ``before``.
    checkpoint: (h, r, c) with c the Checkpoint of h, for the layers that take it, and the backward pass keeps r and y in 8 bits.
    What is not contiguous is copied.  The gradients cannot be differentiated again, and there is no forward mode."""
    h, r, data = capi.host().residual_norm(y, residual, weight, bias, gate, after_weight, after_bias, residual_scale, block_scale, eps, after, before, center, checkpoint)
    if not before:
        return r
    if r is None:
        r = y
    return (h, r, Checkpoint(data, _rows(h), h.shape[-1])) if checkpoint else (h, r)


_KINDS = {"silu": 0, "gelu_tanh": 1}


def gated(x, up=None, kind="silu", checkpoint=False):
    """act(gate) * up, [..., cols]: gate and up are the halves of x [..., 2 cols], side by side as a linear layer with both weights gives them, or x and up, of one shape.
    Views whose elements of a row are consecutive, and whose rows lie one distance apart, are read in place, others are copied.

    kind: "silu", g sigmoid(g), or "gelu_tanh", g sigmoid(2 sqrt(2 / pi) (g + 0.044715 g^3)) = g / 2 (1 + tanh(...)).
    checkpoint: also the Checkpoint of the result, for the layers that take it -- the answer is (out, Checkpoint) -- and the backward pass keeps gate and up in 8 bits.
    The gradients cannot be differentiated again, and there is no forward mode."""
    if kind not in _KINDS:
        raise RuntimeError("gated: unknown activation %r" % (kind,))
    out, data = capi.host().gated(x, up, _KINDS[kind], checkpoint)
    return (out, Checkpoint(data, _rows(out), out.shape[-1])) if checkpoint else out
