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
        return self.data[:self.data.numel() // 33 * 32].view(self.rows, -(-self.cols // 32) * 32)

    @property
    def scales(self):
        """uint8 [rows, b]"""
        return self.data[self.data.numel() // 33 * 32:].view(self.rows, -(-self.cols // 32))

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
