"""8-bit activation checkpoints for soft training.

A soft layer's backward pass needs the layer's input.  Inside :func:`checkpoint8` the logic
layers and conv trees keep it as one byte per value and a (lo, step) pair per row and 128
samples instead of fp32 -- 3.8 times less memory between forward and backward -- and the
backward pass evaluates the layer at the values that the codes stand for (each within half a
step, 1/510 of the block's range).  Binary inputs are kept exactly.

    with silogic_b200.checkpoint8():
        loss = criterion(model(x), y)
    loss.backward()

``train_model`` and ``GraphedTrainStep`` called inside the context train that way too.
"""
import contextlib

import torch

from . import _soft
from ._lib import require_cuda
from ._ops import CKPT_BLOCK, DTYPE_ID, op


class Checkpoint8:
    """Values kept in 8 bits: ``codes`` uint8 ``[rows, ldc]``, ``bounds`` fp32
    ``[rows, ceil(cols / 128), 2]`` = (lo, step); value = code * step + lo."""

    def __init__(self, codes, bounds, shape, dtype):
        self.codes, self.bounds, self.shape, self.dtype = codes, bounds, torch.Size(shape), dtype

    def restore(self, dtype=None):
        """The values that the codes stand for, in the stored tensor's shape (and type)."""
        dtype = dtype or self.dtype
        if dtype not in DTYPE_ID:
            raise TypeError(f"restore: dtype must be float32, bfloat16 or float16, got {dtype}")
        shape = self.shape
        if shape.numel() == 0:
            return torch.empty(shape, dtype=dtype, device=self.codes.device)
        out = op("ckpt_load")(self.codes, self.bounds, shape[-1], dtype)
        return out if len(shape) == 2 else out.view(shape)

    def nbytes(self):
        return self.codes.numel() + 4 * self.bounds.numel()


def checkpoint8_store(x):
    """Keep ``x`` (float32, bfloat16 or float16, at least one dimension) in 8 bits: each run
    of 128 values along the last dimension is cut into 255 steps between its smallest and
    its largest value.  A run that holds a NaN or an infinity reads back as NaN."""
    if x.dtype not in DTYPE_ID:
        raise TypeError(f"checkpoint8_store: x must be float32, bfloat16 or float16, got {x.dtype}")
    if x.dim() == 0:
        raise ValueError("checkpoint8_store: x must have at least one dimension")
    require_cuda(x)
    if x.requires_grad:
        x = x.detach()
    if x.numel() == 0:
        rows, cols = 0, x.shape[-1]
        return Checkpoint8(torch.empty((rows, cols), dtype=torch.uint8, device=x.device),
                           torch.empty((rows, -(-cols // CKPT_BLOCK), 2), device=x.device), x.shape, x.dtype)
    x2 = x if x.dim() == 2 else x.reshape(-1, x.shape[-1])
    return Checkpoint8(*op("ckpt_store")(x2), x.shape, x.dtype)


@contextlib.contextmanager
def checkpoint8(enabled=True):
    """Layers run inside keep their inputs for the backward pass as 8-bit codes
    (``enabled=False`` switches it off inside).  The setting is the calling thread's: other
    threads are not affected, and a thread started inside begins with it off (so does a forward
    pass that autograd repeats in its own thread: enter the context inside the repeated
    function).  The innermost context that is still open decides."""
    mine = [bool(enabled)]          # an object of its own: contexts may end in any order
    opened = _soft._switch.__dict__.setdefault("opened", [])
    opened.append(mine)
    _soft._switch.on = mine[0]
    try:
        yield
    finally:
        opened[:] = [c for c in opened if c is not mine]
        _soft._switch.on = opened[-1][0] if opened else False
