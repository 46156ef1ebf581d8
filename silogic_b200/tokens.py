"""Token input: scaled embedding lookup with a gradient summed over sorted tokens."""
import torch
import torch.nn as nn

from . import _hard
from ._lib import nodes, require_cuda
from ._ops import DTYPE_ID, op


class _TokenEmbedding(torch.autograd.Function):
    """The node that torch.compile traces (eager calls use the native one, ``csrc/autograd.cpp``)."""

    @staticmethod
    def forward(ctx, ids, weight, scale, padding_idx):
        ctx.save_for_backward(ids)
        ctx.args = (weight.shape[0], scale, padding_idx)
        return op("embed_fwd")(ids, weight.contiguous(), scale)

    @staticmethod
    def backward(ctx, g):
        (ids,) = ctx.saved_tensors
        return None, op("embed_bwd")(ids, g, *ctx.args), None, None


def token_embedding(ids, weight, scale=1.0, padding_idx=None, check=False):
    """``scale * weight[ids]``: ``ids`` int32 / int64 of any shape, ``weight`` ``[V, D]``
    float32, bfloat16 or float16 -> ``ids.shape + (D,)`` of weight's type.

    The gradient of ``weight`` is summed in 32 bits in the order of the sorted tokens, so it is
    the same from run to run; tokens equal to ``padding_idx`` add nothing to it.  An id
    outside ``[0, V)`` gives a row of NaN and no gradient; ``check=True`` raises
    ``IndexError`` for it instead (and waits for the GPU)."""
    if weight.dim() != 2 or weight.dtype not in DTYPE_ID:
        raise TypeError("token_embedding: weight must be [V, D] float32, bfloat16 or float16, got "
                        f"{tuple(weight.shape)} {weight.dtype}")
    if ids.dtype is not torch.int64 and ids.dtype is not torch.int32:
        raise TypeError(f"token_embedding: ids must be int32 or int64, got {ids.dtype}")
    if not (ids.is_cuda and weight.is_cuda):
        require_cuda(ids, weight)
    if ids.device != weight.device:
        raise ValueError(f"token_embedding: ids on {ids.device}, weight on {weight.device}")
    V, D = weight.shape
    if V == 0 or D == 0:
        raise ValueError(f"token_embedding: empty weight {tuple(weight.shape)}")
    pad = -1
    if padding_idx is not None:
        if not -V <= padding_idx < V:
            raise ValueError(f"token_embedding: padding_idx {padding_idx} not in [-{V}, {V})")
        pad = int(padding_idx) % V
    if check:
        _hard.check_index_range(ids, V, "token ids")
    ids = ids.contiguous()
    if not torch.compiler.is_compiling():
        return nodes().token_embedding(ids, weight, float(scale), pad)
    if weight.requires_grad and torch.is_grad_enabled():
        return _TokenEmbedding.apply(ids, weight, float(scale), pad)
    return op("embed_fwd")(ids, weight.contiguous(), float(scale))


class TokenEmbedding(nn.Module):
    """Learned table of ``num_tokens`` rows of ``dim`` values, read by token id and scaled
    (``scale=None``: ``sqrt(dim)``, with rows drawn as N(0, 1/dim))."""

    def __init__(self, num_tokens, dim, scale=None, padding_idx=None, dtype=torch.float32):
        super().__init__()
        self.num_tokens, self.dim, self.padding_idx = num_tokens, dim, padding_idx
        self.scale = dim ** 0.5 if scale is None else float(scale)
        w = torch.randn(num_tokens, dim) * dim ** -0.5
        if padding_idx is not None:
            w[padding_idx] = 0.0
        self.weight = nn.Parameter(w.to(dtype))

    def forward(self, ids):
        return token_embedding(ids, self.weight, self.scale, self.padding_idx)
