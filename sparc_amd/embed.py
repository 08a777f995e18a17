"""``embedding``: rows of a table for token ids, scaled, with the table's dense
gradient by sorted tokens, over sparc_embedding_forward /
sparc_embedding_backward.  The reference ships the layer, not a network; this
is how ids enter a network around it."""
from __future__ import annotations

import torch

from . import _lib


def embedding(tokens: torch.Tensor, weight: torch.Tensor, scale: float = 1.0,
              padding_idx: int | None = None) -> torch.Tensor:
    """``scale * weight[tokens]``, [*tokens.shape, D] in weight's dtype,
    differentiable in ``weight`` (a dense gradient of its shape; once, and in
    reverse mode only).

    ``tokens``: int64 or int32, any shape; ``weight``: [V, D], float32 or
    bfloat16.  ``padding_idx``: a row whose gradient is zero (its values are
    still returned; negative counts from the end).  An id outside [0, V) gives
    a row of NaN and no gradient: the ids are not read back to be checked.
    The gradient's sums are fp32 in the order of the positions, rounded once,
    so equal calls give equal bits."""
    y = _lib.native().embedding(tokens, weight, scale, padding_idx)
    return y if y is not None else _refuse(tokens, weight, padding_idx)


def _refuse(tokens, weight, padding_idx):
    """Raise what is wrong with the arguments."""
    if weight.ndim != 2 or weight.numel() == 0:
        raise ValueError(f"embedding expects a table [V, D], got {list(weight.shape)}")
    if tokens.dtype not in (torch.int64, torch.int32):
        raise TypeError(f"embedding takes int64 or int32 ids, got {tokens.dtype}")
    _lib.io_code(weight.dtype)
    if padding_idx is not None and not -weight.shape[0] <= padding_idx < weight.shape[0]:
        raise ValueError(f"padding_idx {padding_idx} is outside the table of {weight.shape[0]} rows")
    _lib.require_gpu(tokens, weight)
    raise ValueError("embedding takes dense tensors")


__all__ = ["embedding"]
