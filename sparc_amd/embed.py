"""``embedding``: rows of a table for token ids, scaled, with the table's dense
gradient by sorted tokens, over sparc_embedding_forward /
sparc_embedding_backward.  The reference ships the layer, not a network; this
is how ids enter a network around it."""
from __future__ import annotations

import torch

from . import _lib


def _forward(tokens, weight, scale):
    """The rows, of contiguous tensors."""
    lib = _lib.load()
    vocab, dim = weight.shape
    dev = weight.device
    y = torch.empty(*tokens.shape, dim, dtype=weight.dtype, device=dev)
    _lib.check(lib.sparc_embedding_forward(
        tokens.numel(), vocab, dim, _lib.io_code(weight.dtype), tokens.element_size(), tokens.data_ptr(),
        weight.data_ptr(), scale, y.data_ptr(), _lib.stream_of(dev)), "sparc_embedding_forward")
    return y


class _Embedding(torch.autograd.Function):
    @staticmethod
    def forward(ctx, weight, tokens, scale, padding_id):
        ctx.save_for_backward(tokens)
        ctx.args = (weight.shape, weight.dtype, scale, padding_id)
        return _forward(tokens, weight.contiguous(), scale)

    @staticmethod
    def backward(ctx, dy):
        if torch.is_grad_enabled():
            raise RuntimeError("embedding is not twice differentiable")
        tokens, = ctx.saved_tensors
        (vocab, dim), dtype, scale, padding_id = ctx.args
        lib = _lib.load()
        n = tokens.numel()
        dy = dy.contiguous()
        dw = torch.empty(vocab, dim, dtype=dtype, device=dy.device)
        need = lib.sparc_embedding_workspace_bytes(n, vocab, dim)
        ws = torch.empty(need, dtype=torch.uint8, device=dy.device)
        _lib.check(lib.sparc_embedding_backward(
            n, vocab, dim, _lib.io_code(dtype), tokens.element_size(), tokens.data_ptr(), padding_id, dy.data_ptr(),
            scale, dw.data_ptr(), ws.data_ptr(), need, _lib.stream_of(dy.device)), "sparc_embedding_backward")
        return dw, None, None, None


def embedding(tokens: torch.Tensor, weight: torch.Tensor, scale: float = 1.0,
              padding_idx: int | None = None) -> torch.Tensor:
    """``scale * weight[tokens]``, [*tokens.shape, D] in weight's dtype,
    differentiable in ``weight`` (a dense gradient of its shape).

    ``tokens``: int64 or int32, any shape; ``weight``: [V, D], float32 or
    bfloat16.  ``padding_idx``: a row whose gradient is zero (its values are
    still returned; negative counts from the end).  An id outside [0, V) gives
    a row of NaN and no gradient: the ids are not read back to be checked.
    The gradient's sums are fp32 in the order of the positions, rounded once,
    so equal calls give equal bits."""
    if weight.ndim != 2 or weight.numel() == 0:
        raise ValueError(f"embedding expects a table [V, D], got {list(weight.shape)}")
    if tokens.dtype not in (torch.int64, torch.int32):
        raise TypeError(f"embedding takes int64 or int32 ids, got {tokens.dtype}")
    _lib.io_code(weight.dtype)
    padding_id = -1
    if padding_idx is not None:
        if not -weight.shape[0] <= padding_idx < weight.shape[0]:
            raise ValueError(f"padding_idx {padding_idx} is outside the table of {weight.shape[0]} rows")
        padding_id = padding_idx % weight.shape[0]
    _lib.require_gpu(tokens, weight)
    tokens = tokens.contiguous()
    if weight.requires_grad and torch.is_grad_enabled():
        return _Embedding.apply(weight, tokens, float(scale), padding_id)
    return _forward(tokens, weight.contiguous(), float(scale))


__all__ = ["embedding"]
