"""``layer_norm``: layer norm over the last dimension with its gradients, over
sparc_layer_norm_forward / sparc_layer_norm_backward.  The reference ships the
layer, not a network; this is what a network around it norms with (RMSNorm is
``sparc_amd.stack.rms_norm``)."""
from __future__ import annotations

import torch

from . import _lib


def layer_norm(x: torch.Tensor, weight: torch.Tensor | None = None, bias: torch.Tensor | None = None,
               eps: float = 1e-5) -> torch.Tensor:
    """(x - mean) / sqrt(var + eps) * weight + bias over the last dimension
    (``torch.nn.functional.layer_norm``'s formula), differentiable in x, weight
    and bias (once, and in reverse mode only).

    ``x``: float32 or bfloat16, [..., D] for any D; ``weight`` and ``bias``: [D]
    or None, in x's dtype or in float32.  The arithmetic is fp32 and every
    result is rounded once; the parameters' gradients are sums over rows in a
    fixed order, so equal calls give equal bits."""
    y = _lib.native().layer_norm(x, weight, bias, eps)
    return y if y is not None else _refuse(x, weight, bias, eps)


def _refuse(x, weight, bias, eps):
    """Raise what is wrong with the arguments."""
    D = x.shape[-1] if x.ndim else 0
    if D < 1:
        raise ValueError(f"layer_norm expects [..., D] inputs with D > 0, got {list(x.shape)}")
    if not eps >= 0.0:
        raise ValueError(f"layer_norm needs eps >= 0, got {eps}")
    _lib.io_code(x.dtype)
    for p, name in ((weight, "weight"), (bias, "bias")):
        if p is not None and (p.ndim != 1 or p.numel() != D or p.dtype not in (x.dtype, torch.float32)):
            raise ValueError(f"{name} must be [{D}] in the input's dtype or float32, got {list(p.shape)} {p.dtype}")
    if weight is not None and bias is not None and weight.dtype != bias.dtype:
        raise ValueError(f"weight and bias must be alike, got {weight.dtype} and {bias.dtype}")
    _lib.require_gpu(x, weight, bias)
    raise ValueError("layer_norm takes dense tensors")


__all__ = ["layer_norm"]
