"""``layer_norm``: layer norm over the last dimension with its gradients, over
sparc_layer_norm_forward / sparc_layer_norm_backward.  The reference ships the
layer, not a network; this is what a network around it norms with (RMSNorm is
``sparc_amd.stack.rms_norm``)."""
from __future__ import annotations

import torch

from . import _lib


def _forward(x, weight, bias, eps, save):
    """(y, mean and rstd [2, rows] or None, the parameters' dtype) of contiguous
    tensors."""
    lib = _lib.load()
    D = x.shape[-1]
    rows = x.numel() // D
    y = torch.empty_like(x)
    pdtype = weight.dtype if weight is not None else bias.dtype if bias is not None else x.dtype
    stats = mean = rstd = None
    if save:
        stats = torch.empty(2, rows, dtype=torch.float32, device=x.device)
        mean = stats.data_ptr()
        rstd = mean + 4 * rows
    _lib.check(lib.sparc_layer_norm_forward(
        rows, D, _lib.io_code(x.dtype), _lib.io_code(pdtype), x.data_ptr(),
        None if weight is None else weight.data_ptr(), None if bias is None else bias.data_ptr(), eps, y.data_ptr(),
        mean, rstd, _lib.stream_of(x.device)), "sparc_layer_norm_forward")
    return y, stats, pdtype


class _LayerNorm(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, weight, bias, eps):
        x = x.contiguous()
        weight = None if weight is None else weight.contiguous()
        y, stats, ctx.pdtype = _forward(x, weight, None if bias is None else bias.contiguous(), eps, True)
        ctx.save_for_backward(x, weight, stats)
        return y

    @staticmethod
    def backward(ctx, dy):
        if torch.is_grad_enabled():
            raise RuntimeError("layer_norm is not twice differentiable")
        x, weight, stats = ctx.saved_tensors
        lib = _lib.load()
        D = x.shape[-1]
        rows = x.numel() // D
        dy = dy.contiguous()
        want = ctx.needs_input_grad
        dx = torch.empty_like(x) if want[0] else None
        dw = torch.empty(D, dtype=ctx.pdtype, device=x.device) if want[1] else None
        db = torch.empty(D, dtype=ctx.pdtype, device=x.device) if want[2] else None
        need = lib.sparc_layer_norm_workspace_bytes(rows, D) if want[1] or want[2] else 0
        ws = torch.empty(need, dtype=torch.uint8, device=x.device) if need else None
        P = _lib.ptr
        mean = stats.data_ptr()
        _lib.check(lib.sparc_layer_norm_backward(
            rows, D, _lib.io_code(x.dtype), _lib.io_code(ctx.pdtype), x.data_ptr(), P(weight), mean, mean + 4 * rows,
            dy.data_ptr(), P(dx), P(dw), P(db), P(ws), need, _lib.stream_of(x.device)), "sparc_layer_norm_backward")
        return dx, dw, db, None


def layer_norm(x: torch.Tensor, weight: torch.Tensor | None = None, bias: torch.Tensor | None = None,
               eps: float = 1e-5) -> torch.Tensor:
    """(x - mean) / sqrt(var + eps) * weight + bias over the last dimension
    (``torch.nn.functional.layer_norm``'s formula), differentiable in x, weight
    and bias.

    ``x``: float32 or bfloat16, [..., D] for any D; ``weight`` and ``bias``: [D]
    or None, in x's dtype or in float32.  The arithmetic is fp32 and every
    result is rounded once; the parameters' gradients are sums over rows in a
    fixed order, so equal calls give equal bits."""
    D = x.shape[-1] if x.ndim else 0
    if D < 1:
        raise ValueError(f"layer_norm expects [..., D] inputs with D > 0, got {list(x.shape)}")
    if not eps >= 0.0:
        raise ValueError(f"layer_norm needs eps >= 0, got {eps}")
    dtype = x.dtype
    _lib.io_code(dtype)
    grad = x.requires_grad
    if weight is not None:
        _param(weight, D, dtype, "weight")
        grad = grad or weight.requires_grad
    if bias is not None:
        _param(bias, D, dtype, "bias")
        grad = grad or bias.requires_grad
        if weight is not None and weight.dtype != bias.dtype:
            raise ValueError(f"weight and bias must be alike, got {weight.dtype} and {bias.dtype}")
    _lib.require_gpu(x, weight, bias)
    if grad and torch.is_grad_enabled():
        return _LayerNorm.apply(x, weight, bias, float(eps))
    return _forward(x.contiguous(), None if weight is None else weight.contiguous(),
                    None if bias is None else bias.contiguous(), float(eps), False)[0]


def _param(p, D, dtype, name):
    if p.ndim != 1 or p.numel() != D or p.dtype != dtype and p.dtype != torch.float32:
        raise ValueError(f"{name} must be [{D}] in the input's dtype or float32, got {list(p.shape)} {p.dtype}")


__all__ = ["layer_norm"]
