"""``layer_norm``: layer norm over the last dimension with its gradients, over
sparc_layer_norm_forward / sparc_layer_norm_backward.  The reference ships the
layer, not a network; this is what a network around it norms with (RMSNorm is
``sparc_amd.stack.rms_norm``)."""
from __future__ import annotations

import torch

from . import _lib


def _forward(x, weight, bias, eps, save):
    lib = _lib.load()
    D = x.shape[-1]
    rows = x.numel() // D
    y = torch.empty_like(x)
    stats = torch.empty(2, rows, dtype=torch.float32, device=x.device) if save else None
    P = _lib.ptr
    pdtype = x.dtype if weight is None and bias is None else (weight if weight is not None else bias).dtype
    _lib.check(lib.sparc_layer_norm_forward(
        rows, D, _lib.io_code(x.dtype), _lib.io_code(pdtype), P(x), P(weight), P(bias), eps, P(y),
        stats.data_ptr() if save else None, stats.data_ptr() + 4 * rows if save else None,
        _lib.stream_of(x.device)), "sparc_layer_norm_forward")
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
        _lib.check(lib.sparc_layer_norm_backward(
            rows, D, _lib.io_code(x.dtype), _lib.io_code(ctx.pdtype), P(x), P(weight), stats.data_ptr(),
            stats.data_ptr() + 4 * rows, P(dy), P(dx), P(dw), P(db), P(ws), need, _lib.stream_of(x.device)),
            "sparc_layer_norm_backward")
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
    if x.ndim < 1 or x.shape[-1] < 1:
        raise ValueError(f"layer_norm expects [..., D] inputs with D > 0, got {list(x.shape)}")
    if not eps >= 0.0:
        raise ValueError(f"layer_norm needs eps >= 0, got {eps}")
    _lib.io_code(x.dtype)
    params = [(n, p) for n, p in (("weight", weight), ("bias", bias)) if p is not None]
    for name, p in params:
        if p.dtype not in (x.dtype, torch.float32) or p.dtype != params[0][1].dtype:
            raise ValueError(f"{name} must be in the input's dtype or float32 (weight and bias alike), got {p.dtype}")
        _lib.expect(p, (x.shape[-1],), p.dtype, name)
    _lib.require_gpu(x, weight, bias)
    if torch.is_grad_enabled() and (x.requires_grad or any(p.requires_grad for _, p in params)):
        return _LayerNorm.apply(x, weight, bias, float(eps))
    return _forward(x.contiguous(), *[None if p is None else p.contiguous() for p in (weight, bias)], float(eps),
                    False)[0]


__all__ = ["layer_norm"]
