"""``gated_linear_unit``: the gated half of a feed-forward block, both projections,
the activation and the product in one kernel, with its gradients, over
sparc_gated_forward / sparc_gated_backward."""
from __future__ import annotations

import torch

from . import _lib

ACTIVATIONS = {"silu": 0, "gelu": 1, "relu": 2, "sigmoid": 3}


def gated_linear_unit(x: torch.Tensor, gate_weight: torch.Tensor, up_weight: torch.Tensor,
                      activation: str = "silu") -> torch.Tensor:
    """act(x gate_weight^T) * (x up_weight^T), differentiable in all three (once,
    and in reverse mode only).

    ``x``: [..., D]; the weights: [F, D] as in ``torch.nn.Linear``, all float32 or
    all bfloat16, of any sizes; ``activation``: "silu" (x sigmoid(x)), "gelu" (x
    Phi(x), exact), "relu" or "sigmoid".  Sums are fp32, and the activation and the
    product are computed from unrounded projections and rounded once (an infinite
    float32 input gives NaN: it is multiplied in parts).  Nothing but
    the inputs is kept for the backward, which computes the projections again;
    their gradients are rounded to the inputs' dtype once before they are
    multiplied with x and the weights (in bfloat16 up to 2^28 = rows D F to a sum of
    two values, whose error does not show)."""
    if activation not in ACTIVATIONS:
        raise ValueError(f"unknown activation {activation!r} ({', '.join(ACTIVATIONS)})")
    y = _lib.native().gated_linear_unit(x, gate_weight, up_weight, ACTIVATIONS[activation])
    return y if y is not None else _refuse(x, gate_weight, up_weight)


def _refuse(x, gate_weight, up_weight):
    """Raise what is wrong with the arguments."""
    D = x.shape[-1] if x.ndim else 0
    if D < 1:
        raise ValueError(f"gated_linear_unit expects [..., D] inputs with D > 0, got {list(x.shape)}")
    if gate_weight.ndim != 2 or gate_weight.shape[0] < 1 or gate_weight.shape[1] != D or \
            up_weight.shape != gate_weight.shape:
        raise ValueError(f"the weights must both be [F, {D}], got {list(gate_weight.shape)} and "
                         f"{list(up_weight.shape)}")
    _lib.io_code(x.dtype)
    if gate_weight.dtype != x.dtype or up_weight.dtype != x.dtype:
        raise ValueError(f"x and the weights must be alike, got {x.dtype}, {gate_weight.dtype} and {up_weight.dtype}")
    _lib.require_gpu(x, gate_weight, up_weight)
    raise ValueError("gated_linear_unit takes dense tensors")


__all__ = ["gated_linear_unit"]
