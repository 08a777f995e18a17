"""``grad_norm`` and ``clip_grad_norm_``: the L2 norm over all gradients of a
model, and the gradients scaled in place to a largest norm, over
sparc_grad_norm / sparc_clip_grad_norm: the norm stays on the device, and one
call takes every tensor."""
from __future__ import annotations

import math

import torch

from . import _lib

_DTYPES = (torch.float32, torch.bfloat16)


def _dense(t: torch.Tensor) -> bool:
    """Whether the tensor's values are one block of memory without gaps or
    repeats, in whatever order."""
    if t.is_contiguous():
        return True
    expect = 1
    for stride, size in sorted((st, sz) for st, sz in zip(t.stride(), t.shape) if sz != 1):
        if stride != expect:
            return False
        expect *= size
    return True


def _repeats(t: torch.Tensor) -> bool:
    """Whether the tensor may name one value more than once (an expanded view)."""
    reach = 0
    for stride, size in sorted((st, sz) for st, sz in zip(t.stride(), t.shape) if sz > 1):
        if stride <= reach:
            return True
        reach += stride * (size - 1)
    return False


def _checked(tensors):
    for t in tensors:
        if t.layout is not torch.strided:
            raise ValueError(f"gradients must be dense tensors, got layout {t.layout}")
        if t.dtype not in _DTYPES:
            raise TypeError(f"SPARC HIP kernels take float32 or bfloat16 tensors, got {t.dtype}")
    return tensors


def grad_norm(tensors) -> torch.Tensor:
    """The L2 norm over all values of ``tensors`` (one or several, float32 and
    bfloat16 mixed, any shapes), a float32 scalar on their device.  Squares are
    summed in fp64 in a fixed order: no overflow, equal calls give equal bits.
    There is no backward: outside ``torch.no_grad()`` tensors that require grad
    are refused."""
    tensors = [tensors] if torch.is_tensor(tensors) else list(tensors)
    if not tensors:
        return torch.zeros(())
    norm = _lib.native().grad_norm(tensors, None, False)
    return _copied_norm(_checked(tensors), None) if norm is None else norm


def clip_grad_norm_(parameters, max_norm: float) -> torch.Tensor:
    """Scale the gradients of ``parameters`` in place by
    ``min(1, max_norm / (norm + 1e-6))``, ``norm`` their common L2 norm before;
    returns ``norm`` (``torch.nn.utils.clip_grad_norm_`` for the L2 norm).

    Nothing waits for the device and nothing is read back; where the norm is
    small enough no gradient is scaled.  Gradients with gaps between their
    values are scaled in copies, which are written back always.  Gradients that
    overlap without being the same are refused.  A norm that is not finite goes
    into the gradients as it does in torch: NaN for NaN, 0 (NaN for the infinite
    values) for infinity.  As in torch, the call is outside any graph, whatever
    the grad mode.  Parameters without a gradient are skipped."""
    max_norm = float(max_norm)
    if math.isnan(max_norm) or max_norm < 0.0:
        raise ValueError(f"clip_grad_norm_ needs max_norm >= 0, got {max_norm}")
    parameters = [parameters] if torch.is_tensor(parameters) else parameters
    grads = [g for g in [p.grad for p in parameters] if g is not None]
    if not grads:
        return torch.zeros(())
    norm = _lib.native().grad_norm(grads, max_norm, False)
    if norm is not None:
        return norm
    for g in _checked(grads):
        if not _dense(g) and _repeats(g):
            raise ValueError("a gradient names one value more than once (an expanded view): it cannot be scaled in "
                             "place")
    return _copied_norm(grads, max_norm)


def _copied_norm(tensors, max_norm):
    """By way of copies where the values are not in a row in memory."""
    _lib.require_gpu(*tensors)
    return _lib.native().grad_norm(tensors, max_norm, True)


__all__ = ["grad_norm", "clip_grad_norm_"]
