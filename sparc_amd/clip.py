"""``grad_norm`` and ``clip_grad_norm_``: the L2 norm over all gradients of a
model, and the gradients scaled in place to a largest norm, over
sparc_grad_norm / sparc_clip_grad_norm: the norm stays on the device, and one
call takes every tensor."""
from __future__ import annotations

import math
from array import array

import torch

from . import _lib

_Tensor = torch.Tensor
_CODES = {torch.float32: _lib.SPARC_F32, torch.bfloat16: _lib.SPARC_BF16}


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


def _call(fn_name, tensors, *args):
    """One library call over the tensors' values (a tensor given twice counts
    once); the norm, [] float32."""
    lib = _lib.load()
    dev = tensors[0].device
    if not tensors[0].is_cuda or len(set(map(_Tensor.get_device, tensors))) > 1:
        _lib.require_gpu(*tensors)
    data = list(map(_Tensor.data_ptr, tensors))
    if len(set(data)) != len(data):
        tensors = list({(p, t.numel(), t.dtype): t for p, t in zip(data, tensors)}.values())
        data = list(map(_Tensor.data_ptr, tensors))
    n = len(data)
    sizes, codes = array("q", map(_Tensor.numel, tensors)), array("i", [_CODES[t.dtype] for t in tensors])
    data = array("Q", data)
    norm = torch.empty((), dtype=torch.float32, device=dev)
    need = lib.sparc_grad_norm_workspace_bytes(n)
    ws = torch.empty(need, dtype=torch.uint8, device=dev)
    _lib.check(getattr(lib, fn_name)(n, data.buffer_info()[0], sizes.buffer_info()[0], codes.buffer_info()[0], *args,
                                     norm.data_ptr(), ws.data_ptr(), need, _lib.stream_of(dev)), fn_name)
    return norm


def _checked(tensors):
    for t in tensors:
        if t.layout is not torch.strided:
            raise ValueError(f"gradients must be dense tensors, got layout {t.layout}")
        if t.dtype not in _CODES:
            raise TypeError(f"SPARC HIP kernels take float32 or bfloat16 tensors, got {t.dtype}")
    return tensors


def grad_norm(tensors) -> torch.Tensor:
    """The L2 norm over all values of ``tensors`` (one or several, float32 and
    bfloat16 mixed, any shapes), a float32 scalar on their device.  Squares are
    summed in fp64 in a fixed order: no overflow, equal calls give equal bits."""
    tensors = [tensors] if torch.is_tensor(tensors) else list(tensors)
    tensors = [t if _dense(t) else t.contiguous() for t in _checked(tensors)]
    return _call("sparc_grad_norm", tensors) if tensors else torch.zeros(())


@torch.no_grad()
def clip_grad_norm_(parameters, max_norm: float) -> torch.Tensor:
    """Scale the gradients of ``parameters`` in place by
    ``min(1, max_norm / (norm + 1e-6))``, ``norm`` their common L2 norm before;
    returns ``norm`` (``torch.nn.utils.clip_grad_norm_`` for the L2 norm).

    Nothing waits for the device and nothing is read back; where the norm is
    small enough no gradient is written.  Gradients that overlap without being
    the same are refused.  A norm that is not finite goes into
    the gradients as it does in torch: NaN for NaN, 0 (NaN for the infinite
    values) for infinity.  Parameters without a gradient are skipped."""
    max_norm = float(max_norm)
    if math.isnan(max_norm) or max_norm < 0.0:
        raise ValueError(f"clip_grad_norm_ needs max_norm >= 0, got {max_norm}")
    parameters = [parameters] if torch.is_tensor(parameters) else parameters
    grads = _checked([g for g in [p.grad for p in parameters] if g is not None])
    if not grads:
        return torch.zeros(())
    copies = []
    for i, g in enumerate(grads if not all(map(_Tensor.is_contiguous, grads)) else ()):
        if not _dense(g):
            if _repeats(g):
                raise ValueError("a gradient names one value more than once (an expanded view): it cannot be scaled "
                                 "in place")
            grads[i] = g.contiguous()
            copies.append((g, grads[i]))
    norm = _call("sparc_clip_grad_norm", grads, max_norm)
    for g, c in copies:
        g.copy_(c)
    return norm


__all__ = ["grad_norm", "clip_grad_norm_"]
