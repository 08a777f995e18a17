"""``linear_attention`` and ``linear_attention_step``: linear attention with a decay
for each head, over sequences (sparc_linear_attention_forward / _backward) and for
one step (sparc_linear_attention_step); ``qk_norm_rotary``: what its queries and
keys go through before, norms for each head and the rotation by their positions
(sparc_qk_norm_rotary_forward / _backward).  The reference's layer keeps a vector
as its state, one value per mode; here a head's state is a matrix."""
from __future__ import annotations

import torch

from . import _lib

MAX_HEAD_DIM = 256     # of linear attention's keys and values
MAX_ROTARY_HEAD_DIM = 512


def rotary_table(length: int, dim: int, base: float = 10000.0, device=None) -> torch.Tensor:
    """Cosines and sines [length, dim] fp32 of the positions 0 .. length - 1: the
    angles position * base^(-2 i / dim) for i < dim / 2, computed in 64 bits; the
    cosines come first.  ``dim`` is even."""
    if length < 0 or dim < 0 or dim % 2:
        raise ValueError(f"rotary_table needs a length >= 0 and an even dim >= 0, got {length} and {dim}")
    i = torch.arange(0, dim, 2, device=device, dtype=torch.float64)
    angle = torch.arange(length, device=device, dtype=torch.float64)[:, None] * base ** (-i / max(dim, 1))
    return torch.cat((angle.cos(), angle.sin()), dim=-1).float()


def keep_reach(positions: torch.Tensor, reach: int | None) -> torch.Tensor:
    """``positions``, with how far they reach at most (the steps behind them) kept on
    the host beside them, so that a limit is checked without waiting for the device.
    It holds until the tensor is written; an inference tensor, which does not count
    its writes, keeps none."""
    if reach is not None and not positions.is_inference():
        positions.reach = (reach, positions._version)
    return positions


def reach_of(positions: torch.Tensor) -> int | None:
    """What ``keep_reach`` has kept beside the tensor, or None."""
    reach, version = getattr(positions, "reach", (None, None))
    return reach if version is not None and positions._version == version else None


def qk_norm_rotary(q: torch.Tensor, k: torch.Tensor, q_weight: torch.Tensor | None, k_weight: torch.Tensor | None,
                   table: torch.Tensor, positions: torch.Tensor | None = None, interleaved: bool = False,
                   eps: float = 1e-6) -> tuple[torch.Tensor, torch.Tensor]:
    """RMS norms of queries and keys for each head and the rotation by their
    positions, in one pass: ``x / sqrt(mean(x^2) + eps) * weight`` over the last
    dimension, whose first R values are then turned in pairs, (i, i + R / 2) or with
    ``interleaved`` (2 i, 2 i + 1), by the angles of the token's position.

    ``q``: [B, T, H, D], ``k``: [B, T, G, D], float32 or bfloat16, D up to 512, at
    any strides whose last one is 1 (parts of one projection's output are read where
    they are); ``q_weight``, ``k_weight``: [D] or None, in their dtype or in
    float32; ``table``: [P, R] float32 with R even and at most D, as
    ``rotary_table`` makes it (no gradient); ``positions``: int64 or int32,
    [B, T], [T] or broadcast to it, by default 0 .. T - 1.  A position outside the
    table gives NaN.  Returns contiguous tensors, differentiable in q, k and the
    weights (once, and in reverse mode only).  The arithmetic is fp32 and every
    result is rounded once; equal calls give equal bits."""
    y = _lib.native().qk_norm_rotary(q, k, q_weight, k_weight, table, positions, interleaved, eps)
    return y if y is not None else _refuse_rotary(q, k, q_weight, k_weight, table, positions, eps)


def _refuse_rotary(q, k, q_weight, k_weight, table, positions, eps):
    """Raise what is wrong with the arguments."""
    if q.ndim != 4 or k.ndim != 4 or q.shape[:2] != k.shape[:2] or q.shape[3] != k.shape[3] or 0 in q.shape[2:] or \
            0 in k.shape[2:]:
        raise ValueError(f"q and k must be [B, T, H, D] and [B, T, G, D], got {list(q.shape)} and {list(k.shape)}")
    D = q.shape[3]
    if D > MAX_ROTARY_HEAD_DIM:
        raise ValueError(f"heads of up to {MAX_ROTARY_HEAD_DIM} values are supported, got {D}")
    if not eps >= 0.0:
        raise ValueError(f"qk_norm_rotary needs eps >= 0, got {eps}")
    _lib.io_code(q.dtype)
    if k.dtype != q.dtype:
        raise ValueError(f"q and k must be alike, got {q.dtype} and {k.dtype}")
    for p, name in ((q_weight, "q_weight"), (k_weight, "k_weight")):
        if p is not None and (p.ndim != 1 or p.numel() != D or p.dtype not in (q.dtype, torch.float32)):
            raise ValueError(f"{name} must be [{D}] in the input's dtype or float32, got {list(p.shape)} {p.dtype}")
    if q_weight is not None and k_weight is not None and q_weight.dtype != k_weight.dtype:
        raise ValueError(f"q_weight and k_weight must be alike, got {q_weight.dtype} and {k_weight.dtype}")
    if table.ndim != 2 or table.dtype != torch.float32 or table.shape[1] > D or table.shape[1] % 2:
        raise ValueError(f"table must be [P, R] float32 with an even R of at most {D}, got {list(table.shape)} "
                         f"{table.dtype}")
    if positions is not None:
        if positions.dtype not in (torch.int64, torch.int32):
            raise ValueError(f"positions must be int64 or int32, got {positions.dtype}")
        want = list(q.shape[:2])
        if positions.ndim not in (1, 2) or any(
                n not in (1, m) for n, m in zip(reversed(positions.shape), reversed(want))):
            raise ValueError(f"positions must be {want}, [{want[1]}] or broadcast to it, got {list(positions.shape)}")
    _lib.require_gpu(q, k, q_weight, k_weight, table, positions)
    raise ValueError("qk_norm_rotary takes dense tensors")


def linear_attention(q: torch.Tensor, k: torch.Tensor, v: torch.Tensor, log_decay: torch.Tensor,
                     state: torch.Tensor | None = None, scale: float | None = None,
                     lengths: torch.Tensor | None = None) -> tuple[torch.Tensor, torch.Tensor]:
    """Linear attention with a decay a = exp(log_decay) for each head:

        S_t = a S_(t-1) + k_t v_t^T,    o_t = scale * q_t S_t

    and (o, the state after the last step).  ``q``: [B, T, H, K], ``k``: [B, T, G,
    K], ``v``: [B, T, G, V], float32 or bfloat16, K and V up to 256, at any strides
    whose last one is 1; H is a multiple of G, and query head h reads key head
    h // (H // G).  ``log_decay``: [H] float32, at most 0 (-inf: no memory; no
    gradient); ``state``: [B, H, K, V] float32, by default zero; ``scale``: by
    default 1 / sqrt(K); ``lengths``: [B] int64 or int32, the steps that each row
    has (cut to 0 .. T): what lies behind them is not read, their outputs are zero,
    and the state is that after the last step there is.

    Differentiable in q, k, v and state (once, and in reverse mode only); nothing
    but the inputs is kept for it.  Sums and states are fp32, and results are rounded
    once.  bfloat16 inputs are multiplied as they are; what is computed on the way
    enters a product with them as a sum of bfloat16 values: what is added to a state
    that is returned as three, which hold all of it, the rest (scores, the state where
    it is read, decayed values) as two, which hold all but 2^-17 (an infinite one of
    these becomes NaN).  Equal calls give equal bits."""
    y = _lib.native().linear_attention(q, k, v, log_decay, state, scale, lengths)
    return y if y is not None else _refuse_linear(q, k, v, log_decay, state, lengths, 4)


def linear_attention_step(q: torch.Tensor, k: torch.Tensor, v: torch.Tensor, log_decay: torch.Tensor,
                          state: torch.Tensor, scale: float | None = None,
                          out_state: torch.Tensor | None = None) -> tuple[torch.Tensor, torch.Tensor]:
    """One step of ``linear_attention`` without the time dimension: q [B, H, K], k
    [B, G, K], v [B, G, V] and the state [B, H, K, V] give (o [B, H, V], the new
    state).  ``out_state``: where the new state goes, contiguous; it may be ``state``
    itself (in place).  The arithmetic is fp32.

    There is no backward: outside ``torch.no_grad()`` tensors that require grad
    are refused."""
    y = _lib.native().linear_attention_step(q, k, v, log_decay, state, scale, out_state)
    return y if y is not None else _refuse_linear(q, k, v, log_decay, state, None, 3, out_state)


def _refuse_linear(q, k, v, log_decay, state, lengths, dim, out_state=None):
    """Raise what is wrong with the arguments."""
    lead = "B, T" if dim == 4 else "B"
    if any(x.ndim != dim for x in (q, k, v)) or q.shape[:-2] != k.shape[:-2] or q.shape[:-2] != v.shape[:-2] or \
            k.shape[-2] != v.shape[-2] or q.shape[-1] != k.shape[-1]:
        raise ValueError(f"q, k and v must be [{lead}, H, K], [{lead}, G, K] and [{lead}, G, V], got {list(q.shape)}, "
                         f"{list(k.shape)} and {list(v.shape)}")
    H, G, K, V = q.shape[-2], k.shape[-2], q.shape[-1], v.shape[-1]
    if H < 1 or G < 1 or H % G:
        raise ValueError(f"the {H} query heads must be a multiple of the {G} key heads")
    if not (1 <= K <= MAX_HEAD_DIM and 1 <= V <= MAX_HEAD_DIM):
        raise ValueError(f"keys and values of 1 to {MAX_HEAD_DIM} per head are supported, got {K} and {V}")
    _lib.io_code(q.dtype)
    if k.dtype != q.dtype or v.dtype != q.dtype:
        raise ValueError(f"q, k and v must be alike, got {q.dtype}, {k.dtype} and {v.dtype}")
    _lib.expect(log_decay, (H,), torch.float32, "log_decay")
    if state is not None or dim == 3:
        _lib.expect(state, (q.shape[0], H, K, V), torch.float32, "state")
    if lengths is not None and (tuple(lengths.shape) != (q.shape[0],) or
                                lengths.dtype not in (torch.int64, torch.int32)):
        raise ValueError(f"lengths must be [{q.shape[0]}] int64 or int32, got {list(lengths.shape)} {lengths.dtype}")
    if out_state is not None:
        _lib.expect(out_state, (q.shape[0], H, K, V), torch.float32, "out_state")
        if not out_state.is_contiguous() or out_state.is_conj() or out_state.is_neg():
            raise ValueError("out_state must be a contiguous tensor, no view that conjugates or negates")
    _lib.require_gpu(q, k, v, log_decay, state, lengths, out_state)
    raise ValueError("linear attention takes dense tensors")


__all__ = ["rotary_table", "qk_norm_rotary", "linear_attention", "linear_attention_step"]
