"""``beam_search_step`` and ``reorder_states``: one step of beam search over
beams and vocabulary, and recurrent states in the new beams' order, over
sparc_beam_step / sparc_reorder_states.  The states are those of
``SPARCMixer.step`` with one row per hypothesis."""
from __future__ import annotations

from array import array
from typing import NamedTuple, Sequence

import torch

from . import _lib

MAX_BEAMS = 32


class BeamStep(NamedTuple):
    """The hypotheses after a step, best first."""
    tokens: torch.Tensor      # [B, K] int64: the token appended
    parents: torch.Tensor     # [B, K] int64: the beam it was appended to
    scores: torch.Tensor      # [B, K] float32
    finished: torch.Tensor | None  # [B, K] bool
    states: list              # as given, in the new order


def _planes(states):
    return [p for s in states for p in (s if isinstance(s, (tuple, list)) else (s,))]


def _like(states, planes):
    """``planes`` in the structure of ``states``."""
    at = iter(planes)
    return [tuple([next(at) for _ in s]) if isinstance(s, (tuple, list)) else next(at) for s in states]


def _fresh(planes, alike):
    """Contiguous tensors of the planes' shapes and dtypes; those of one shape
    and dtype (``alike``: all of them) share an allocation."""
    if alike:
        p = planes[0]
        return torch.empty(len(planes), *p.shape, dtype=p.dtype, device=p.device).unbind(0)
    return [torch.empty_like(p, memory_format=torch.contiguous_format) for p in planes]


def _check_out(planes, out):
    if len(out) != len(planes):
        raise ValueError(f"out_states has {len(out)} tensors for {len(planes)} states")
    spans = []  # (first byte, end, whether it is written)
    for o, p in zip(out, planes):
        if o is not p:
            _lib.expect(o, p.shape, p.dtype, "out_states")
        if not o.is_contiguous():
            raise ValueError("out_states must be contiguous tensors")
        at, src, size = o.data_ptr(), p.data_ptr(), o.numel() * o.element_size()
        if size:
            spans.append((at, at + size, True))
            if src != at:
                spans.append((src, src + _reach(p), False))
    spans.sort()
    end, written_end = 0, 0
    for first, last, written in spans:
        if first < (end if written else written_end):
            raise ValueError("a tensor of out_states overlaps another one, or another one of the states")
        end = max(end, last)
        if written:
            written_end = max(written_end, last)


def _reach(t):
    """Bytes from a tensor's first value to behind its last."""
    return (sum((n - 1) * st for n, st in zip(t.shape, t.stride())) + 1) * t.element_size()


@torch.no_grad()
def reorder_states(states: Sequence, parents: torch.Tensor, out_states: Sequence | None = None) -> list:
    """Every tensor's row b * K + k replaced by its row b * K + parents[b, k].

    ``states``: tensors [B * K, ...], or tuples of them such as the (re, im) of
    ``SPARCMixer.step``, in a list; ``parents``: [B, K] int64, K up to 32.
    ``out_states``: the same structure to write to; it may be ``states`` itself
    (in place: rows that stay are neither read nor written), but no tensor of it
    may overlap another of the states.  By default fresh tensors are returned,
    which share one allocation where all states are of one shape and dtype.  A
    parent outside [0, K) gives a row of NaN."""
    if parents.ndim != 2 or parents.dtype != torch.int64 or not 1 <= parents.shape[1] <= MAX_BEAMS:
        raise ValueError(f"parents must be [B, K] int64 with K from 1 to {MAX_BEAMS}, got {list(parents.shape)} "
                         f"{parents.dtype}")
    return _reorder(states, parents.contiguous(), out_states)


def _reorder(states, parents, out_states):
    B, K = parents.shape
    planes, rows, dev = _planes(states), B * K, parents.device
    shapes = [p.shape for p in planes]
    alike = shapes.count(shapes[0]) == len(shapes) if shapes else False
    for shape in shapes[:1] if alike else shapes:
        if not len(shape) or shape[0] != rows:
            raise ValueError(f"states must have {rows} rows (one per beam), got {list(shape)}")
    _lib.require_gpu(parents)
    index = dev.index
    if any([p.get_device() != index for p in planes]):
        _lib.require_gpu(parents, *planes)
    sizes = [p.element_size() for p in planes]
    if alike:
        dtype = planes[0].dtype
        alike = all([p.dtype is dtype for p in planes])
    if out_states is None:
        out = _fresh(planes, alike)
    else:
        out = _planes(out_states)
        _check_out(planes, out)
        if out_states is not states:
            _lib.require_gpu(parents, *out)
    planes = [p if p.is_contiguous() else p.contiguous() for p in planes]
    if alike:
        row_bytes = [planes[0].numel() // rows * sizes[0] if rows else 0] * len(planes)
    else:
        row_bytes = [p.numel() // rows * n if rows else 0 for p, n in zip(planes, sizes)]
    if any([n & 1 for n in row_bytes]):
        raise ValueError("state rows must have an even number of bytes")
    src, dst = array("Q", [p.data_ptr() for p in planes]), array("Q", [o.data_ptr() for o in out])
    row_bytes = array("q", row_bytes)
    _lib.check(_lib.load().sparc_reorder_states(
        B, K, len(planes), src.buffer_info()[0], dst.buffer_info()[0], row_bytes.buffer_info()[0],
        parents.data_ptr(), _lib.stream_of(dev)), "sparc_reorder_states")
    return _like(states, out)


@torch.no_grad()
def beam_search_step(logits: torch.Tensor, scores: torch.Tensor, finished: torch.Tensor | None = None,
                     eos_id: int | None = None, states: Sequence = (),
                     out_states: Sequence | None = None) -> BeamStep:
    """The best K continuations of K hypotheses, for every batch row.

    ``logits``: [B, K, V] float32 or bfloat16 (rows may lie apart, as in
    ``logits[:, -1]`` of a sequence); ``scores``: [B, K] float32
    log-probabilities, -inf for a beam that is not there (before the first
    token: 0 and -inf).  A candidate's score is ``score + (x - logsumexp(x))``
    in fp32.  With ``eos_id``, beams in ``finished`` ([B, K] bool) keep their
    score and append ``eos_id``, and the result's ``finished`` marks the beams
    that have ended.  Ties go to the lowest (beam, token).  A beam whose logits
    are all -inf has -inf candidates; NaN or +inf among its logits make all of
    them NaN, and NaN ranks first, so that it shows.

    ``states``, ``out_states``: as in ``reorder_states``; the states come back
    in the new beams' order.  Nothing waits for the device."""
    if logits.ndim != 3 or 0 in logits.shape[1:] or logits.shape[1] > MAX_BEAMS:
        raise ValueError(f"logits must be [B, K, V] with K from 1 to {MAX_BEAMS}, got {list(logits.shape)}")
    B, K, V = logits.shape
    io = _lib.io_code(logits.dtype)
    _lib.expect(scores, (B, K), torch.float32, "scores")
    if finished is not None:
        _lib.expect(finished, (B, K), torch.bool, "finished")
        if eos_id is None:
            raise ValueError("finished beams need an eos_id")
    if eos_id is not None and not 0 <= eos_id < V:
        raise ValueError(f"eos_id {eos_id} is outside the vocabulary of {V}")
    dev = _lib.require_gpu(logits, scores, finished)
    stride = logits.stride(1) if K > 1 else logits.stride(0) if B > 1 else V
    if (V > 1 and logits.stride(2) != 1) or stride < V or (B > 1 and logits.stride(0) != K * stride):
        logits, stride = logits.contiguous(), V
    scores = scores.contiguous()
    finished = None if finished is None else finished.contiguous()
    lib = _lib.load()
    chosen = torch.empty(2, B, K, dtype=torch.int64, device=dev)
    new_scores = torch.empty(B, K, dtype=torch.float32, device=dev)
    new_finished = None if eos_id is None else torch.empty(B, K, dtype=torch.bool, device=dev)
    need = lib.sparc_beam_workspace_bytes(B, K, V)
    ws = torch.empty(need, dtype=torch.uint8, device=dev)
    P = _lib.ptr
    tokens, parents = chosen[0], chosen[1]
    _lib.check(lib.sparc_beam_step(
        B, K, V, stride, io, logits.data_ptr(), P(scores), P(finished), -1 if eos_id is None else eos_id, P(tokens),
        P(parents), P(new_scores), P(new_finished), P(ws), need, _lib.stream_of(dev)), "sparc_beam_step")
    if len(states):
        states = _reorder(states, parents, out_states)
    return BeamStep(tokens, parents, new_scores, new_finished, list(states))


__all__ = ["BeamStep", "beam_search_step", "reorder_states"]
