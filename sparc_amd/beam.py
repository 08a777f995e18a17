"""``beam_search_step`` and ``reorder_states``: one step of beam search over
beams and vocabulary, and recurrent states in the new beams' order, over
sparc_beam_step / sparc_reorder_states.  The states are those of
``SPARCMixer.step`` with one row per hypothesis."""
from __future__ import annotations

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


def _check_out(planes, out):
    if len(out) != len(planes):
        raise ValueError(f"out_states has {len(out)} tensors for {len(planes)} states")
    for o, p in zip(out, planes):
        if o is not p:
            _lib.expect(o, p.shape, p.dtype, "out_states")
        if not o.is_contiguous() or o.is_conj() or o.is_neg():
            raise ValueError("out_states must be contiguous tensors, no views that conjugate or negate")


def reorder_states(states: Sequence, parents: torch.Tensor, out_states: Sequence | None = None) -> list:
    """Every tensor's row b * K + k replaced by its row b * K + parents[b, k].

    ``states``: tensors [B * K, ...], or tuples of them such as the (re, im) of
    ``SPARCMixer.step``, in a list; ``parents``: [B, K] int64, K up to 32.
    ``out_states``: the same structure to write to; it may be ``states`` itself
    (in place: rows that stay are neither read nor written), but no tensor of it
    may overlap another of the states.  By default fresh tensors are returned,
    which share one allocation where all states are of one shape and dtype.  A
    parent outside [0, K) gives a row of NaN.

    There is no backward: outside ``torch.no_grad()`` tensors that require grad
    are refused."""
    if parents.ndim != 2 or parents.dtype != torch.int64 or not 1 <= parents.shape[1] <= MAX_BEAMS:
        raise ValueError(f"parents must be [B, K] int64 with K from 1 to {MAX_BEAMS}, got {list(parents.shape)} "
                         f"{parents.dtype}")
    return _reorder(states, parents, out_states)


def _reorder(states, parents, out_states):
    planes = _planes(states)
    out = None if out_states is None else planes if out_states is states else _planes(out_states)
    new = _lib.native().reorder(planes, parents, out)
    if new is None:
        _refuse_states(planes, parents, out)
    return _like(states, new)


def _refuse_states(planes, parents, out):
    """Raise what is wrong with the states."""
    if out is not None:
        _check_out(planes, out)
    rows = parents.numel()
    for p in planes:
        if not p.ndim or p.shape[0] != rows:
            raise ValueError(f"states must have {rows} rows (one per beam), got {list(p.shape)}")
    _lib.require_gpu(parents, *planes, *(out or ()))
    for p in planes:
        if rows and p.numel() // rows * p.element_size() % 2:
            raise ValueError("state rows must have an even number of bytes")
    raise ValueError("states must be dense tensors")


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
    in the new beams' order.  Nothing waits for the device.

    There is no backward: outside ``torch.no_grad()`` tensors that require grad
    are refused."""
    chosen = _lib.native().beam_step(logits, scores, finished, eos_id, MAX_BEAMS)
    if chosen is None:
        _refuse_step(logits, scores, finished, eos_id)
    if len(states):
        states = _reorder(states, chosen[1], out_states)
    return BeamStep(*chosen, list(states))


def _refuse_step(logits, scores, finished, eos_id):
    """Raise what is wrong with the arguments."""
    if logits.ndim != 3 or 0 in logits.shape[1:] or logits.shape[1] > MAX_BEAMS:
        raise ValueError(f"logits must be [B, K, V] with K from 1 to {MAX_BEAMS}, got {list(logits.shape)}")
    B, K, V = logits.shape
    _lib.io_code(logits.dtype)
    _lib.expect(scores, (B, K), torch.float32, "scores")
    if finished is not None:
        _lib.expect(finished, (B, K), torch.bool, "finished")
        if eos_id is None:
            raise ValueError("finished beams need an eos_id")
    if eos_id is not None and not 0 <= eos_id < V:
        raise ValueError(f"eos_id {eos_id} is outside the vocabulary of {V}")
    _lib.require_gpu(logits, scores, finished)
    raise ValueError("beam_search_step takes dense tensors")


__all__ = ["BeamStep", "beam_search_step", "reorder_states"]
