"""A language model around the SPARC block stack, for training and for beam
search: ids -> scaled embedding -> blocks with layer norms -> logits over the
(tied) embedding table.

It runs the operators around the stack together as they are used: ``embedding``
with its gradient by sorted tokens, ``layer_norm``, ``clip_grad_norm_`` in a
training step, and ``beam_search_step`` with the blocks' recurrent states
reordered in place.  The reference ships the layer, not a network.

``python -m sparc_amd.lm`` trains a small model on a synthetic sequence task
and continues a prompt with beam search.
"""
from __future__ import annotations

import argparse
import math

import torch
import torch.nn.functional as F
from torch import nn

from .beam import beam_search_step
from .clip import clip_grad_norm_
from .embed import embedding
from .stack import SPARCStack


class SPARCLanguageModel(nn.Module):
    """Logits [B, T, vocab] of ids [B, T].  The embedding is scaled by
    sqrt(d_model) and its table is the output projection too; ``padding_idx``
    takes no gradient from the lookup (negative counts from the end)."""

    def __init__(self, vocab: int, n_layers: int, d_model: int, n_states: int, padding_idx: int | None = None,
                 norm: str = "layer"):
        super().__init__()
        if padding_idx is not None:
            if not -vocab <= padding_idx < vocab:
                raise ValueError(f"padding_idx {padding_idx} is outside the vocabulary of {vocab}")
            padding_idx %= vocab  # the id itself: targets are compared with it
        self.weight = nn.Parameter(torch.randn(vocab, d_model) * d_model ** -0.5)
        self.scale = math.sqrt(d_model)
        self.padding_idx = padding_idx
        self.stack = SPARCStack(n_layers, d_model, n_states, norm=norm)

    def embed(self, tokens: torch.Tensor) -> torch.Tensor:
        return embedding(tokens, self.weight, scale=self.scale, padding_idx=self.padding_idx)

    def forward(self, tokens: torch.Tensor) -> torch.Tensor:
        return F.linear(self.stack(self.embed(tokens)), self.weight)

    def prefill(self, tokens: torch.Tensor):
        """(logits [B, vocab] after the last position, states)."""
        h, states = self.stack.prefill(self.embed(tokens))
        return F.linear(h[:, -1], self.weight), states

    @torch.no_grad()
    def step(self, tokens: torch.Tensor, states):
        """(logits [B, vocab], new states) after one more id each, [B]; no
        gradient, like the mixers' steps."""
        h, states = self.stack.step(self.embed(tokens), states)
        return F.linear(h, self.weight), states


def train_step(model: SPARCLanguageModel, optimizer: torch.optim.Optimizer, tokens: torch.Tensor, max_norm: float):
    """One step of next-token training on ids [B, T + 1]; returns (loss,
    gradient norm before clipping), both on the device."""
    logits = model(tokens[:, :-1])
    ignore = -100 if model.padding_idx is None else model.padding_idx
    loss = F.cross_entropy(logits.flatten(0, 1).float(), tokens[:, 1:].reshape(-1).long(), ignore_index=ignore)
    optimizer.zero_grad(set_to_none=True)
    loss.backward()
    norm = clip_grad_norm_(model.parameters(), max_norm)
    optimizer.step()
    return loss.detach(), norm


@torch.no_grad()
def beam_search(model: SPARCLanguageModel, prompt: torch.Tensor, beams: int, steps: int, eos_id: int | None = None):
    """The ``beams`` best continuations of each prompt row [B, T] by ``steps``
    ids: (ids [B, beams, steps], scores [B, beams]), best first.  With
    ``eos_id`` a hypothesis that has ended keeps its score and repeats
    ``eos_id``.  Nothing waits for the device between the steps."""
    model.stack.prepare_inference()
    logits, states = model.prefill(prompt)
    B, V = logits.shape
    states = [tuple(p.repeat_interleave(beams, dim=0) for p in s) for s in states]
    logits = logits.repeat_interleave(beams, dim=0)
    scores = torch.full((B, beams), -math.inf, device=prompt.device)
    scores[:, 0] = 0.0  # one hypothesis so far
    finished = None
    ids = torch.empty(B, beams, 0, dtype=torch.int64, device=prompt.device)
    for k in range(steps):
        # the states are this loop's own, so they are reordered in place
        step = beam_search_step(logits.view(B, beams, V), scores, finished=finished, eos_id=eos_id, states=states,
                                out_states=states)
        scores, finished, states = step.scores, step.finished, step.states
        ids = torch.cat((ids.gather(1, step.parents[..., None].expand(-1, -1, k)), step.tokens[..., None]), dim=-1)
        if k + 1 < steps:
            logits, states = model.step(step.tokens.reshape(-1), states)
    return ids, scores


def main(argv=None) -> None:
    """Trains on sequences that count up by a step of their own, modulo the
    vocabulary, and continues one of them."""
    ap = argparse.ArgumentParser(description=main.__doc__)
    ap.add_argument("--vocab", type=int, default=64)
    ap.add_argument("--layers", type=int, default=2)
    ap.add_argument("--d-model", type=int, default=64)
    ap.add_argument("--states", type=int, default=8)
    ap.add_argument("--steps", type=int, default=200)
    ap.add_argument("--beams", type=int, default=4)
    a = ap.parse_args(argv)
    torch.manual_seed(0)
    model = SPARCLanguageModel(a.vocab, a.layers, a.d_model, a.states).cuda()
    optimizer = torch.optim.AdamW(model.parameters(), lr=3e-3)
    for i in range(a.steps):
        start, by = torch.randint(0, a.vocab, (32, 1)), torch.randint(1, 4, (32, 1))
        tokens = ((start + by * torch.arange(33)) % a.vocab).cuda()
        loss, norm = train_step(model, optimizer, tokens, max_norm=1.0)
        if i % 20 == 0 or i + 1 == a.steps:
            print(f"step {i}: loss {loss.item():.4f}, gradient norm {norm.item():.3f}", flush=True)
    prompt = ((5 + 2 * torch.arange(12)) % a.vocab)[None].cuda()
    ids, scores = beam_search(model, prompt, a.beams, 8)
    print("prompt ", prompt[0].tolist())
    for k in range(a.beams):
        print(f"beam {k}: score {scores[0, k].item():8.3f}  {ids[0, k].tolist()}")


if __name__ == "__main__":
    main()

__all__ = ["SPARCLanguageModel", "train_step", "beam_search"]
