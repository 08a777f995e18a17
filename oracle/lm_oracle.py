"""Float64 CPU restatements of the operators around the block stack, from
their formulas: layer norm, embedding, gradient clipping, one beam search step
and the states' reordering.  Test infrastructure."""
from __future__ import annotations

import math

import torch


def layer_norm(x, weight, bias, eps):
    x = x.double()
    mu = x.mean(-1, keepdim=True)
    y = (x - mu) / torch.sqrt((x - mu).square().mean(-1, keepdim=True) + eps)
    y = y if weight is None else y * weight.double()
    return y if bias is None else y + bias.double()


def layer_norm_grads(x, weight, eps, dy):
    """dx, dweight, dbias of the formula for the incoming gradient dy."""
    x, dy = x.double(), dy.double()
    mu = x.mean(-1, keepdim=True)
    rstd = 1.0 / torch.sqrt((x - mu).square().mean(-1, keepdim=True) + eps)
    xhat = (x - mu) * rstd
    g = dy if weight is None else dy * weight.double()
    dx = rstd * (g - g.mean(-1, keepdim=True) - xhat * (g * xhat).mean(-1, keepdim=True))
    D = x.shape[-1]
    return dx, (dy * xhat).reshape(-1, D).sum(0), dy.reshape(-1, D).sum(0)


def embedding(tokens, weight, scale):
    flat = tokens.reshape(-1).long()
    y = torch.full((flat.numel(), weight.shape[1]), math.nan, dtype=torch.float64)
    ok = (flat >= 0) & (flat < weight.shape[0])
    y[ok] = weight.double()[flat[ok]] * scale
    return y.view(*tokens.shape, weight.shape[1])


def embedding_grad(tokens, vocab, dy, scale, padding_idx=None):
    flat = tokens.reshape(-1).long()
    dy = dy.double().reshape(flat.numel(), -1)
    ok = (flat >= 0) & (flat < vocab)
    if padding_idx is not None:
        ok &= flat != padding_idx % vocab
    dw = torch.zeros(vocab, dy.shape[1], dtype=torch.float64)
    for n in torch.nonzero(ok).reshape(-1).tolist():
        dw[flat[n]] += scale * dy[n]
    return dw


def grad_norm(tensors):
    return math.sqrt(sum(float(t.double().square().sum()) for t in tensors))


def clip_factor(tensors, max_norm):
    return min(1.0, max_norm / (grad_norm(tensors) + 1e-6))


def beam_candidates(logits, scores, finished=None, eos_id=None):
    """All candidates' scores [B, K, V]."""
    x, scores = logits.double(), scores.double()
    top = x.amax(-1, keepdim=True)
    lse = top + torch.log(torch.exp(x - top).sum(-1, keepdim=True))
    logp = torch.where(torch.isneginf(top), torch.full_like(x, -math.inf), x - lse)
    cand = scores[..., None] + logp
    if finished is not None:
        cand = torch.where(finished[..., None], torch.full_like(cand, -math.inf), cand)
        cand[..., eos_id] = torch.where(finished, scores, cand[..., eos_id])
    return cand


def beam_step(logits, scores, finished=None, eos_id=None):
    """(tokens, parents, scores, finished) with ties to the lowest beam * V +
    token and NaN above every number."""
    cand = beam_candidates(logits, scores, finished, eos_id)
    B, K, V = cand.shape
    best, at = torch.sort(cand.reshape(B, K * V), dim=-1, descending=True, stable=True)
    best, at = best[:, :K], at[:, :K]
    parents, tokens = at // V, at % V
    if eos_id is None:
        return tokens, parents, best, None
    was = torch.zeros_like(scores, dtype=torch.bool) if finished is None else finished
    return tokens, parents, best, was.gather(1, parents) | (tokens == eos_id)


def reorder(plane, parents):
    B, K = parents.shape
    rows = (parents + K * torch.arange(B)[:, None]).reshape(-1)
    return plane[rows]
