"""Float64 CPU restatements of a linear attention block's operators, from their
formulas: norms and rotation of queries and keys, linear attention one step after
another, the gated linear unit.  All are differentiable by autograd.  Test
infrastructure."""
from __future__ import annotations

import math

import torch


def rotary_table(length, dim, base=10000.0):
    table = torch.empty(length, dim, dtype=torch.float64)
    for p in range(length):
        for i in range(dim // 2):
            angle = p * base ** (-2.0 * i / dim)
            table[p, i], table[p, dim // 2 + i] = math.cos(angle), math.sin(angle)
    return table


def norm_rotary(x, weight, table, positions, interleaved, eps):
    """One of queries and keys [B, T, H, D]; positions [B, T]."""
    x = x.double()
    y = x / torch.sqrt(x.square().mean(-1, keepdim=True) + eps)
    y = y if weight is None else y * weight.double()
    R = table.shape[1]
    known = (positions >= 0) & (positions < len(table))
    rows = table.double()[positions.clamp(0, max(len(table) - 1, 0))] if len(table) else torch.zeros(*positions.shape, R)
    rows = torch.where(known[..., None], rows, math.nan)[:, :, None]
    cos, sin = rows[..., :R // 2], rows[..., R // 2:]
    first = torch.arange(R // 2) * (2 if interleaved else 1)
    second = first + (1 if interleaved else R // 2)
    a, b = y[..., first], y[..., second]
    y = y.index_copy(-1, first, a * cos - b * sin).index_copy(-1, second, b * cos + a * sin)
    return torch.where(known[..., None, None], y, math.nan)


def linear_attention(q, k, v, log_decay, state=None, scale=None, lengths=None):
    B, T, H, K = q.shape
    G, V = k.shape[2], v.shape[3]
    scale = K ** -0.5 if scale is None else scale
    q, k, v = q.double(), k.double().repeat_interleave(H // G, 2), v.double().repeat_interleave(H // G, 2)
    a = torch.exp(log_decay.double())[:, None, None]
    s = torch.zeros(B, H, K, V, dtype=torch.float64) if state is None else state.double()
    out = []
    for t in range(T):
        new = a * s + k[:, t, :, :, None] * v[:, t, :, None, :]
        o = scale * (q[:, t, :, :, None] * new).sum(-2)
        if lengths is not None:
            there = (t < lengths)[:, None, None]
            new, o = torch.where(there[..., None], new, s), torch.where(there, o, 0.0)
        s = new
        out.append(o)
    return torch.stack(out, 1) if out else torch.zeros(B, 0, H, V, dtype=torch.float64), s


def activation(g, name):
    if name == "gelu":
        return g * 0.5 * torch.erfc(-g / math.sqrt(2.0))
    if name == "relu":
        return torch.relu(g)  # slope 0 at 0
    return torch.sigmoid(g) if name == "sigmoid" else g * torch.sigmoid(g)


def gated_linear_unit(x, wg, wu, name):
    return activation(x.double() @ wg.double().T, name) * (x.double() @ wu.double().T)
