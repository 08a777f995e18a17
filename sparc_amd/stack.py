"""A stack of SPARC blocks: the model of the 12-layer training configuration.

Each block is pre-norm and residual:

    x <- x + out_proj(SPARCMixer(in_proj(rms_norm(x))))

with ``in_proj`` d_model -> 2M and ``out_proj`` 2M -> d_model (M = d_model *
N complex modes, so the mixer's width is 2M), and a final RMSNorm; with
``norm="layer"`` every norm is a layer norm with a bias instead.  With
``mixer="linear"`` the blocks mix tokens by linear attention with a decay for each
head instead (``LinearAttentionBlock``), and ``feed_forward=F`` puts a gated
feed-forward half of F values behind either mixer.  ``prefill``
and ``step`` run a prompt and then one token at a time, carrying the mixers'
states.  The
projections are plain GEMMs (torch -> hipBLASLt on MI355X); the mixer is the
fused HIP sequence path, with its two control dot products folded into the
input projection (``fuse_projection``).  The reference ships the layer, not a network
(sparc-kernal/sparc.py:58-128); this stack is the configuration the layer is
benchmarked in.
"""
from __future__ import annotations

import os

import torch
import torch.nn.functional as F
from torch import nn

from . import _lib
from . import mixer as _mixer
from .attention import (keep_reach, linear_attention, linear_attention_step, qk_norm_rotary, reach_of,
                        rotary_table)
from .control import aligned16
from .feed_forward import gated_linear_unit
from .norm import layer_norm
from .sparc import SPARCMixer

# Fold the controls into the input projection (see mixer._ProjectedMixer);
# False runs the projection and the module separately, as do hooks on either and
# modules of other classes.
fuse_projection = True
# RMSNorm through sparc_rms_norm_forward / _backward where the shape allows
# (rms_norm below); False keeps torch's RMSNorm.
fused_norm = True


class _RMSNorm(torch.autograd.Function):
    """y = x / sqrt(mean(x^2) + eps) * weight over the last dimension
    (torch.nn.RMSNorm's formula) through the library's RMSNorm kernels; the
    backward's weight gradient is a fixed-order sum over rows."""

    @staticmethod
    def forward(ctx, x, weight, eps):
        lib = _lib.load()
        dev = _lib.require_gpu(x, weight)
        D = x.shape[-1]
        x2 = aligned16(x.detach().reshape(-1, D))
        w = aligned16(weight.detach())
        y = torch.empty_like(x2)
        rstd = torch.empty(x2.shape[0], dtype=torch.float32, device=dev)
        P = _lib.ptr
        _lib.check(lib.sparc_rms_norm_forward(x2.shape[0], D, _lib.io_code(x.dtype), P(x2), P(w), float(eps), P(y),
                                              P(rstd), _lib.stream_of(dev)), "sparc_rms_norm_forward")
        ctx.save_for_backward(x2, w, rstd)
        ctx.wdtype = weight.dtype
        return y.view(x.shape)

    @staticmethod
    def backward(ctx, dy):
        x2, w, rstd = ctx.saved_tensors
        lib = _lib.load()
        dev = x2.device
        rows, D = x2.shape
        dy2 = aligned16(dy.to(x2.dtype).reshape(rows, D))
        dx = torch.empty_like(x2)
        dw = torch.empty(D, dtype=torch.float32, device=dev)
        ws = torch.empty(lib.sparc_rms_norm_workspace_bytes(rows, D), dtype=torch.uint8, device=dev)
        P = _lib.ptr
        _lib.check(lib.sparc_rms_norm_backward(rows, D, _lib.io_code(x2.dtype), P(x2), P(w), P(rstd), P(dy2), P(dx),
                                               P(dw), P(ws), ws.numel(), _lib.stream_of(dev)),
                   "sparc_rms_norm_backward")
        return dx.view(dy.shape), dw.to(ctx.wdtype), None


def _is_observed(module: nn.Module) -> bool:
    """Whether a call of the module does more than its class's forward (hooks, of its
    own or of all modules; a forward of its own)."""
    m = nn.modules.module
    return any(("forward" in vars(module), module._forward_hooks, module._forward_pre_hooks, module._backward_hooks,
                module._backward_pre_hooks, m._global_forward_hooks, m._global_forward_pre_hooks,
                m._global_backward_hooks, m._global_backward_pre_hooks))


def rms_norm(norm: nn.RMSNorm, x: torch.Tensor) -> torch.Tensor:
    """``norm(x)`` through the library's RMSNorm kernels when ``fused_norm``
    is set and the shape allows (GPU tensors, float32 or bfloat16 with the
    weight in the same dtype, a last dimension that is a multiple of 8 up to
    4096), else torch's.  A norm with hooks, or of a class of its own, is called."""
    if type(norm) is not nn.RMSNorm or _is_observed(norm):
        return norm(x)
    D = x.shape[-1]
    w = norm.weight
    if (fused_norm and x.is_cuda and x.dtype in (torch.float32, torch.bfloat16) and w is not None
            and w.dtype == x.dtype and w.shape == (D,) and D % 8 == 0 and D <= 4096 and x.numel() > 0):
        eps = norm.eps if norm.eps is not None else torch.finfo(x.dtype).eps
        return _RMSNorm.apply(x, w, eps)
    return norm(x)


def _make_norm(kind: str, d_model: int, eps: float) -> nn.Module:
    if kind == "rms":
        return nn.RMSNorm(d_model, eps=eps)
    if kind == "layer":
        return nn.LayerNorm(d_model, eps=eps)
    raise ValueError(f"unknown norm {kind!r} (rms or layer)")


def apply_norm(norm: nn.Module, x: torch.Tensor) -> torch.Tensor:
    """``norm(x)`` through the library's kernels: ``layer_norm`` for an
    nn.LayerNorm over the last dimension on the GPU, ``rms_norm`` for an
    nn.RMSNorm.  A norm with hooks, or of a class of its own, is called."""
    if isinstance(norm, nn.LayerNorm):
        if (type(norm) is nn.LayerNorm and not _is_observed(norm) and x.is_cuda
                and x.dtype in (torch.float32, torch.bfloat16) and norm.normalized_shape == (x.shape[-1],)):
            return layer_norm(x, norm.weight, norm.bias, norm.eps)
        return norm(x)
    return rms_norm(norm, x)


def _only_multiplies(module: nn.Module) -> bool:
    """Whether a call of the module is the product with its weight and nothing more,
    so that an operator may take the weight in place of the call."""
    return type(module) is nn.Linear and module.bias is None and not _is_observed(module)


_ACTIVATIONS = {"silu": F.silu, "gelu": F.gelu, "relu": F.relu, "sigmoid": torch.sigmoid}


class GatedFeedForward(nn.Module):
    """down(act(gate(x)) * up(x)): ``gated_linear_unit`` and the projection back.  Where
    ``gate`` or ``up`` does more than multiply by its weight (hooks, a bias, a module
    put in its place), both are called."""

    def __init__(self, d_model: int, hidden: int, activation: str = "silu"):
        super().__init__()
        self.gate = nn.Linear(d_model, hidden, bias=False)
        self.up = nn.Linear(d_model, hidden, bias=False)
        self.down = nn.Linear(hidden, d_model, bias=False)
        if activation not in _ACTIVATIONS:
            raise ValueError(f"unknown activation {activation!r} ({', '.join(_ACTIVATIONS)})")
        self.activation = activation

    def forward(self, x: torch.Tensor) -> torch.Tensor:
        if _only_multiplies(self.gate) and _only_multiplies(self.up):
            return self.down(gated_linear_unit(x, self.gate.weight, self.up.weight, self.activation))
        return self.down(_ACTIVATIONS[self.activation](self.gate(x)) * self.up(x))


class _Block(nn.Module):
    """What blocks of either mixer share: the feed-forward half behind it."""

    def _make_feed_forward(self, d_model: int, hidden: int, norm: str, eps: float) -> None:
        if hidden:
            self.ff_norm = _make_norm(norm, d_model, eps)
            self.ff = GatedFeedForward(d_model, hidden)

    def _feed_forward(self, x: torch.Tensor) -> torch.Tensor:
        return x + self.ff(apply_norm(self.ff_norm, x)) if hasattr(self, "ff") else x

    def prepare_inference(self) -> None:
        """What a decode step needs once."""


class LinearAttentionBlock(_Block):
    """A pre-norm residual block of linear attention: queries, keys and values of one
    projection, the norms of queries and keys with the rotation by their positions
    (``qk_norm_rotary``), ``linear_attention`` with a decay for each head from 32 steps
    of memory to 4096, a norm of each head's output, and the projection back.  The
    state of a row is (S [heads, D, D] fp32, position); positions reach
    ``max_length``, and a prompt or a step behind it is refused.  (How far positions
    reach is kept on the host beside their tensor, and ``step`` and ``reorder_states``
    hand it on.  Positions that a program has made or written itself, copies among
    them, are not checked: behind ``max_length`` outputs and states are NaN.)
    ``table``: the positions' ``rotary_table(max_length, D)``, where other blocks have
    it already."""

    def __init__(self, d_model: int, heads: int, kv_heads: int | None = None, eps: float = 1e-6, norm: str = "rms",
                 feed_forward: int = 0, max_length: int = 65536, table: torch.Tensor | None = None):
        super().__init__()
        kv_heads = heads if kv_heads is None else kv_heads
        if heads < 1 or kv_heads < 1 or d_model % heads or heads % kv_heads or d_model // heads % 2:
            raise ValueError(f"d_model {d_model} must be an even multiple of the {heads} heads, and these a multiple of "
                             f"the {kv_heads} key heads")
        self.heads, self.kv_heads, self.head_dim, self.eps = heads, kv_heads, d_model // heads, eps
        self.norm = _make_norm(norm, d_model, eps)
        self.qkv = nn.Linear(d_model, (heads + 2 * kv_heads) * self.head_dim, bias=False)
        self.q_weight = nn.Parameter(torch.ones(self.head_dim))
        self.k_weight = nn.Parameter(torch.ones(self.head_dim))
        self.head_norm = nn.RMSNorm(self.head_dim, eps=eps)
        self.out_proj = nn.Linear(d_model, d_model, bias=False)
        decay = torch.log1p(-torch.exp2(-5.0 - 7.0 * torch.arange(heads) / max(1, heads - 1)))
        self.register_buffer("log_decay", decay, persistent=False)
        self.register_buffer("table", rotary_table(max_length, self.head_dim) if table is None else table,
                             persistent=False)
        self._make_feed_forward(d_model, feed_forward, norm, eps)

    def _apply(self, fn, recurse=True):
        # the operators take both in fp32, whatever the parameters are converted to
        decay, table = self.log_decay, self.table
        super()._apply(fn, recurse)
        if self.log_decay.dtype != torch.float32:
            self.log_decay, self.table = (t.to(self.log_decay.device) for t in (decay, table))
        return self

    @property
    def max_length(self) -> int:
        return self.table.shape[0]

    def _heads(self, x: torch.Tensor):
        """(q, k, v) [B, T, heads, D] of the block's input, before norms and rotation."""
        both = self.qkv(apply_norm(self.norm, x))
        sizes = [self.heads, self.kv_heads, self.kv_heads]
        return [p.unflatten(-1, (-1, self.head_dim)) for p in both.split([n * self.head_dim for n in sizes], dim=-1)]

    def _out(self, x: torch.Tensor, o: torch.Tensor) -> torch.Tensor:
        return self._feed_forward(x + self.out_proj(rms_norm(self.head_norm, o).flatten(-2)))

    def _attend(self, x: torch.Tensor):
        if x.shape[1] > self.max_length:
            raise ValueError(f"{x.shape[1]} positions are more than max_length {self.max_length}")
        q, k, v = self._heads(x)
        q, k = qk_norm_rotary(q, k, self.q_weight, self.k_weight, self.table, eps=self.eps)
        o, state = linear_attention(q, k, v, self.log_decay)
        return self._out(x, o), state

    def forward(self, x: torch.Tensor) -> torch.Tensor:
        return self._attend(x)[0]

    def prefill(self, x: torch.Tensor):
        """(output, state) of a sequence [B, T, d_model]."""
        y, state = self._attend(x)
        with torch.inference_mode(False):
            position = torch.full((x.shape[0],), x.shape[1], dtype=torch.int64, device=x.device)
        return y, (state, keep_reach(position, x.shape[1]))

    @torch.no_grad()
    def step(self, x: torch.Tensor, state):
        """(output, new state) of one position [B, d_model]; no gradient."""
        s, position = state
        reach = reach_of(position)
        if reach is not None and reach >= self.max_length:
            raise ValueError(f"{reach + 1} positions are more than max_length {self.max_length}")
        q, k, v = self._heads(x[:, None])
        q, k = qk_norm_rotary(q, k, self.q_weight, self.k_weight, self.table, position[:, None], eps=self.eps)
        o, s = linear_attention_step(q[:, 0], k[:, 0], v[:, 0], self.log_decay, s)
        with torch.inference_mode(False):
            position = position + 1
        return self._out(x, o), (s, position if reach is None else keep_reach(position, reach + 1))


class SPARCBlock(_Block):
    def __init__(self, d_model: int, n_states: int, eps: float = 1e-6, norm: str = "rms", feed_forward: int = 0):
        super().__init__()
        modes = d_model * n_states
        self.norm = _make_norm(norm, d_model, eps)
        self.in_proj = nn.Linear(d_model, 2 * modes, bias=False)
        self.mixer = SPARCMixer(2 * modes)
        self.out_proj = nn.Linear(2 * modes, d_model, bias=False)
        with torch.no_grad():  # keep the residual stream's scale at init
            self.out_proj.weight.mul_(1.0 / (2 * modes) ** 0.5)
        self._make_feed_forward(d_model, feed_forward, norm, eps)

    def forward(self, x: torch.Tensor) -> torch.Tensor:
        xn = apply_norm(self.norm, x)
        if fuse_projection and _mixer.get_mixer_path() != "composed" and _only_multiplies(self.in_proj) and \
                type(self.mixer) is SPARCMixer and not _is_observed(self.mixer) and \
                _mixer.projected_fused_supported(xn, self.in_proj.weight):
            y, _ = _mixer.projected_sequence(self.mixer, xn, self.in_proj.weight)
        else:
            y, _ = self.mixer(self.in_proj(xn))
        return self._feed_forward(x + self.out_proj(y))

    def prefill(self, x: torch.Tensor):
        """(output, state) of a sequence [B, T, d_model]: the state is the
        mixer's (re, im) after the last position, fp32 [B, M]."""
        y, state = self.mixer(self.in_proj(apply_norm(self.norm, x)), return_cache=True)
        return self._feed_forward(x + self.out_proj(y)), state

    @torch.no_grad()
    def step(self, x: torch.Tensor, state):
        """(output, new state) of one position [B, d_model]; no gradient, like the
        mixer's step."""
        y, state = self.mixer.step(self.in_proj(apply_norm(self.norm, x)), state, None)
        return self._feed_forward(x + self.out_proj(y)), state

    def prepare_inference(self) -> None:
        """The mixer's fused decode step."""
        self.mixer.prepare_inference()


class SPARCStack(nn.Module):
    """``n_layers`` blocks on a [B, T, d_model] stream: SPARC blocks, or with
    ``mixer="linear"`` ``LinearAttentionBlock`` of ``heads`` (and ``kv_heads``) heads,
    which have no use for ``n_states``; each with a gated feed-forward half of
    ``feed_forward`` values where that is not 0."""

    def __init__(self, n_layers: int, d_model: int, n_states: int, eps: float = 1e-6, norm: str = "rms",
                 mixer: str = "sparc", heads: int | None = None, kv_heads: int | None = None, feed_forward: int = 0,
                 max_length: int = 65536):
        super().__init__()
        if mixer == "sparc":
            make = lambda: SPARCBlock(d_model, n_states, eps, norm, feed_forward)
        elif mixer == "linear":
            if heads is None:
                raise ValueError("linear attention needs heads")
            # one table of angles for all of them (33 MB at 65536 positions and heads of 128)
            make = lambda: LinearAttentionBlock(d_model, heads, kv_heads, eps, norm, feed_forward, max_length,
                                                self.blocks[0].table if len(self.blocks) else None)
        else:
            raise ValueError(f"unknown mixer {mixer!r} (sparc or linear)")
        self.blocks = nn.ModuleList()
        for _ in range(n_layers):
            self.blocks.append(make())
        self.norm = _make_norm(norm, d_model, eps)

    def _apply(self, fn, recurse=True):
        # torch moves the buffers block by block: tables that were one are made one again
        blocks = [blk for blk in self.blocks if isinstance(blk, LinearAttentionBlock)]
        before, after = [blk.table for blk in blocks], {}
        super()._apply(fn, recurse)
        for blk, table in zip(blocks, before):
            blk.table = after.setdefault(id(table), blk.table)
        return self

    @property
    def max_length(self) -> int | None:
        """The positions that all blocks have, or None where there is no limit."""
        return min((blk.max_length for blk in self.blocks if isinstance(blk, LinearAttentionBlock)), default=None)

    def forward(self, x: torch.Tensor) -> torch.Tensor:
        for blk in self.blocks:
            x = blk(x)
        return apply_norm(self.norm, x)

    def prefill(self, x: torch.Tensor):
        """(output, states): ``forward`` and each block's state after the last
        position."""
        states = []
        for blk in self.blocks:
            x, state = blk.prefill(x)
            states.append(state)
        return apply_norm(self.norm, x), states

    @torch.no_grad()
    def step(self, x: torch.Tensor, states):
        """(output, new states) of one position [B, d_model]; no gradient."""
        new = []
        for blk, state in zip(self.blocks, states):
            x, state = blk.step(x, state)
            new.append(state)
        return apply_norm(self.norm, x), new

    def prepare_inference(self) -> None:
        """The mixers' fused decode steps (``SPARCMixer.prepare_inference``)."""
        for blk in self.blocks:
            blk.prepare_inference()


GEMM_TUNING_FILE = os.path.join(os.path.dirname(__file__), "tuning", "gemm_stack_gfx950.csv")


def use_tuned_gemms(path: str = GEMM_TUNING_FILE) -> bool:
    """Route torch's GEMMs through TunableOp with the solutions recorded in
    ``path`` (by default the stack's shapes measured on MI355X, written by
    ``python -m sparc_amd.tuning.tune_stack_gemms``).  Tuning stays off:
    shapes missing from the file keep torch's default solution, and nothing
    is written back.  Returns whether the file was accepted (its validator
    lines must match this torch, HIP, hipBLASLt, rocBLAS and GPU).  The
    setting is process-wide; ``use_default_gemms()`` undoes it."""
    import torch.cuda.tunable as tn
    tn.enable(True)
    tn.tuning_enable(False)
    tn.set_filename(path)
    return bool(tn.read_file(path))


def use_default_gemms() -> None:
    """Switch TunableOp off again (torch's default GEMM solutions)."""
    import torch.cuda.tunable as tn
    tn.enable(False)


def rms_norm_reference(x: torch.Tensor, weight: torch.Tensor, eps: float) -> torch.Tensor:
    """RMSNorm as torch.nn.RMSNorm computes it (for references in other dtypes)."""
    return F.rms_norm(x, (x.shape[-1],), weight, eps)


__all__ = ["SPARCBlock", "LinearAttentionBlock", "GatedFeedForward", "SPARCStack", "apply_norm", "rms_norm", "rms_norm_reference", "use_tuned_gemms", "use_default_gemms",
           "GEMM_TUNING_FILE"]
