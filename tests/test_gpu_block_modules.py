"""What a block's modules do beyond their formulas: hooks, adapters, biases and forwards
of their own count in the stack as they do where torch calls the module.

The comparisons are of fp32 results of sums of 48 terms or fewer that two programs
compute in different orders, one after the other: 4 roundings of such sums, each of up to
48 2^-24 of terms that exceed the results by up to ten times: 1.2e-4."""
import pytest
import torch
import torch.nn.functional as F
from torch import nn

from sparc_amd import stack

pytestmark = pytest.mark.gpu
TOL = dict(rtol=1.2e-4, atol=1.2e-4)
D, HIDDEN = 32, 48


class Adapted(nn.Linear):
    """A low-rank adapter beside a projection."""

    def __init__(self, d_in, d_out):
        super().__init__(d_in, d_out, bias=False)
        self.down, self.up = nn.Linear(d_in, 2, bias=False), nn.Linear(2, d_out, bias=False)

    def forward(self, x):
        return super().forward(x) + self.up(self.down(x))


class Wrapped(nn.Module):
    """A projection without a weight of its own."""

    def __init__(self, d_in, d_out):
        super().__init__()
        self.inner = nn.Linear(d_in, d_out, bias=False)

    def forward(self, x):
        return 2.0 * self.inner(x)


def _change(parent, name, kind, seen):
    """The kind of change at a module; returns a handle or None."""
    module = getattr(parent, name)
    if kind == "forward hook":
        return module.register_forward_hook(lambda mod, args, y: y + 1.0)
    if kind == "pre hook":
        return module.register_forward_pre_hook(lambda mod, args: (args[0] * 0.5,))
    if kind == "backward hook":
        return module.register_full_backward_hook(lambda mod, gx, gy: seen.append(mod))
    if kind == "global hook":
        return nn.modules.module.register_module_forward_hook(
            lambda mod, args, y: y + 1.0 if mod is module else None)
    if kind == "own forward":
        inner = module.forward
        module.forward = lambda x: 3.0 * inner(x)
    elif kind == "bias":
        module.bias = nn.Parameter(torch.randn(module.out_features, device="cuda"))
    elif kind == "adapter":
        setattr(parent, name, Adapted(module.in_features, module.out_features).cuda())
    elif kind == "wrapper":
        setattr(parent, name, Wrapped(module.in_features, module.out_features).cuda())
    elif kind == "parametrization":
        class Double(nn.Module):
            def forward(self, w):
                return 2.0 * w
        nn.utils.parametrize.register_parametrization(module, "weight", Double())
    return None


KINDS = ["forward hook", "pre hook", "backward hook", "global hook", "own forward", "bias", "adapter", "wrapper",
         "parametrization"]
ACTS = {"silu": F.silu, "gelu": F.gelu, "relu": F.relu, "sigmoid": torch.sigmoid}


def _both(run, want_of, x, handle):
    """A result and what it should be, each with the gradient of x."""
    found = []
    try:
        for f in (run, want_of):
            leaf = x.clone().requires_grad_()
            y = f(leaf)
            y.square().sum().backward()
            found.append((y.detach(), leaf.grad))
    finally:
        if handle is not None:
            handle.remove()
    for got, want in zip(*found):
        torch.testing.assert_close(got / want.abs().max(), want / want.abs().max(), **TOL)


@pytest.mark.parametrize("activation", ["silu", "gelu", "relu", "sigmoid"])
def test_a_feed_forward_half_is_its_modules(activation):
    torch.manual_seed(0)
    ff = stack.GatedFeedForward(D, HIDDEN, activation).cuda()
    act = ACTS[activation]
    _both(ff, lambda x: ff.down(act(ff.gate(x)) * ff.up(x)), torch.randn(3, 5, D, device="cuda"), None)


@pytest.mark.parametrize("name", ["gate", "up"])
@pytest.mark.parametrize("kind", KINDS)
def test_changed_projections_of_a_feed_forward_half(kind, name):
    print(f"[case] {kind} at {name}", flush=True)
    torch.manual_seed(1)
    ff, seen = stack.GatedFeedForward(D, HIDDEN).cuda(), []
    handle = _change(ff, name, kind, seen)
    _both(ff, lambda x: ff.down(F.silu(ff.gate(x)) * ff.up(x)), torch.randn(3, 5, D, device="cuda"), handle)
    assert len(seen) == (2 if kind == "backward hook" else 0)


def test_unknown_activations_are_refused():
    with pytest.raises(ValueError, match="activation"):
        stack.GatedFeedForward(D, HIDDEN, "tanh").cuda()(torch.zeros(1, D, device="cuda"))


@pytest.mark.parametrize("kind", ["forward hook", "pre hook", "backward hook", "global hook", "own forward", "subclass",
                                  "another module"])
def test_an_rms_norm_is_called_with_its_hooks(kind):
    print(f"[case] rms norm, {kind}", flush=True)
    torch.manual_seed(2)
    block, seen = stack.LinearAttentionBlock(D, heads=4, max_length=8).cuda(), []
    if kind == "subclass":
        class Centred(nn.RMSNorm):
            def forward(self, x):
                return super().forward(x - x.mean(-1, keepdim=True))
        block.head_norm, handle = Centred(D // 4).cuda(), None
    elif kind == "another module":
        block.head_norm, handle = nn.Tanh(), None
    else:
        handle = _change(block, "head_norm", kind, seen)
    _both(lambda x: stack.apply_norm(block.head_norm, x), lambda x: block.head_norm(x),
          torch.randn(3, 5, D // 4, device="cuda"), handle)
    assert len(seen) == (2 if kind == "backward hook" else 0)


@pytest.mark.parametrize("mixer", ["sparc", "linear"])
def test_a_stack_calls_every_norm_that_is_observed(mixer):
    torch.manual_seed(3)
    model = stack.SPARCStack(2, D, 2, mixer=mixer, heads=4, feed_forward=HIDDEN, max_length=8).cuda()
    norms, seen = [m for m in model.modules() if isinstance(m, nn.RMSNorm)], []
    for m in norms:
        m.register_forward_hook(lambda mod, args, y: seen.append(mod))
    model(torch.randn(2, 8, D, device="cuda"))
    assert set(seen) == set(norms) and len(seen) == len(norms) == (7 if mixer == "linear" else 5)


@pytest.mark.parametrize("kind,name", [(kind, "in_proj") for kind in KINDS] + [
    (kind, "mixer") for kind in ("pre hook", "backward hook", "own forward")])
def test_changed_modules_of_a_sparc_block(kind, name):
    """A fused call takes the projection and the mixer together where neither does more."""
    print(f"[case] {kind} at {name}", flush=True)
    torch.manual_seed(4)
    block, seen = stack.SPARCBlock(D, 2).cuda(), []
    if name == "mixer" and kind == "own forward":
        inner, handle = block.mixer.forward, None
        block.mixer.forward = lambda x, return_cache=False: inner(-x, return_cache)
    else:
        handle = _change(block, name, kind, seen)
    _both(block, lambda x: x + block.out_proj(block.mixer(block.in_proj(block.norm(x)))[0]),
          torch.randn(2, 16, D, device="cuda"), handle)
    assert len(seen) == (2 if kind == "backward hook" else 0)
