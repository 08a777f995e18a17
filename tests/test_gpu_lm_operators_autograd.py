"""The operators around the stack and autograd: what they write in place counts
as written, and what they have no derivative for is refused, never dropped."""
import pytest
import torch

import sparc_amd
from oracle import lm_oracle as L

pytestmark = pytest.mark.gpu


# ---------------------------------------------------------------------------
# tensors written in place
# ---------------------------------------------------------------------------
@pytest.mark.parametrize("strided", [False, True])
def test_a_clipped_gradient_counts_as_written(strided):
    """A backward that has saved the gradient must not read what it was clipped
    to: autograd sees by the version that it was written."""
    print(f"[case] clip version strided={strided}", flush=True)
    wide = torch.randn(20, 30, device="cuda")
    p = torch.nn.Parameter(torch.zeros(20, 9, device="cuda"))
    p.grad = wide[:, 2:11] if strided else wide[:6].view(20, 9)
    q = torch.ones(20, 9, device="cuda", requires_grad=True)
    loss = (q * p.grad).sum()
    version = p.grad._version
    sparc_amd.grad_norm([p.grad])
    assert p.grad._version == version  # read only
    sparc_amd.clip_grad_norm_([p], 0.5)
    assert p.grad._version > version
    with pytest.raises(RuntimeError, match="inplace operation"):
        loss.backward()


@pytest.mark.parametrize("in_place", [False, True])
def test_a_reordered_state_counts_as_written(in_place):
    print(f"[case] reorder version in_place={in_place}", flush=True)
    state, out = torch.randn(6, 8, device="cuda"), torch.randn(6, 8, device="cuda")
    parents = torch.tensor([[2, 1, 0], [0, 0, 1]], device="cuda")
    written = state if in_place else out
    q = torch.ones(6, 8, device="cuda", requires_grad=True)
    of_state, of_written = (q * state).sum(), (q * written).sum()
    sparc_amd.reorder_states([state], parents)
    assert state._version == out._version == 0
    sparc_amd.reorder_states([state], parents, out_states=[written])
    assert written._version == 1
    with pytest.raises(RuntimeError, match="inplace operation"):
        of_written.backward()
    if not in_place:  # a state that was only read is as it was
        of_state.backward()
        assert torch.equal(q.grad, state)


def test_states_of_a_step_count_as_written():
    print("[case] beam step version", flush=True)
    logits, scores = torch.randn(2, 3, 50, device="cuda"), torch.zeros(2, 3, device="cuda")
    states = [(torch.randn(6, 8, device="cuda"), torch.randn(6, 8, device="cuda"))]
    q = torch.ones(6, 8, device="cuda", requires_grad=True)
    loss = (q * states[0][1]).sum()
    sparc_amd.beam_search_step(logits, scores, states=states, out_states=states)
    with pytest.raises(RuntimeError, match="inplace operation"):
        loss.backward()


def test_a_leaf_that_requires_grad_is_not_written():
    """As torch: an error, except under no_grad."""
    print("[case] reorder into a leaf", flush=True)
    state, leaf = torch.randn(6, 8, device="cuda"), torch.zeros(6, 8, device="cuda", requires_grad=True)
    parents = torch.tensor([[2, 1, 0], [0, 0, 1]], device="cuda")
    with pytest.raises(RuntimeError, match="require"):
        sparc_amd.reorder_states([state], parents, out_states=[leaf])
    torch.cuda.synchronize()
    assert not leaf.detach().any()
    with torch.no_grad():
        sparc_amd.reorder_states([state], parents, out_states=[leaf])
    assert torch.equal(leaf.detach().cpu(), L.reorder(state.cpu(), parents.cpu()))


def test_clipping_under_no_grad_rules():
    """A gradient that is part of a graph is clipped as torch clips it: in place,
    whatever the grad mode."""
    print("[case] clip gradient with a graph", flush=True)
    w = torch.randn(40, device="cuda", requires_grad=True)
    w.grad, = torch.autograd.grad(w.pow(3).sum(), w, create_graph=True)
    want = w.grad.detach().double()
    norm = sparc_amd.clip_grad_norm_([w], 0.25)
    assert not norm.requires_grad
    assert ((w.grad.double() - want * (0.25 / (want.norm() + 1e-6))).abs() <= 2.0 ** -21 * want.abs()).all()
