"""The last position that a block of linear attention has angles for, and the one behind
it: in prompts, steps and beam search."""
import pytest
import torch

from sparc_amd import lm, reorder_states
from sparc_amd.stack import SPARCStack

pytestmark = pytest.mark.gpu
LENGTH = 12


def _stack(**options):
    torch.manual_seed(0)
    return SPARCStack(2, 32, 1, mixer="linear", heads=4, kv_heads=2, max_length=LENGTH, **options).cuda()


def test_steps_end_at_max_length():
    stack = _stack()
    x = torch.randn(3, LENGTH + 1, 32, device="cuda")
    with torch.no_grad():
        want = stack(x[:, :LENGTH])
        _, states = stack.prefill(x[:, :LENGTH - 2])
        for t in (LENGTH - 2, LENGTH - 1):
            y, states = stack.step(x[:, t], states)
    torch.testing.assert_close(y, want[:, -1], rtol=1e-4, atol=1e-4)
    before = [(s.clone(), position.clone()) for s, position in states]
    with pytest.raises(ValueError, match="max_length"):
        stack.step(x[:, LENGTH], states)
    assert all(torch.equal(a, b) for old, new in zip(before, states) for a, b in zip(old, new))


def test_a_whole_prompt_leaves_no_step():
    stack = _stack()
    x = torch.randn(1, LENGTH, 32, device="cuda")
    with torch.no_grad():
        _, states = stack.prefill(x)
    with pytest.raises(ValueError, match="max_length"):
        stack.step(x[:, 0], states)
    with pytest.raises(ValueError, match="max_length"):
        stack.blocks[1].step(x[:, 0], states[1])


@pytest.mark.parametrize("in_place", [False, True])
def test_reordered_states_end_there_too(in_place):
    stack = _stack()
    x = torch.randn(4, LENGTH, 32, device="cuda")
    with torch.no_grad():
        _, states = stack.prefill(x[:, :LENGTH - 1])
        states = reorder_states(states, torch.tensor([[1, 0], [1, 1]], device="cuda"),
                                out_states=states if in_place else None)
        _, states = stack.step(x[:, -1], states)
    with pytest.raises(ValueError, match="max_length"):
        stack.step(x[:, 0], states)


@pytest.mark.parametrize("mode", [torch.no_grad, torch.inference_mode], ids=["no_grad", "inference"])
def test_positions_that_a_program_writes(mode):
    """A state used again from the first position on is no longer at its end."""
    stack = _stack()
    x = torch.randn(2, LENGTH, 32, device="cuda")
    with mode():
        want = stack(x)
        _, states = stack.prefill(x)
        with pytest.raises(ValueError, match="max_length"):
            stack.step(x[:, 0], states)
        for s, position in states:
            s.zero_(), position.zero_()
        parts = []
        for t in range(LENGTH):
            y, states = stack.step(x[:, t], states)
            parts.append(y)
        assert states[0][1].tolist() == [LENGTH] * 2
        _, states = stack.prefill(x[:, :LENGTH - 1])
        _, states = stack.step(x[:, -1], states)
        with pytest.raises(ValueError, match="max_length"):
            stack.step(x[:, 0], states)
    torch.testing.assert_close(torch.stack(parts, 1), want, rtol=1e-4, atol=1e-4)


def test_max_length_of_a_stack():
    assert _stack().max_length == LENGTH
    assert SPARCStack(1, 32, 1).max_length is None
    stack = _stack()
    stack.blocks[1] = SPARCStack(1, 32, 1, mixer="linear", heads=4, max_length=LENGTH - 1).blocks[0].cuda()
    assert stack.max_length == LENGTH - 1


def test_beam_search_ends_at_max_length():
    torch.manual_seed(1)
    model = lm.SPARCLanguageModel(20, 2, 32, 1, mixer="linear", heads=4, max_length=LENGTH).cuda()
    prompt = torch.randint(0, 20, (2, LENGTH - 3), device="cuda")
    ids, scores = lm.beam_search(model, prompt, beams=2, steps=4)  # the last id needs no position
    assert ids.shape == (2, 2, 4) and scores.isfinite().all()
    with pytest.raises(ValueError, match="max_length"):
        lm.beam_search(model, prompt, beams=2, steps=5)
    full = torch.randint(0, 20, (1, LENGTH), device="cuda")
    assert lm.beam_search(model, full, beams=2, steps=1)[1].isfinite().all()
    assert lm.beam_search(model, full, beams=2, steps=0)[0].shape == (1, 2, 0)
    sparc = lm.SPARCLanguageModel(20, 1, 32, 1).cuda()
    assert lm.beam_search(sparc, prompt, beams=2, steps=5)[1].isfinite().all()


@pytest.mark.parametrize("mode", [torch.no_grad, torch.inference_mode], ids=["no_grad", "inference"])
def test_a_captured_step(mode):
    """Replays read positions from the state's tensors, which the host does not follow:
    the last one's angles are there, and behind it outputs are NaN."""
    stack = _stack(feed_forward=48)
    x = torch.randn(2, LENGTH + 1, 32, device="cuda")
    with mode():
        want = stack(x[:, :LENGTH])
        _, states = stack.prefill(x[:, :3])
        token = x[:, 3].clone()
        side = torch.cuda.Stream()
        side.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(side):  # what the first call allocates
            stack.step(token, states)
        torch.cuda.current_stream().wait_stream(side)
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            y, new = stack.step(token, states)
        for t in range(3, LENGTH + 1):
            token.copy_(x[:, t])
            graph.replay()
            for old, fresh in zip(states, new):
                for a, b in zip(old, fresh):
                    a.copy_(b)
            if t < LENGTH:
                torch.testing.assert_close(y, want[:, t], rtol=1e-4, atol=1e-4)
            else:
                assert y.isnan().all()
