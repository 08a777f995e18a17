"""Linear attention blocks and gated feed-forward halves in the stack and the language
model: against the same block in 64 bits, and a prompt in pieces, a training step and
a beam search over them."""
import pytest
import torch
import torch.nn.functional as F

from oracle import block_oracle as O
from sparc_amd import lm
from sparc_amd.stack import LinearAttentionBlock, SPARCStack

pytestmark = pytest.mark.gpu


def _reference(block, x):
    """The block's formula in 64 bits on the CPU, differentiable in its parameters."""
    p = {n: t.detach().cpu().double().requires_grad_() for n, t in block.named_parameters()}
    eps, H, G, D = block.eps, block.heads, block.kv_heads, block.head_dim
    rms = lambda y, w: y / torch.sqrt(y.square().mean(-1, keepdim=True) + eps) * w
    B, T, _ = x.shape
    both = rms(x, p["norm.weight"]) @ p["qkv.weight"].T
    q, k, v = (t.unflatten(-1, (-1, D)) for t in both.split([H * D, G * D, G * D], -1))
    at = torch.arange(T).expand(B, T)
    table = O.rotary_table(T, D)
    q, k = (O.norm_rotary(t, p[n], table, at, False, eps) for t, n in ((q, "q_weight"), (k, "k_weight")))
    o, state = O.linear_attention(q, k, v, block.log_decay.cpu())
    y = x + rms(o, p["head_norm.weight"]).flatten(-2) @ p["out_proj.weight"].T
    h = rms(y, p["ff_norm.weight"])
    y = y + O.gated_linear_unit(h, p["ff.gate.weight"], p["ff.up.weight"], "silu") @ p["ff.down.weight"].T
    return y, state, p


def test_a_block_is_its_formula():
    """fp32: the largest error of a result against its largest value.  Some 20
    operators follow one another, none of sums longer than 64 terms or steps, which
    each add at most 64 2^-24 of their terms' sizes; sizes exceed results by up to ten
    times: 20 * 64 * 10 * 2^-24 = 8e-4."""
    torch.manual_seed(0)
    block = LinearAttentionBlock(48, heads=4, kv_heads=2, feed_forward=40, max_length=64).cuda()
    x = torch.randn(2, 33, 48)
    dy = torch.randn(2, 33, 48)
    leaf = x.cuda().requires_grad_()
    y = block(leaf)
    y.backward(dy.cuda())
    ref_x = x.double().requires_grad_()
    ref, state, params = _reference(block, ref_x)
    ref.backward(dy.double())
    near = lambda a, b: (a.detach().cpu().double() - b).abs().max() <= 8e-4 * b.abs().max()
    assert near(y, ref.detach()) and near(leaf.grad, ref_x.grad)
    for n, p in block.named_parameters():
        assert near(p.grad, params[n].grad), n
    _, (s, position) = block.prefill(x.cuda())
    assert near(s, state.detach()) and position.tolist() == [33, 33]


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16], ids=["f32", "bf16"])
@pytest.mark.parametrize("mixer", ["sparc", "linear"])
def test_a_prompt_and_steps_are_the_sequence(mixer, dtype):
    """In bfloat16 every operator rounds, the steps' and the sequence's alike but not at
    the same values: compared by the 2-norm, at 3 layers * 10 roundings * 2^-8 / 2."""
    torch.manual_seed(1)
    stack = SPARCStack(3, 64, 4, mixer=mixer, heads=4, kv_heads=2, feed_forward=96, max_length=32).cuda().to(dtype)
    x = torch.randn(2, 20, 64, device="cuda", dtype=dtype)
    with torch.no_grad():
        y = stack(x)
        stack.prepare_inference()
        z, states = stack.prefill(x[:, :13])
        parts = [z]
        for t in range(13, 20):
            z, states = stack.step(x[:, t], states)
            parts.append(z[:, None])
    off = (torch.cat(parts, 1).float() - y.float()).norm() / y.float().norm()
    assert off <= (1e-4 if dtype == torch.float32 else 0.06)


def test_buffers_stay_fp32_where_parameters_do_not():
    block = LinearAttentionBlock(32, heads=2, max_length=8).to(torch.bfloat16).cuda()
    assert block.log_decay.dtype == block.table.dtype == torch.float32 and block.table.is_cuda
    assert block.qkv.weight.dtype == torch.bfloat16
    assert not {"log_decay", "table"} & set(block.state_dict())
    with pytest.raises(ValueError, match="max_length"):
        block(torch.zeros(1, 9, 32, device="cuda", dtype=torch.bfloat16))


@pytest.mark.parametrize("mixer", ["sparc", "linear"])
def test_training_step_and_beam_search(mixer):
    torch.manual_seed(2)
    model = lm.SPARCLanguageModel(50, 2, 64, 4, mixer=mixer, heads=4, feed_forward=80).cuda()
    optimizer = torch.optim.SGD(model.parameters(), lr=0.1)
    tokens = torch.randint(0, 50, (3, 12), device="cuda")
    loss, norm = lm.train_step(model, optimizer, tokens, 1.0)
    assert loss.isfinite() and norm.isfinite()
    assert all(p.grad is not None and p.grad.isfinite().all() for p in model.parameters())
    ids, scores = lm.beam_search(model, tokens, beams=3, steps=4)
    assert ids.shape == (3, 3, 4) and (scores[:, :-1] >= scores[:, 1:]).all()
    # a hypothesis' score is that of its ids after the prompt
    for k in range(3):
        with torch.no_grad():
            logp = F.log_softmax(model(torch.cat((tokens, ids[:, k]), 1)[:, :-1]).float(), -1)
        own = logp[:, 11:].gather(-1, ids[:, k, :, None]).sum((1, 2))
        torch.testing.assert_close(own, scores[:, k], rtol=1e-4, atol=1e-4)


def test_the_command_runs(capsys):
    lm.main(["--mixer", "linear", "--feed-forward", "64", "--steps", "3", "--layers", "1"])
    out = capsys.readouterr().out
    assert "step 2" in out and "beam 3" in out
