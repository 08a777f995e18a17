"""The language model around the stack: its training step against the same
model on torch's own embedding, layer norm and clipping, and beam search
against an exhaustive search over the model's whole-sequence logits."""
import itertools
import math

import pytest
import torch
import torch.nn.functional as F

from sparc_amd import lm, stack

pytestmark = pytest.mark.gpu


def _model(vocab, layers, d_model, n_states, seed=0, **kw):
    torch.manual_seed(seed)
    m = lm.SPARCLanguageModel(vocab, layers, d_model, n_states, **kw)
    g = torch.Generator().manual_seed(seed + 1)
    with torch.no_grad():
        for blk in m.stack.blocks:
            w = blk.mixer.width
            blk.mixer.phase_direction.copy_(0.5 * torch.randn(w + 1, generator=g) / math.sqrt(w))
            blk.mixer.radial_direction.copy_(0.5 * torch.randn(w + 1, generator=g) / math.sqrt(w))
            blk.mixer.write_phase_response.copy_(torch.randn(w // 2, generator=g))
            blk.norm.weight.copy_(1.0 + 0.2 * torch.randn(d_model, generator=g))
            blk.norm.bias.copy_(0.2 * torch.randn(d_model, generator=g))
            blk.out_proj.weight.mul_(8.0)
    return m.cuda()


def test_training_step_against_torch_operators(monkeypatch):
    """fp32: loss, gradients and norm with the library's operators and with
    torch's, through the same mixers.  Both round every operator at 2^-24 over
    sums of up to 90 tokens x 24 channels; held to 1e-4 of each gradient's
    largest value, the tolerance of the mixers' own gradients."""
    print("[case] lm training step", flush=True)
    m = _model(53, 2, 24, 4, padding_idx=0)
    g = torch.Generator().manual_seed(5)
    tokens = torch.randint(1, 53, (3, 31), generator=g)
    tokens[1, 20:] = 0
    tokens = tokens.cuda()

    def run():
        opt = torch.optim.SGD(m.parameters(), lr=0.0)
        loss, norm = lm.train_step(m, opt, tokens, max_norm=0.1)
        return float(loss), float(norm), {n: p.grad.clone() for n, p in m.named_parameters() if p.grad is not None}

    ours = run()
    monkeypatch.setattr(lm, "embedding", lambda t, w, scale, padding_idx: scale * F.embedding(t, w, padding_idx))
    monkeypatch.setattr(stack, "apply_norm", lambda n, x: F.layer_norm(x, (x.shape[-1],), n.weight, n.bias, n.eps))
    monkeypatch.setattr(lm, "clip_grad_norm_", torch.nn.utils.clip_grad_norm_)
    theirs = run()
    assert abs(ours[0] - theirs[0]) <= 1e-5 * abs(theirs[0]) and abs(ours[1] - theirs[1]) <= 1e-4 * theirs[1]
    assert theirs[1] > 0.1 and ours[2].keys() == theirs[2].keys()
    for n, a in ours[2].items():
        b = theirs[2][n]
        assert (a - b).abs().max() <= 1e-4 * b.abs().max().clamp_min(1e-30), n


def test_steps_follow_the_sequence():
    """prefill and step give the logits of the whole-sequence forward (fp32; the
    decode step and the scan agree to 1e-4)."""
    print("[case] lm steps", flush=True)
    m = _model(40, 2, 16, 4)
    g = torch.Generator().manual_seed(6)
    tokens = torch.randint(0, 40, (2, 12), generator=g).cuda()
    with torch.no_grad():
        want = m(tokens)
        m.stack.prepare_inference()
        logits, states = m.prefill(tokens[:, :5])
        for t in range(5, 12):
            assert (logits - want[:, t - 1]).abs().max() <= 1e-4 * want.abs().max()
            logits, states = m.step(tokens[:, t], states)
        assert (logits - want[:, 11]).abs().max() <= 1e-4 * want.abs().max()


@pytest.mark.parametrize("eos", [None, 2])
def test_beam_search_is_exact_with_enough_beams(eos):
    """With at least as many beams as hypotheses of the step before, beam search
    is exhaustive: the best continuations by the model's own whole-sequence
    logits, scored in float64."""
    print(f"[case] lm beam search eos={eos}", flush=True)
    V, steps, beams, T = 5, 3, 25, 4
    m = _model(V, 2, 16, 4, seed=3)
    prompt = torch.tensor([[1, 3, 0, 2], [4, 4, 1, 0]], device="cuda")
    ids, scores = lm.beam_search(m, prompt, beams, steps, eos_id=eos)
    tails = torch.tensor(list(itertools.product(range(V), repeat=steps)), device="cuda")
    for b in range(2):
        with torch.no_grad():
            logp = m(torch.cat((prompt[b].expand(len(tails), T), tails), 1)).double().log_softmax(-1).cpu()
        total = {}
        for row, tail in zip(logp, tails.tolist()):
            score, out = 0.0, []
            for k, t in enumerate(tail):
                ended = eos is not None and eos in out
                out.append(eos if ended else t)
                score += 0.0 if ended else float(row[T - 1 + k, t])
            total[tuple(out)] = score
        best = sorted(total.items(), key=lambda kv: -kv[1])[:beams]
        assert [tuple(r) for r in ids[b].tolist()] == [k for k, _ in best]
        assert max(abs(float(s) - v) for s, (_, v) in zip(scores[b], best)) <= 1e-3


def test_training_learns(capsys):
    print("[case] lm example", flush=True)
    lm.main(["--steps", "60", "--vocab", "32", "--d-model", "32"])
    out = [line for line in capsys.readouterr().out.splitlines() if line.startswith("step")]
    losses = [float(line.split("loss ")[1].split(",")[0]) for line in out]
    assert losses[-1] < 0.5 * losses[0]


def test_norm_kinds():
    with pytest.raises(ValueError, match="unknown norm"):
        stack.SPARCStack(1, 16, 4, norm="batch")
    s = stack.SPARCStack(1, 16, 4)
    assert isinstance(s.norm, torch.nn.RMSNorm) and isinstance(s.blocks[0].norm, torch.nn.RMSNorm)


def test_padding_counted_from_the_end():
    """padding_idx=-1 is the last id, for the lookup and for the targets."""
    print("[case] lm padding from the end", flush=True)
    tokens = torch.randint(0, 20, (3, 12), generator=torch.Generator().manual_seed(4))
    tokens[:, 8:] = 19
    tokens = tokens.cuda()
    results = []
    for pad in (19, -1):
        m = _model(20, 1, 16, 4, padding_idx=pad)
        loss, norm = lm.train_step(m, torch.optim.SGD(m.parameters(), lr=0.0), tokens, max_norm=1.0)
        results.append((float(loss), float(norm), [p.grad.clone() for p in m.parameters() if p.grad is not None]))
    assert results[0][:2] == results[1][:2]
    assert all(torch.equal(a, b) for a, b in zip(results[0][2], results[1][2]))


def test_ids_of_32_bits_train():
    print("[case] lm int32 ids", flush=True)
    tokens = torch.randint(0, 20, (2, 9), generator=torch.Generator().manual_seed(4)).cuda()
    losses = []
    for ids in (tokens, tokens.int()):
        m = _model(20, 1, 16, 4)
        losses.append(float(lm.train_step(m, torch.optim.SGD(m.parameters(), lr=0.0), ids, max_norm=1.0)[0]))
    assert losses[0] == losses[1]


@pytest.mark.parametrize("beams", [1, 3])
def test_beam_search_of_no_steps(beams):
    print(f"[case] lm beam search of no steps, {beams} beams", flush=True)
    m = _model(20, 1, 16, 4)
    ids, scores = lm.beam_search(m, torch.ones(2, 3, dtype=torch.int64, device="cuda"), beams, 0)
    assert ids.shape == (2, beams, 0) and ids.dtype == torch.int64 and ids.is_cuda
    assert scores.tolist() == [[0.0] + [-math.inf] * (beams - 1)] * 2


def test_steps_have_no_gradient():
    """The mixers' step has none, so what is around them has none either: the
    gradient of the projections alone would be a wrong one."""
    print("[case] lm steps and gradients", flush=True)
    m = _model(20, 2, 16, 4)
    tokens = torch.ones(2, 3, dtype=torch.int64, device="cuda")
    with torch.no_grad():
        _, states = m.prefill(tokens)
    x = torch.randn(2, 16, device="cuda", requires_grad=True)
    logits, new = m.step(tokens[:, 0], states)
    for out in (logits, m.stack.step(x, states)[0], m.stack.blocks[0].step(x, states[0])[0]):
        assert not out.requires_grad
    assert not any(p.requires_grad for s in new for p in s)


@pytest.mark.parametrize("kind", ["forward", "pre", "backward", "global", "subclass"])
def test_a_norm_is_called_with_its_hooks(kind):
    print(f"[case] layer norm module hooks {kind}", flush=True)
    seen = []
    norm = torch.nn.LayerNorm(16).cuda()
    x = torch.randn(3, 16, device="cuda", requires_grad=True)
    handle = None
    if kind == "forward":
        handle = norm.register_forward_hook(lambda mod, args, y: y + 1.0)
    elif kind == "pre":
        handle = norm.register_forward_pre_hook(lambda mod, args: (args[0] * torch.arange(16.0, device="cuda"),))
    elif kind == "backward":
        handle = norm.register_full_backward_hook(lambda mod, gx, gy: seen.append(gy))
    elif kind == "global":
        handle = torch.nn.modules.module.register_module_forward_hook(lambda mod, args, y: y + 1.0)
    else:
        class Centred(torch.nn.LayerNorm):
            def forward(self, x):
                return x - x.mean(-1, keepdim=True)
        norm = Centred(16).cuda()
    try:
        y, want = stack.apply_norm(norm, x), norm(x)
        y.sum().backward()
    finally:
        if handle is not None:
            handle.remove()
    torch.testing.assert_close(y, want, rtol=1e-5, atol=1e-5)
    assert len(seen) == (1 if kind == "backward" else 0)
