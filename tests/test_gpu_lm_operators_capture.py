"""The operators around the stack in captured graphs: replayed several times
with other inputs, eager work and synchronisations in between, every replay bit
for bit the eager call's results; and the layer norm's and the embedding's
refusal of a second differentiation."""
import pytest
import torch

import sparc_amd

pytestmark = pytest.mark.gpu


def _replays(make_inputs, run):
    """run(inputs) -> tensors, captured on the first inputs; the others are
    copied into them."""
    static = make_inputs(0)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        run(static)
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = run(static)
    for seed in (1, 2, 3, 1):
        fresh = make_inputs(seed)
        want = [t.clone() for t in run(make_inputs(seed))]
        with torch.no_grad():
            for s, f in zip(static, fresh):
                s.copy_(f)
        graph.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(out, want)), seed


def _gen(seed):
    return torch.Generator(device="cuda").manual_seed(seed)


def test_layer_norm_graph():
    print("[case] layer norm graph", flush=True)

    def make(seed):
        g = _gen(seed)
        r = lambda *s: torch.randn(*s, device="cuda", generator=g)  # noqa: E731
        return [r(1500, 200).requires_grad_(), r(200).requires_grad_(), r(200).requires_grad_(), r(1500, 200)]

    def run(i):
        y = sparc_amd.layer_norm(*i[:3])
        return [y.detach(), *torch.autograd.grad(y, i[:3], i[3])]

    _replays(make, run)


@pytest.mark.parametrize("n", [900, 9000])
def test_embedding_graph(n):
    print(f"[case] embedding graph n={n}", flush=True)

    def make(seed):
        g = _gen(seed)
        return [torch.randint(0, 500, (n,), device="cuda", generator=g),
                torch.randn(500, 72, device="cuda", generator=g).requires_grad_(),
                torch.randn(n, 72, device="cuda", generator=g)]

    def run(i):
        y = sparc_amd.embedding(i[0], i[1], scale=2.0)
        return [y.detach(), *torch.autograd.grad(y, [i[1]], i[2])]

    _replays(make, run)


def test_beam_graph():
    print("[case] beam graph", flush=True)

    def make(seed):
        g = _gen(seed)
        r = lambda *s: torch.randn(*s, device="cuda", generator=g)  # noqa: E731
        return [r(3, 4, 5000), -r(3, 4).abs(), r(3, 4) > 1.0, *[r(12, 333) for _ in range(4)]]

    def run(i):
        step = sparc_amd.beam_search_step(i[0], i[1], finished=i[2], eos_id=7,
                                          states=[(i[3], i[4]), (i[5], i[6])])
        return [step.tokens, step.parents, step.scores, step.finished, *[p for s in step.states for p in s]]

    _replays(make, run)


def test_second_differentiation_is_refused():
    print("[case] second differentiation", flush=True)
    x = torch.randn(4, 8, device="cuda", requires_grad=True)
    with pytest.raises(RuntimeError, match="twice differentiable"):
        torch.autograd.grad(sparc_amd.layer_norm(x).square().sum(), x, create_graph=True)
    ids = torch.zeros(3, dtype=torch.int64, device="cuda")
    with pytest.raises(RuntimeError, match="twice differentiable"):
        torch.autograd.grad(sparc_amd.embedding(ids, x).square().sum(), x, create_graph=True)


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16], ids=["f32", "bf16"])
def test_embedding_of_few_ids_graph(dtype):
    print(f"[case] embedding graph n=100 {dtype}", flush=True)

    def make(seed):
        g = _gen(seed)
        return [torch.randint(0, 500, (100,), device="cuda", generator=g),
                torch.randn(500, 700, device="cuda", generator=g).to(dtype).requires_grad_(),
                torch.randn(100, 700, device="cuda", generator=g).to(dtype)]

    def run(i):
        y = sparc_amd.embedding(i[0], i[1], scale=2.0)
        return [y.detach(), *torch.autograd.grad(y, [i[1]], i[2])]

    _replays(make, run)


def test_states_in_place_graph():
    """The beam step with its states reordered in place, many rows and few."""
    print("[case] states in place graph", flush=True)
    for B, width in ((3, 333), (300, 1028)):
        def make(seed):
            g = _gen(seed)
            r = lambda *s: torch.randn(*s, device="cuda", generator=g)  # noqa: E731
            return [r(B, 4, 500), -r(B, 4).abs(), *[r(4 * B, width) for _ in range(4)]]

        def run(i):
            states = [(i[2], i[3]), (i[4], i[5])]
            step = sparc_amd.beam_search_step(i[0], i[1], states=states, out_states=states)
            return [step.tokens, step.parents, step.scores, *i[2:]]

        _replays(make, run)
