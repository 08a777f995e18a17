"""The operators of a linear attention block in captured graphs (replayed several times
with other inputs, eager work and synchronisations in between, every replay bit for
bit the eager call's results), on other streams, and where offsets pass 32 bits."""
import pytest
import torch

import sparc_amd
from oracle import block_oracle as O

pytestmark = pytest.mark.gpu
F32, BF16 = torch.float32, torch.bfloat16
IDS = dict(ids=lambda d: str(d).replace("torch.", ""))


def _replays(make_inputs, run):
    """run(inputs) -> tensors, captured on the first inputs; the others are copied into
    them.  Two graphs of the same calls are replayed in turn."""
    static = make_inputs(0)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        run(static)
    torch.cuda.current_stream().wait_stream(side)
    graphs, outs = [], []
    for _ in range(2):
        graphs.append(torch.cuda.CUDAGraph())
        with torch.cuda.graph(graphs[-1]):
            outs.append(run(static))
    for seed in (1, 2, 3, 1):
        fresh = make_inputs(seed)
        want = [t.clone() for t in run(make_inputs(seed))]
        with torch.no_grad():
            for s, f in zip(static, fresh):
                s.copy_(f)
        for graph in graphs:
            graph.replay()
        torch.cuda.synchronize()
        for out in outs:
            assert all(torch.equal(a, b) for a, b in zip(out, want)), seed


def _make(shapes, dtype, grads=0):
    def make(seed):
        g = torch.Generator(device="cuda").manual_seed(seed)
        t = [torch.randn(*s, device="cuda", generator=g).to(dtype) for s in shapes]
        return [x.requires_grad_() if n < grads else x for n, x in enumerate(t)]
    return make


@pytest.mark.parametrize("dtype", [F32, BF16], **IDS)
def test_rotary_graph(dtype):
    print(f"[case] rotary graph {dtype}", flush=True)
    table = sparc_amd.rotary_table(70, 32, device="cuda")

    def run(i):
        y = sparc_amd.qk_norm_rotary(*i[:4], table)
        return [*(t.detach() for t in y), *torch.autograd.grad(y, i[:4], i[4:])]

    _replays(_make([(3, 70, 4, 40), (3, 70, 2, 40), (40,), (40,), (3, 70, 4, 40), (3, 70, 2, 40)], dtype, 4), run)


@pytest.mark.parametrize("dtype", [F32, BF16], **IDS)
@pytest.mark.parametrize("T", [90, 700])  # one pass, and segments
def test_linear_attention_graph(T, dtype):
    print(f"[case] linear attention graph {T} {dtype}", flush=True)
    decay = torch.tensor([-0.01, -0.1, -0.3, -2.0], device="cuda")

    def run(i):
        o, s = sparc_amd.linear_attention(*i[:3], decay)
        return [o.detach(), s.detach(), *torch.autograd.grad(o, i[:3], i[3])]

    _replays(_make([(2, T, 4, 24), (2, T, 2, 24), (2, T, 2, 40), (2, T, 4, 40)], dtype, 3), run)


def test_step_graph():
    """In place: the state goes on from replay to replay."""
    print("[case] step graph", flush=True)
    make = _make([(3, 4, 24), (3, 2, 24), (3, 2, 40), (3, 4, 24, 40)], F32)
    decay = torch.tensor([-0.01, -0.1, -0.3, -2.0], device="cuda")

    def run(i):
        o, s = sparc_amd.linear_attention_step(*i[:3], decay, i[3], out_state=i[3])
        return [o, s]

    static = make(0)
    run(static)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = run(static)
    eager = make(5)
    for s, f in zip(static, make(5)):
        s.copy_(f)
    for _ in range(3):
        graph.replay()
        want = run(eager)
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(out, want))


@pytest.mark.parametrize("dtype", [F32, BF16], **IDS)
def test_gated_graph(dtype):
    print(f"[case] gated graph {dtype}", flush=True)

    def run(i):
        y = sparc_amd.gated_linear_unit(*i[:3])
        return [y.detach(), *torch.autograd.grad(y, i[:3], i[3])]

    # all products split over workgroups, with sums behind them
    _replays(_make([(2000, 96), (400, 96), (400, 96), (2000, 400)], dtype, 3), run)


def test_on_another_stream():
    """Calls and gradients on a stream that is not the default one, beside work on it."""
    print("[case] another stream", flush=True)
    make = _make([(2, 300, 4, 32), (2, 300, 2, 32), (2, 300, 2, 32), (2, 300, 4, 32)], BF16, 3)
    decay = torch.tensor([-0.01, -0.1, -0.3, -2.0], device="cuda")
    w = torch.randn(2, 64, 32, device="cuda").to(BF16)
    table = sparc_amd.rotary_table(300, 32, device="cuda")

    def run(i):
        q, k = sparc_amd.qk_norm_rotary(i[0], i[1], None, None, table)
        o, _ = sparc_amd.linear_attention(q, k, i[2], decay)
        y = sparc_amd.gated_linear_unit(o, w[0], w[1])
        return [y.detach(), *torch.autograd.grad(y, i[:3], y.detach())]

    want = run(make(3))
    torch.cuda.synchronize()
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        inputs = make(3)
        torch.cuda._sleep(10_000_000)  # what comes before on this stream
        for t in inputs[:3]:
            t.detach().mul_(2.0).mul_(0.5)
        got = run(inputs)
    busy = torch.zeros(1 << 26, device="cuda").add_(1.0)
    side.synchronize()
    assert all(torch.equal(a, b) for a, b in zip(got, want)) and busy.sum() == 1 << 26


def test_linear_attention_beyond_32_bits():
    """2^31 and more elements of each operand: the last chain's rows lie behind them."""
    B, T, H, D = 33, 4096, 128, 128
    print(f"[case] linear attention {B} x {T} x {H} x {D}", flush=True)
    q = torch.zeros(B, T, H, D, dtype=BF16, device="cuda")
    decay = torch.full((H,), -0.05, device="cuda")
    g = torch.Generator().manual_seed(1)
    qs, ks, vs, ds = (torch.randn(1, T, 1, D, generator=g).to(BF16) for _ in range(4))
    k, v = torch.zeros_like(q), torch.zeros_like(q)
    for t, x in ((q, qs), (k, ks), (v, vs)):
        t[-1:, :, -1:] = x.cuda()
    assert q.numel() >= 1 << 31
    do = torch.zeros_like(q)
    do[-1:, :, -1:] = ds.cuda()
    leaves = [t.requires_grad_() for t in (q, k, v)]
    o, s = sparc_amd.linear_attention(*leaves, decay)
    grads = torch.autograd.grad(o, leaves, do)
    alone = [t.cuda().requires_grad_() for t in (qs, ks, vs)]
    o1, s1 = sparc_amd.linear_attention(*alone, decay[-1:])
    want = torch.autograd.grad(o1, alone, ds.cuda())
    # one chain's sums are the same but for the number of segments: fp32 sums of the same
    # terms in another order, and one rounding to bf16 on either side
    for x, y in ((o, o1), *zip(grads, want)):
        far = (x[-1:, :, -1:].detach().float() - y.detach().float()).abs()
        assert (far <= 2.0 ** -7 * y.detach().float().abs() + 2.0 ** -11 * y.detach().float().abs().max()).all()
        assert not x[:-1].any() and not x[-1, :, :-1].any()
    assert (s[-1, -1] - s1[0, 0]).abs().max() <= 2.0 ** -16 * s1.abs().max()


def test_rotary_beyond_32_bits():
    B, T, H, D = 66, 2048, 128, 128
    print(f"[case] rotary {B} x {T} x {H} x {D}", flush=True)
    q = torch.zeros(B, T, H, D, dtype=BF16, device="cuda")
    g = torch.Generator().manual_seed(1)
    row = torch.randn(1, T, 1, D, generator=g).to(BF16)
    q[-1:, :, -1:] = row.cuda()
    assert q.numel() >= 1 << 31
    table = O.rotary_table(T, D).float()
    y, _ = sparc_amd.qk_norm_rotary(q, q[:, :, :1], None, None, table.cuda())
    want = O.norm_rotary(row, None, table, torch.arange(T)[None], False, 1e-6)
    got = y[-1:, :, -1:].cpu().double()
    assert ((got - want).abs() <= 2.0 ** -8 * want.abs() + 2.0 ** -16 * want.abs().amax(-1, keepdim=True)).all()
    assert not y[:-1].any() and not y[-1, :, :-1].any()


def test_gated_beyond_32_bits():
    """2^31 and more outputs: rows at both ends and around the border."""
    N, D, F = 530_000, 8, 4096
    print(f"[case] gated {N} x {D} x {F}", flush=True)
    g = torch.Generator().manual_seed(1)
    x = torch.randn(N, D, generator=g).to(BF16)
    wg, wu = (torch.randn(F, D, generator=g).to(BF16) for _ in range(2))
    y = sparc_amd.gated_linear_unit(x.cuda(), wg.cuda(), wu.cuda())
    assert y.numel() >= 1 << 31
    at = [0, 1, (1 << 31) // F - 1, (1 << 31) // F, (1 << 31) // F + 1, N - 1]
    want = O.gated_linear_unit(x[at], wg, wu, "silu")
    # activation 2^-20, projections of 8 terms
    size = (x[at].double().abs() @ wg.double().abs().T) * (x[at].double().abs() @ wu.double().abs().T)
    assert ((y[at].cpu().double() - want).abs() <= 2.0 ** -8 * want.abs() + 2.0 ** -18 * size).all()
