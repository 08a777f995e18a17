"""linear_attention and linear_attention_step against the recurrence in 64 bits.

Tolerances.  All results are sums of products with factors that are not negative
(powers of the decay, the scale), so the same call on absolute values gives A, the
sum of the terms' sizes.  A chain of n roundings of fp32 is off by n 2^-24 A at most;
here n counts a dot product over the head (K or V), the steps that a value passes
(T), and 64 for the powers and the rest.  With bfloat16 inputs the state, the scores
and decayed values enter products as two or three bfloat16 values, truncated to 2^-15
of each or better, two of them for a term at most: another 2^-14 A.  A result in bfloat16 is rounded once: 2^-8 of its value."""
import pytest
import torch

import sparc_amd
from oracle import block_oracle as O

pytestmark = pytest.mark.gpu
F32, BF16 = torch.float32, torch.bfloat16
IDS = dict(ids=lambda d: str(d).replace("torch.", ""))


def _case(B, T, H, G, K, V, dtype, seed, state=False, lengths=None, layout="plain", decay=None):
    g = torch.Generator().manual_seed(seed)
    r = lambda *s: torch.randn(*s, generator=g)
    if layout == "fused":  # parts of one projection
        both = r(B, T, H * K + G * K + G * V).to(dtype)
        q, k, v = (x.unflatten(-1, (n, -1)) for x, n in zip(both.split([H * K, G * K, G * V], -1), (H, G, G)))
    elif layout == "heads first":
        q, k, v = (r(B, n, T, d).to(dtype).transpose(1, 2) for n, d in ((H, K), (G, K), (G, V)))
    else:
        q, k, v = (r(B, T, n, d).to(dtype) for n, d in ((H, K), (G, K), (G, V)))
    if decay is None:
        decay = torch.log1p(-torch.exp2(-1.0 - 8.0 * torch.rand(H, generator=g)))
    s = dict(q=q, k=k, v=v, log_decay=decay)
    if state:
        s["state"] = r(B, H, K, V)
    if lengths is not None:
        s["lengths"] = torch.tensor(lengths)
    return s, r(B, T, H, V).to(dtype), r(B, H, K, V)


def _on_gpu(x):
    """The tensor on the GPU with its strides."""
    if not isinstance(x, torch.Tensor):
        return x
    y = torch.empty_strided(x.shape, x.stride(), dtype=x.dtype, device="cuda")
    return y.copy_(x)


def _all(call, s, do, ds, with_state):
    """Outputs and gradients of a call on copies of the inputs."""
    if call is O.linear_attention:  # leaves in 64 bits, and so their gradients
        s = {n: x.double() if isinstance(x, torch.Tensor) and x.is_floating_point() else x for n, x in s.items()}
    s = {n: x.detach().requires_grad_(n in ("q", "k", "v", "state")) if isinstance(x, torch.Tensor) and
         x.is_floating_point() else x for n, x in s.items()}
    o, after = call(**s)
    names = [n for n in ("q", "k", "v", "state") if n in s]
    outs, grads = ((o, after), (do.to(o.dtype), ds)) if with_state else ((o,), (do.to(o.dtype),))
    got = torch.autograd.grad(outs, [s[n] for n in names], grads)
    return {"o": o.detach(), "after": after.detach(), **dict(zip(names, got))}


def _check(got, want, size, n, bf16):
    for name, x in got.items():
        x, y, a = x.cpu().double(), want[name].double(), size[name].double()
        tol = (n * 2.0 ** -24 + (2.0 ** -14 if bf16 else 0.0)) * a
        if name in ("after", "state"):
            tol = (n * 2.0 ** -24) * a
        elif bf16:
            tol = tol + 2.0 ** -8 * y.abs()
        off = ((x - y).abs() - tol).max().item() if x.numel() else -1.0
        assert off <= 0.0, f"{name}: {off} over a tolerance of up to {tol.max().item()}"


def _run(s, do, ds, dtype, with_state=True):
    want = _all(O.linear_attention, s, do.double(), ds.double(), with_state)
    size = {n: x.abs() if isinstance(x, torch.Tensor) and x.is_floating_point() and n != "log_decay" else x
            for n, x in s.items()}
    size = _all(O.linear_attention, size, do.double().abs(), ds.double().abs(), with_state)
    g = {n: _on_gpu(x) for n, x in s.items()}
    got = _all(sparc_amd.linear_attention, g, do.cuda(), ds.cuda(), with_state)
    B, T, H, K = s["q"].shape
    assert got["o"].dtype == dtype and got["after"].dtype == F32 and got["q"].dtype == dtype
    _check(got, want, size, T + max(K, s["v"].shape[-1]) * (H // s["k"].shape[2]) + 64, dtype == BF16)


SHAPES = [  # B, T, H, G, K, V
    (1, 1, 1, 1, 1, 1), (2, 3, 2, 1, 5, 7), (1, 16, 1, 1, 16, 16), (2, 63, 3, 3, 31, 33), (1, 64, 2, 2, 64, 64),
    (1, 65, 4, 2, 64, 64), (2, 130, 2, 2, 128, 128), (1, 97, 6, 2, 40, 72), (1, 200, 2, 1, 65, 129),
    (1, 70, 1, 1, 200, 60), (1, 70, 1, 1, 60, 200), (1, 129, 1, 1, 256, 256), (3, 33, 2, 2, 96, 8),
]


@pytest.mark.parametrize("dtype", [F32, BF16], **IDS)
@pytest.mark.parametrize("shape", SHAPES, ids=str)
def test_against_the_recurrence(shape, dtype):
    print(f"[case] linear attention {shape} {dtype}", flush=True)
    s, do, ds = _case(*shape, dtype, seed=sum(shape), state=True)
    _run(s, do, ds, dtype)


@pytest.mark.parametrize("dtype", [F32, BF16], **IDS)
@pytest.mark.parametrize("K,V", [(32, 128), (64, 72), (64, 128), (128, 128), (100, 128)])
def test_many_chains(K, V, dtype):
    """More workgroups than CUs."""
    s, do, ds = _case(33, 70, 8, 8, K, V, dtype, seed=K + V, state=True)
    _run(s, do, ds, dtype)


@pytest.mark.parametrize("dtype", [F32, BF16], **IDS)
@pytest.mark.parametrize("T", [257, 1000])
def test_long_enough_for_segments(T, dtype):
    """Few chains over many chunks are cut into segments, with a ragged end."""
    print(f"[case] segments {T} {dtype}", flush=True)
    s, do, ds = _case(2, T, 2, 1, 24, 40, dtype, seed=T, state=True, lengths=[T - 130, T])
    _run(s, do, ds, dtype)


@pytest.mark.parametrize("dtype", [F32, BF16], **IDS)
@pytest.mark.parametrize("layout", ["fused", "heads first"])
def test_strides(layout, dtype):
    s, do, ds = _case(2, 90, 4, 2, 20, 24, dtype, seed=3, layout=layout)
    _run(s, do, ds, dtype, with_state=False)


@pytest.mark.parametrize("dtype", [F32, BF16], **IDS)
@pytest.mark.parametrize("stride", [(1 << 22) - 1, 1 << 22, (1 << 23) + 8])
def test_steps_that_lie_far_apart(stride, dtype):
    """At the largest stride that is read in place and behind it: the plain call's bits."""
    T, K, V = 70, 30, 24
    s, do, _ = _case(1, T, 2, 1, K, V, dtype, seed=stride)
    s = {n: x.cuda() for n, x in s.items()}
    far = dict(s)
    for n in ("q", "k", "v"):
        h, d = s[n].shape[2:]
        far[n] = torch.full((stride * (T - 1) + h * d,), float("nan"), dtype=dtype, device="cuda").as_strided(
            (1, T, h, d), (stride * T, stride, d, 1)).copy_(s[n])
    got, want = (_all(sparc_amd.linear_attention, x, do.cuda(), None, False) for x in (far, s))
    assert all(torch.equal(got[n], want[n]) for n in want)


@pytest.mark.parametrize("dtype", [F32, BF16], **IDS)
@pytest.mark.parametrize("state", [False, True])
def test_lengths(state, dtype):
    lengths = [0, 1, 64, 65, 100, 1000, -3]
    s, do, ds = _case(len(lengths), 100, 2, 2, 32, 32, dtype, seed=9, state=state, lengths=lengths)
    want = dict(s, lengths=s["lengths"].clamp(0, 100))
    print("[case] lengths", flush=True)
    g = {n: _on_gpu(x) for n, x in s.items()}
    _run(want, do, ds, dtype, with_state=state)
    o, after = sparc_amd.linear_attention(**g)
    o2, after2 = sparc_amd.linear_attention(**{n: _on_gpu(x) for n, x in want.items()})
    assert torch.equal(o, o2) and torch.equal(after, after2)
    o3, _ = sparc_amd.linear_attention(**dict(g, lengths=g["lengths"].int()))
    assert torch.equal(o, o3)


@pytest.mark.parametrize("dtype", [F32, BF16], **IDS)
def test_what_lies_behind_a_length_is_not_read(dtype):
    s, do, _ = _case(2, 80, 2, 2, 32, 32, dtype, seed=10, lengths=[17, 70])
    bad = {n: _on_gpu(x.clone()) for n, x in s.items()}
    do_bad = do.clone()
    for b, n in enumerate((17, 70)):
        for name in ("q", "k", "v"):
            bad[name][b, n:] = float("nan")
        do_bad[b, n:] = float("inf")
    good = {n: _on_gpu(x) for n, x in s.items()}
    outs = []
    for g, d in ((good, do), (bad, do_bad)):
        leaves = [g[n].requires_grad_() for n in ("q", "k", "v")]
        o, after = sparc_amd.linear_attention(**g)
        outs.append([o, after, *torch.autograd.grad(o, leaves, d.cuda())])
    for x, y in zip(*outs):
        assert torch.equal(x, y)
    for x in (outs[1][0], *outs[1][2:]):
        assert not x[0, 17:].any() and not x[1, 70:].any()


@pytest.mark.parametrize("dtype", [F32, BF16], **IDS)
def test_decays_of_one_and_of_nothing(dtype):
    s, do, ds = _case(1, 150, 3, 3, 16, 16, dtype, seed=11, state=True,
                      decay=torch.tensor([0.0, -float("inf"), -40.0]))
    _run(s, do, ds, dtype)


@pytest.mark.parametrize("bad", [float("nan"), float("inf")])
@pytest.mark.parametrize("name", ["k", "v"])
@pytest.mark.parametrize("dtype", [F32, BF16], **IDS)
def test_a_value_that_is_not_finite_reaches_no_earlier_step(dtype, name, bad):
    s, _, _ = _case(1, 150, 2, 2, 32, 32, dtype, seed=12)
    g = {n: _on_gpu(x) for n, x in s.items()}
    o, _ = sparc_amd.linear_attention(**g)
    g[name] = g[name].clone()
    g[name][0, 75, 1, 3] = bad
    o2, _ = sparc_amd.linear_attention(**g)
    assert torch.equal(o[:, :, 0], o2[:, :, 0])
    # the steps before it in its block are summed in another order: both sums are off
    # by (T + K + 64) 2^-24 A at most, and a result in bfloat16 by 2^-8 of its value
    size = O.linear_attention(s["q"].abs(), s["k"].abs(), s["v"].abs(), s["log_decay"])[0][:, :75]
    x, y = o[:, :75].cpu().double(), o2[:, :75].cpu().double()
    tol = 2 * (150 + 32 + 64) * 2.0 ** -24 * size
    if dtype == BF16:
        tol = tol + 2 * (2.0 ** -14 * size + 2.0 ** -8 * x.abs().maximum(y.abs()))
    assert ((x - y).abs() <= tol).all()
    assert not torch.isfinite(o2[0, 75:, 1]).all()


def test_equal_calls_give_equal_bits():
    s, do, ds = _case(2, 500, 4, 2, 64, 64, BF16, seed=13, state=True)
    g = {n: _on_gpu(x) for n, x in s.items()}
    first, second = (_all(sparc_amd.linear_attention, g, do.cuda(), ds.cuda(), True) for _ in range(2))
    assert all(torch.equal(first[n], second[n]) for n in first)


def test_a_sequence_in_pieces_is_the_sequence():
    """The state carries a sequence from call to call, and from call to step."""
    s, _, _ = _case(2, 100, 4, 2, 48, 40, F32, seed=14)
    g = {n: _on_gpu(x) for n, x in s.items()}
    o, after = sparc_amd.linear_attention(**g)
    state, parts = None, []
    for t0, t1 in ((0, 1), (1, 64), (64, 99)):
        piece = {n: x[:, t0:t1] if n in ("q", "k", "v") else x for n, x in g.items()}
        y, state = sparc_amd.linear_attention(**piece, state=state)
        parts.append(y)
    y, state = sparc_amd.linear_attention_step(*(g[n][:, 99] for n in ("q", "k", "v")), g["log_decay"], state)
    size, size_after = O.linear_attention(s["q"].abs(), s["k"].abs(), s["v"].abs(), s["log_decay"])
    tol = 2 * (100 + 48 + 64) * 2.0 ** -24
    assert ((torch.cat((*parts, y[:, None]), 1) - o).cpu().abs() <= tol * size).all()
    assert ((state - after).cpu().abs() <= tol * size_after).all()


@pytest.mark.parametrize("dtype", [F32, BF16], **IDS)
@pytest.mark.parametrize("shape", [(1, 1, 1, 1, 1), (1, 16, 16, 128, 128), (3, 6, 2, 40, 72), (2, 2, 1, 255, 3),
                                   (5, 4, 4, 64, 256), (70, 16, 16, 64, 64)], ids=str)
def test_step(shape, dtype):
    B, H, G, K, V = shape
    print(f"[case] step {shape} {dtype}", flush=True)
    s, _, _ = _case(B, 1, H, G, K, V, dtype, seed=sum(shape), state=True)
    want, after = O.linear_attention(**s)
    size, size_after = O.linear_attention(s["q"].abs(), s["k"].abs(), s["v"].abs(), s["log_decay"], s["state"].abs())
    one = [_on_gpu(s[n])[:, 0] for n in ("q", "k", "v")]
    state, decay = s["state"].cuda(), s["log_decay"].cuda()
    o, new = sparc_amd.linear_attention_step(*one, decay, state)
    assert torch.equal(state.cpu(), s["state"])
    tol = (K + 16) * 2.0 ** -24 * size + (2.0 ** -8 * want.abs() if dtype == BF16 else 0.0)
    assert o.dtype == dtype and ((o[:, None].cpu().double() - want).abs() <= tol).all()
    assert ((new.cpu().double() - after).abs() <= 8 * 2.0 ** -24 * size_after).all()
    version = state._version
    o2, same = sparc_amd.linear_attention_step(*one, decay, state, out_state=state)
    assert same.data_ptr() == state.data_ptr() and torch.equal(state, new) and torch.equal(o, o2)
    assert state._version > version


def test_step_refuses_overlapping_memory():
    s, _, _ = _case(2, 1, 2, 2, 8, 8, F32, seed=1, state=True)
    one = [_on_gpu(s[n])[:, 0] for n in ("q", "k", "v")]
    decay, buffer = s["log_decay"].cuda(), torch.zeros(3, 2, 8, 8, device="cuda")
    with pytest.raises(ValueError, match="overlaps the state"):
        sparc_amd.linear_attention_step(*one, decay, buffer[:2], out_state=buffer[1:])
    q = buffer.flatten()[:32].view(2, 2, 8)
    with pytest.raises(ValueError, match="overlaps an input"):
        sparc_amd.linear_attention_step(q, *one[1:], decay, s["state"].cuda(), out_state=buffer[:2])


def test_empty_calls():
    s, do, ds = _case(2, 0, 2, 2, 8, 8, F32, seed=2, state=True)
    g = {n: _on_gpu(x) for n, x in s.items()}
    got = _all(sparc_amd.linear_attention, g, do.cuda(), ds.cuda(), True)
    assert got["o"].shape == (2, 0, 2, 8) and torch.equal(got["after"].cpu(), s["state"])
    assert torch.equal(got["state"].cpu(), ds)
    o, after = sparc_amd.linear_attention(*(g[n][:0] for n in ("q", "k", "v")), g["log_decay"])
    assert o.shape == (0, 0, 2, 8) and after.shape == (0, 2, 8, 8)


def test_gradients_are_the_differences():
    """Central differences of a call in fp32: o and the state are linear in each
    input, so a step of 1 has no error but rounding's."""
    s, do, ds = _case(1, 70, 2, 1, 6, 5, F32, seed=21, state=True)
    g = {n: _on_gpu(x) for n, x in s.items()}
    got = _all(sparc_amd.linear_attention, g, do.cuda(), ds.cuda(), True)
    loss = lambda x: sum((y.double() * w.cuda().double()).sum() for y, w in zip(sparc_amd.linear_attention(**x), (do, ds)))
    size = _all(O.linear_attention, {n: x if n == "log_decay" else x.abs() for n, x in s.items()}, do.double().abs(),
                ds.double().abs(), True)
    total = (size["o"] * do.double().abs()).sum() + (size["after"] * ds.double().abs()).sum()
    for name in ("q", "k", "v", "state"):
        d = torch.randn(s[name].shape, generator=torch.Generator().manual_seed(5))
        up, down = (dict(g, **{name: g[name] + m * d.cuda()}) for m in (1.0, -1.0))
        diff = (loss(up) - loss(down)).item() / 2
        # the moved inputs are up to a few times larger: 8 times the terms' sizes
        assert abs(diff - (got[name].double().cpu() * d.double()).sum().item()) <= 8 * (70 + 70) * 2.0 ** -24 * total


def test_no_backward_where_there_is_none():
    s, do, _ = _case(1, 5, 2, 2, 8, 8, F32, seed=4, state=True)
    g = {n: _on_gpu(x) for n, x in s.items()}
    one = [g[n][:, 0].requires_grad_() for n in ("q", "k", "v")]
    with pytest.raises(RuntimeError, match="no backward"):
        sparc_amd.linear_attention_step(*one, g["log_decay"], g["state"])
    with pytest.raises(RuntimeError, match="no backward"):
        sparc_amd.linear_attention(g["q"], g["k"], g["v"], g["log_decay"].clone().requires_grad_())
    q = g["q"].requires_grad_()
    o, _ = sparc_amd.linear_attention(q, g["k"], g["v"], g["log_decay"])
    with pytest.raises(RuntimeError, match="not twice"):
        torch.autograd.grad(o, q, do.cuda(), create_graph=True)
    o, _ = sparc_amd.linear_attention(q, g["k"], g["v"], g["log_decay"])
    g["k"].add_(1.0)
    with pytest.raises(RuntimeError, match="modified by an inplace"):
        o.sum().backward()
