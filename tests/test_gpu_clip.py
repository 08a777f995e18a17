"""grad_norm and clip_grad_norm_ on the GPU against float64: mixed types, odd
sizes and alignments, many tensors, values that are not finite.

Tolerances: squares are summed in fp64 and the norm is rounded once (2^-24; 4
of them allowed); a scaled value is one fp32 product with a factor that is off
by at most 2^-22, rounded once more in bf16 (2^-8)."""
import math
import random

import pytest
import torch

import sparc_amd
from oracle import lm_oracle as L

pytestmark = pytest.mark.gpu

F32, BF16 = torch.float32, torch.bfloat16


def _params(shapes, dtypes, seed, scale=0.02):
    g = torch.Generator().manual_seed(seed)
    params = []
    for shape, dtype in zip(shapes, dtypes):
        p = torch.nn.Parameter(torch.zeros(shape, dtype=dtype, device="cuda"))
        p.grad = (scale * torch.randn(shape, generator=g)).to(dtype).cuda()
        params.append(p)
    return params


def _check(params, max_norm):
    before = [p.grad.detach().cpu().clone() for p in params]
    norm = sparc_amd.clip_grad_norm_(params, max_norm)
    want = L.grad_norm(before)
    assert norm.shape == () and norm.dtype == F32
    assert abs(float(norm) - want) <= 2.0 ** -22 * want
    factor = L.clip_factor(before, max_norm)
    for p, g in zip(params, before):
        if factor == 1.0:
            assert torch.equal(p.grad.cpu(), g)
            continue
        ref = g.double() * factor
        off = (p.grad.cpu().double() - ref).abs()
        assert (off <= ref.abs() * (2.0 ** -21 + (2.0 ** -8 if g.dtype == BF16 else 0.0)) + 1e-45).all()


@pytest.mark.parametrize("clips", [True, False])
@pytest.mark.parametrize("sizes", [[(1,)], [(7,), (1, 3)], [(2049,), (64, 24)], [(16384,), (16385,), (16383,)],
                                   [(300, 500), (3,), (1000, 17)]])
def test_sizes(sizes, clips):
    print(f"[case] clip {sizes} {clips}", flush=True)
    for dtypes in ([F32] * len(sizes), [BF16] * len(sizes), [BF16 if i % 2 else F32 for i in range(len(sizes))]):
        params = _params(sizes, dtypes, len(sizes))
        n = sum(math.prod(s) for s in sizes)
        _check(params, (0.3 if clips else 100.0) * 0.02 * math.sqrt(n) + (0.0 if clips else 1.0))


@pytest.mark.parametrize("count", [128, 129, 300])
def test_many_tensors(count):
    """More tensors than one launch takes; some without values."""
    print(f"[case] clip {count} tensors", flush=True)
    shapes = [(i % 37 * 11,) for i in range(count)]
    _check(_params(shapes, [BF16 if i % 3 else F32 for i in range(count)], count), 0.1)


def test_alignment_and_order():
    """Views that begin off a 16-byte boundary, transposed gradients, and
    gradients with gaps between their rows."""
    print("[case] clip layouts", flush=True)
    params = _params([(40, 30), (33, 65), (50, 20), (20, 9)], [BF16, F32, F32, BF16], 5)
    flat = torch.randn(5000, device="cuda").mul_(0.02)
    params[0].grad = flat.bfloat16()[3:1203].view(40, 30)
    params[1].grad = flat[1:2146].view(33, 65)
    params[2].grad = flat[3000:4000].view(20, 50).t()
    wide = flat[:400].bfloat16().view(20, 20)
    params[3].grad = wide[:, 2:11]
    rest = wide.clone()
    rest[:, 2:11] = 0
    _check(params, 0.2)
    wide[:, 2:11] = 0
    assert torch.equal(wide, rest)  # what lies between is not touched


def test_a_gradient_given_twice_counts_once():
    print("[case] clip twice", flush=True)
    params = _params([(700,)], [F32], 6)
    g = params[0].grad.clone()
    norm = sparc_amd.clip_grad_norm_([params[0], params[0]], 0.1)
    assert abs(float(norm) - L.grad_norm([g.cpu()])) <= 1e-6
    assert ((params[0].grad - g * (0.1 / float(norm))).abs() <= 1e-6 * g.abs() + 1e-12).all()


def test_gradients_that_overlap_are_refused():
    """Two workgroups would scale the shared values at once."""
    print("[case] clip overlap", flush=True)
    params = _params([(40,), (20,), (30,)], [F32] * 3, 11)
    flat = torch.ones(100, device="cuda")
    for a, b, c in ((flat[:40], flat[30:50], flat[60:90]), (flat[60:100], flat[:20], flat[40:70]),
                    (flat[:40], flat[:20], flat[50:80])):
        for p, g in zip(params, (a, b, c)):
            p.grad = g
        with pytest.raises(RuntimeError, match="overlap"):
            sparc_amd.clip_grad_norm_(params, 0.5)
        assert abs(float(sparc_amd.grad_norm([a, b, c])) - math.sqrt(90.0)) <= 1e-5
    assert torch.equal(flat, torch.ones_like(flat))
    for p, g in zip(params, (flat[40:80], flat[20:40], None)):  # side by side, in any order
        p.grad = g
    sparc_amd.clip_grad_norm_(params, 0.5)
    assert flat[80:].eq(1.0).all() and flat[:20].eq(1.0).all() and flat[20:80].lt(1.0).all()


@pytest.mark.parametrize("scale", [1e-30, 1e30])
def test_squares_neither_vanish_nor_overflow(scale):
    print(f"[case] clip scale {scale}", flush=True)
    params = _params([(3000,), (17,)], [F32, BF16], 7, scale)
    want = L.grad_norm([p.grad.cpu() for p in params])
    assert abs(float(sparc_amd.grad_norm([p.grad for p in params])) - want) <= 2.0 ** -22 * want


def test_values_that_are_not_finite():
    """As torch: NaN goes into every gradient; infinity scales by 0."""
    print("[case] clip NaN and infinity", flush=True)
    params = _params([(100,), (9,)], [F32, BF16], 8)
    params[1].grad[3] = math.nan
    assert math.isnan(float(sparc_amd.clip_grad_norm_(params, 1.0)))
    assert all(p.grad.isnan().all() for p in params)
    params = _params([(100,), (9,)], [F32, BF16], 8)
    params[0].grad[3] = -math.inf
    assert float(sparc_amd.clip_grad_norm_(params, 1.0)) == math.inf
    assert params[0].grad.isnan().sum() == 1 and params[0].grad.nan_to_num().abs().max() == 0
    assert not params[1].grad.any()


def test_norm_zero_and_max_norm_zero():
    print("[case] clip zero", flush=True)
    p, = _params([(50,)], [F32], 9, 0.0)
    assert float(sparc_amd.clip_grad_norm_([p], 1.0)) == 0.0 and not p.grad.any()
    p, = _params([(50,)], [F32], 9)
    sparc_amd.clip_grad_norm_([p], 0.0)
    assert not p.grad.any()


def test_matches_torch_and_replays_in_a_graph():
    """The same values as torch.nn.utils.clip_grad_norm_ up to fp32 rounding, and
    in a captured graph, replayed with eager work in between."""
    print("[case] clip graph", flush=True)
    mine, theirs = _params([(1000, 30), (77,)], [F32, F32], 10), _params([(1000, 30), (77,)], [F32, F32], 10)
    a, b = sparc_amd.clip_grad_norm_(mine, 0.5), torch.nn.utils.clip_grad_norm_(theirs, 0.5)
    torch.testing.assert_close(a, b, rtol=1e-6, atol=0)
    for p, q in zip(mine, theirs):
        torch.testing.assert_close(p.grad, q.grad, rtol=1e-6, atol=0)
    start = [p.grad.clone() for p in mine]
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        sparc_amd.clip_grad_norm_(mine, 0.25)
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        norm = sparc_amd.clip_grad_norm_(mine, 0.25)
    for k in range(3):
        for p, s in zip(mine, start):
            p.grad.copy_(s * (k + 1))
        eager = [torch.nn.Parameter(torch.zeros_like(s)) for s in start]
        for p, s in zip(eager, start):
            p.grad = s * (k + 1)
        graph.replay()
        want = sparc_amd.clip_grad_norm_(eager, 0.25)
        torch.cuda.synchronize()
        assert torch.equal(norm, want) and all(torch.equal(p.grad, q.grad) for p, q in zip(mine, eager))


def _strided(*grads):
    params = [torch.nn.Parameter(torch.zeros(g.shape, dtype=g.dtype, device="cuda")) for g in grads]
    for p, g in zip(params, grads):
        p.grad = g
    return params


def test_a_strided_gradient_given_twice_counts_once():
    print("[case] clip strided twice", flush=True)
    wide = torch.randn(20, 30, device="cuda")
    before = wide.double()
    want = before[:, 2:11].norm()
    p, = _strided(wide[:, 2:11])
    for params in ([p, p], _strided(wide[:, 2:11], wide[:, 2:11]), [p, *_strided(torch.zeros(7, device="cuda"))]):
        wide.copy_(before)
        assert abs(float(sparc_amd.grad_norm([q.grad for q in params])) - float(want)) <= 2.0 ** -22 * float(want)
        norm = sparc_amd.clip_grad_norm_(params, 0.25)
        assert abs(float(norm) - float(want)) <= 2.0 ** -22 * float(want)
        ref = before.clone()
        ref[:, 2:11] *= 0.25 / (want + 1e-6)
        assert ((wide.double() - ref).abs() <= 2.0 ** -21 * ref.abs()).all()


def test_strided_gradients_that_overlap_are_refused():
    """And those that only lie between one another are not."""
    print("[case] clip strided overlap", flush=True)
    wide = torch.ones(20, 30, device="cuda")
    flat = wide.view(-1)
    for grads in ((wide[:, :6], wide[:, 3:9]), (wide[:, 3:9], wide[:, :6]), (wide[:, :6], wide[5:9, 2:4]),
                  (wide[:, ::2], wide[:, ::3]), (wide[:, :6], wide[::3]), (wide[:, :6], wide[4:6]),
                  (wide[2:, :6].t(), wide[:5, 5:9]), (flat[::7], flat[3::5]),
                  (wide[:, :6], wide[:, 10:], wide[:, 5:9]), (wide[::2, ::3], flat[100:250])):
        with pytest.raises(RuntimeError, match="overlap"):
            sparc_amd.clip_grad_norm_(_strided(*grads), 0.5)
    assert torch.equal(wide, torch.ones_like(wide))
    for grads in ((wide[:, :6], wide[:, 6:12], wide[:, 12:]), (wide[:, ::2], wide[:, 1::2]), (wide[::2], wide[1::2, 3:]),
                  (wide[:10, :6], wide[10:]), (wide[:, :6].t(), wide[:, 6:9]), (flat[::6], flat[3::4]),
                  (wide[::2, ::3], wide[1::2, 1::2], wide[::2, 1::3])):
        wide.fill_(1.0)
        inside = torch.zeros_like(wide)
        for g in grads:
            inside.as_strided(g.shape, g.stride(), g.storage_offset()).add_(1.0)
        count = float(inside.sum())
        norm = sparc_amd.clip_grad_norm_(_strided(*grads), 0.5)
        assert abs(float(norm) - math.sqrt(count)) <= 2.0 ** -22 * math.sqrt(count)
        want = torch.where(inside > 0, 0.5 / (math.sqrt(count) + 1e-6), 1.0).double()
        assert ((wide.double() - want).abs() <= 2.0 ** -21).all()


def test_strided_gradients_of_both_types():
    """bf16 values between fp32 ones of the same memory, and the same bytes under
    both types."""
    print("[case] clip strided types", flush=True)
    buf = torch.zeros(12, 16, device="cuda")
    half = buf.view(BF16)  # [12, 32]
    params = _strided(buf[:, :8], half[:, 16:20], half[:, 20::2])
    for p in params:
        p.grad.fill_(0.5)
    _check(params, 0.125)
    with pytest.raises(RuntimeError, match="overlap"):
        sparc_amd.clip_grad_norm_(_strided(buf[:, :8], half[:, 15:20]), 0.5)


@pytest.mark.parametrize("strides", [(5, 3), (10, 2), (0, 0)])
def test_gradients_without_values_in_any_layout(strides):
    print(f"[case] clip empty strides {strides}", flush=True)
    empty = torch.zeros(60, device="cuda").as_strided((0, 5), strides)
    params = _params([(40,)], [F32], 12) + _strided(empty)
    want = L.grad_norm([params[0].grad.cpu()])
    assert abs(float(sparc_amd.grad_norm([p.grad for p in params])) - want) <= 2.0 ** -22 * want
    _check(params, 0.01)


def test_overlaps_of_any_two_layouts():
    """Views with 1 to 3 dimensions and any strides without repeats: refused where,
    and only where, two of them name one value."""
    print("[case] clip overlap of any layouts", flush=True)
    r = random.Random(7)
    base, index, overlapping = torch.zeros(400, device="cuda"), torch.arange(400), 0
    for _ in range(400):
        views = []
        while len(views) < 2:
            shape, strides, reach = [], [], 0
            for _ in range(r.randint(1, 3)):
                shape.append(r.randint(1, 5))
                strides.append(reach + r.randint(1, 7))
                reach += strides[-1] * (shape[-1] - 1)
            if reach < 150:
                order = r.sample(range(len(shape)), len(shape))
                views.append(([shape[k] for k in order], [strides[k] for k in order], r.randint(0, 200)))
        sets = [set(index.as_strided(*v).reshape(-1).tolist()) for v in views]
        params = _strided(*[base.as_strided(*v) for v in views])
        same = views[0] == views[1]
        if sets[0] & sets[1] and not same:
            overlapping += 1
            with pytest.raises(RuntimeError, match="overlap"):
                sparc_amd.clip_grad_norm_(params, 0.5)
        else:
            sparc_amd.clip_grad_norm_(params, 0.5)
    assert 50 < overlapping < 350
