"""gated_linear_unit against its formula in 64 bits.

Tolerances.  A projection of D terms is off by e = (D + 8) 2^-24 of the sum of its
terms' sizes.  The activations' slopes are at most 1.13 and change by at most 0.8 a
unit, so y is off by 1.2 e_g |u| + |act| e_u, and what the gradients are made of, dg
= dy u act'(g) and du = dy act(g), by |dy| (1.2 e_u + 0.8 |u| e_g) and 1.2 |dy| e_g;
16 further roundings each.  With bfloat16 inputs both are rounded before their
products (2^-8 each; in small calls what that leaves is multiplied too, 2^-16), and so
is every result (2^-8)."""
import pytest
import torch

import sparc_amd
from oracle import block_oracle as O

pytestmark = pytest.mark.gpu
F32, BF16 = torch.float32, torch.bfloat16
IDS = dict(ids=lambda d: str(d).replace("torch.", ""))
ACTS = ("silu", "gelu", "relu", "sigmoid")
U = 2.0 ** -24


def _case(N, D, F, dtype, seed):
    g = torch.Generator().manual_seed(seed)
    r = lambda *s: torch.randn(*s, generator=g)
    return r(N, D).to(dtype), (r(F, D) * D ** -0.5).to(dtype), (r(F, D) * D ** -0.5).to(dtype), r(N, F).to(dtype)


def _run(x, wg, wu, dy, act, shape=None, rest=2.0 ** -8):
    dtype = x.dtype
    half = 2.0 ** -8 if dtype == BF16 else U
    X, G, W, DY = (t.double() for t in (x, wg, wu, dy))
    N, D = x.shape
    F = len(wg)
    g = (X @ G.T).requires_grad_()
    u, a = X @ W.T, O.activation(g, act)
    slope, = torch.autograd.grad(a.sum(), g)
    g, a = g.detach(), a.detach()
    eg, eu = ((D + 8) * U * (X.abs() @ w.abs().T) for w in (G, W))
    if act == "relu":  # no sign may depend on rounding
        assert ((g.abs() > eg) | (g == 0)).all()
    y, ey = a * u, 1.2 * eg * u.abs() + a.abs() * eu + 16 * U * (a * u).abs()
    dg, du = DY * u * slope, DY * a
    edg = DY.abs() * (1.2 * eu + 0.8 * u.abs() * eg) + 16 * U * (DY * u).abs() * 1.2
    edu = 1.2 * DY.abs() * eg + 16 * U * du.abs()
    if dtype == BF16:
        edg, edu = edg + rest * dg.abs(), edu + rest * du.abs()
    want = {"y": (y, ey),
            "dx": (dg @ G + du @ W, edg @ G.abs() + edu @ W.abs() + (2 * F + 8) * U * (dg.abs() @ G.abs() + du.abs() @ W.abs())),
            "dwg": (dg.T @ X, edg.T @ X.abs() + (N + 72) * U * (dg.abs().T @ X.abs())),
            "dwu": (du.T @ X, edu.T @ X.abs() + (N + 72) * U * (du.abs().T @ X.abs()))}
    leaves = [t.cuda().requires_grad_() for t in (x, wg, wu)]
    inp = leaves[0] if shape is None else leaves[0].view(*shape, D)
    out = sparc_amd.gated_linear_unit(inp, leaves[1], leaves[2], activation=act)
    assert out.shape == (*inp.shape[:-1], F)
    grads = torch.autograd.grad(out, leaves, dy.cuda().view(out.shape))
    for (name, (ref, tol)), got in zip(want.items(), (out.detach().view(N, F), *grads)):
        assert got.dtype == dtype and got.shape == ref.shape
        off = ((got.cpu().double() - ref).abs() - tol - half * (ref.abs() + tol)).max().item()
        assert off <= 0.0, f"{name}: {off} over a tolerance of up to {tol.max().item()}"


SHAPES = [(1, 1, 1), (1, 8, 8), (3, 5, 7), (16, 32, 64), (17, 33, 65), (128, 64, 64), (129, 96, 200), (5, 1000, 3),
          (1, 256, 513), (300, 40, 31), (64, 512, 256), (256, 128, 128), (700, 136, 72), (2000, 24, 40),
          (6000, 520, 1032)]  # the last one in large tiles, all products split


@pytest.mark.parametrize("dtype", [F32, BF16], **IDS)
@pytest.mark.parametrize("shape", SHAPES, ids=str)
def test_against_the_formula(shape, dtype):
    print(f"[case] gated {shape} {dtype}", flush=True)
    _run(*_case(*shape, dtype, seed=sum(shape)), "silu")


@pytest.mark.parametrize("dtype", [F32, BF16], **IDS)
@pytest.mark.parametrize("act", ACTS)
def test_activations(act, dtype):
    x, wg, wu, dy = _case(70, 24, 40, dtype, seed=2)
    if act == "relu":  # projections that are not near zero: one value each
        x, wg = torch.where(x.abs() < 0.1, torch.ones_like(x), x), torch.eye(40, 24).to(dtype)
    _run(x, wg, wu, dy, act, shape=(7, 10))


def test_large_and_odd_values():
    wg = torch.tensor([[1.0], [-1.0]], device="cuda")
    wu = torch.ones(2, 1, device="cuda")
    x = torch.tensor([[0.0], [1e4], [-1e4], [float("nan")], [88.0], [-104.0]], device="cuda")
    for act in ACTS:
        leaf = x.clone().requires_grad_()
        y = sparc_amd.gated_linear_unit(leaf, wg, wu, activation=act)
        y.sum().backward()
        ref = x.cpu().double().requires_grad_()
        r = O.gated_linear_unit(ref, wg.cpu(), wu.cpu(), act)
        r.sum().backward()
        assert y[3].isnan().all() and leaf.grad[3].isnan().all()
        ok = [0, 1, 2, 4, 5]
        torch.testing.assert_close(y.detach().cpu().double()[ok], r.detach()[ok], rtol=1e-5, atol=1e-30)
        torch.testing.assert_close(leaf.grad.cpu().double()[ok], ref.grad[ok], rtol=1e-5, atol=1e-30)


@pytest.mark.parametrize("dtype", [F32, BF16], **IDS)
def test_a_projection_that_overflows(dtype):
    """relu of -inf is zero, and so are its gradients."""
    x, wg, wu = (torch.tensor([[v]], dtype=dtype, device="cuda").requires_grad_() for v in (-3e38, 10.0, 1e-38))
    y = sparc_amd.gated_linear_unit(x, wg, wu, activation="relu")
    y.sum().backward()
    assert not y.any() and not x.grad.any() and not wg.grad.any() and not wu.grad.any()


@pytest.mark.parametrize("shape", [(2, 59, 3183), (32, 64, 96), (150, 416, 2272), (1001, 256, 1000), (700, 72, 4000)],
                         ids=str)
def test_small_calls_lose_nothing_between_their_products(shape):
    _run(*_case(*shape, BF16, seed=sum(shape)), "silu", rest=2.0 ** -16)


@pytest.mark.parametrize("rows", [1, 64, 65, 128, 129, 256])
def test_few_rows_over_wide_weights(rows):
    """Tiles of every size, whatever the rows."""
    _run(*_case(rows, 136, 2056, BF16, seed=rows), "silu")


def test_views_some_gradients_and_equal_bits():
    x, wg, wu, dy = _case(150, 72, 56, BF16, seed=7)
    x, wg, wu, dy = x.cuda(), wg.cuda(), wu.cuda(), dy.cuda()
    wide = torch.stack((x, x), -1)[..., 0]  # strides of 2

    def grads(which, x=x):
        leaves = [t.detach().requires_grad_(n in which) for n, t in enumerate((x, wg.T.contiguous().T, wu))]
        y = sparc_amd.gated_linear_unit(*leaves)
        return dict(zip(which, torch.autograd.grad(y, [leaves[n] for n in which], dy)), y=y.detach())

    every = grads((0, 1, 2))
    for which in ((0,), (1,), (2,), (0, 2), (0, 1, 2)):
        got = grads(which, wide)
        assert all(torch.equal(got[n], every[n]) for n in got)


def test_no_rows():
    x, wg, wu, dy = (t.cuda().requires_grad_() for t in _case(0, 8, 16, F32, seed=1))
    y = sparc_amd.gated_linear_unit(x, wg, wu)
    assert y.shape == (0, 16)
    g = torch.autograd.grad(y, (x, wg, wu), dy.detach())
    assert g[0].shape == (0, 8) and not g[1].any() and not g[2].any()


def test_once_differentiable():
    x, wg, wu, dy = (t.cuda().requires_grad_() for t in _case(4, 8, 8, F32, seed=1))
    y = sparc_amd.gated_linear_unit(x, wg, wu)
    with pytest.raises(RuntimeError, match="not twice"):
        torch.autograd.grad(y, x, dy.detach(), create_graph=True)
    y = sparc_amd.gated_linear_unit(x, wg, wu)
    with torch.no_grad():
        wg.add_(1.0)
    with pytest.raises(RuntimeError, match="modified by an inplace"):
        y.sum().backward()
