"""layer_norm on the GPU against float64: outputs and gradients over widths of
every form (lanes of 1 to 16 bytes, one to sixteen waves per row, rows read
again), types, strides and alignments.

Tolerances, from the arithmetic: fp32 sums over a row of D values in registers
and across lanes add at most some 32 + log2(D) roundings of 2^-24, and a fixed
number of further operations follows, so fp32 results are held to 2^-17 of the
largest; bf16 results are one rounding (2^-8) of such a value.  Sums over R rows
add sqrt(R) such terms in partial sums."""
import pytest
import torch

import sparc_amd
from oracle import lm_oracle as L

pytestmark = pytest.mark.gpu

F32, BF16 = torch.float32, torch.bfloat16


def _case(rows, D, dtype, pdtype, seed, mean=0.4):
    g = torch.Generator().manual_seed(seed)
    x = (torch.randn(rows, D, generator=g) * 1.7 + mean).to(dtype)
    w = (1.0 + 0.3 * torch.randn(D, generator=g)).to(pdtype)
    b = (0.2 * torch.randn(D, generator=g)).to(pdtype)
    dy = torch.randn(rows, D, generator=g).to(dtype)
    return x, w, b, dy


def _close(got, want, what, scale=1.0):
    """Within 2^-17 of the largest value, and one rounding of bf16 results."""
    assert got.shape == want.shape, what
    want = want.double()
    off = (got.detach().cpu().double() - want).abs()
    bound = scale * 2.0 ** -17 * want.abs().max().clamp_min(1e-30)
    if got.dtype == BF16:
        bound = bound + want.abs() * 2.0 ** -8
    worst = (off - bound).max().item()
    assert worst <= 0.0, f"{what}: {worst:.3g} over the bound, largest {want.abs().max():.3g}"


def _check(rows, D, dtype, pdtype, weight=True, bias=True, seed=0):
    x, w, b, dy = _case(rows, D, dtype, pdtype, seed)
    w, b = w if weight else None, b if bias else None
    leaves = [t.cuda().requires_grad_() for t in (x, w, b) if t is not None]
    at = iter(leaves)
    args = [next(at) if t is not None else None for t in (x, w, b)]
    y = sparc_amd.layer_norm(*args, eps=1e-5)
    grads = torch.autograd.grad(y, leaves, dy.cuda())
    _close(y, L.layer_norm(x, w, b, 1e-5), "y")
    dx, dw, db = L.layer_norm_grads(x, w, 1e-5, dy)
    want = [dx] + ([dw] if weight else []) + ([db] if bias else [])
    for got, ref, name in zip(grads, want, ("dx", "first parameter", "second parameter")):
        _close(got, ref, name, scale=1.0 if name == "dx" else 4.0)
    with torch.no_grad():  # the form without saved statistics: the same values
        assert torch.equal(sparc_amd.layer_norm(*[None if a is None else a.detach() for a in args]), y)


@pytest.mark.parametrize("dtype,pdtype", [(F32, F32), (BF16, BF16), (BF16, F32)], ids=["f32", "bf16", "bf16_f32"])
@pytest.mark.parametrize("D", [1, 2, 7, 64, 200, 513, 768, 1001, 1024, 1536, 2050, 4096, 5000])
def test_widths(D, dtype, pdtype):
    print(f"[case] layer norm D={D} {dtype} {pdtype}", flush=True)
    _check(37, D, dtype, pdtype, seed=D)


@pytest.mark.parametrize("D,dtype", [(8193, F32), (16384, F32), (16388, F32), (24576, BF16), (24577, BF16),
                                     (16386, BF16), (40000, BF16)])
def test_wide_rows(D, dtype):
    print(f"[case] layer norm D={D} {dtype}", flush=True)
    _check(5, D, dtype, F32, seed=D)


@pytest.mark.parametrize("dtype", [F32, BF16], ids=["f32", "bf16"])
@pytest.mark.parametrize("vectors", [1, 8, 9, 16, 17, 32, 33, 64, 65, 96, 97, 128, 129, 192, 193, 256, 257, 512, 513, 768,
                                     769, 1024, 1025, 1536, 1537, 2048])
def test_where_forms_meet(vectors, dtype):
    """Rows of as many 16-byte vectors as a form holds, and of one value less or
    more, with few rows and with many."""
    print(f"[case] layer norm {vectors} vectors {dtype}", flush=True)
    V = 4 if dtype == F32 else 8
    _check(5, vectors * V, dtype, dtype, seed=vectors)
    _check(3, vectors * V - 1, dtype, F32, seed=vectors)
    _check(1030, vectors * V - V + 1, dtype, dtype, seed=vectors)


@pytest.mark.parametrize("rows", [1, 2, 63, 1023, 1024, 4500])
def test_row_counts(rows):
    print(f"[case] layer norm rows={rows}", flush=True)
    _check(rows, 96, BF16, BF16, seed=rows)
    _check(rows, 97, F32, F32, seed=rows)


@pytest.mark.parametrize("weight,bias", [(False, False), (True, False), (False, True)])
def test_without_parameters(weight, bias):
    print(f"[case] layer norm weight={weight} bias={bias}", flush=True)
    _check(19, 264, F32, F32, weight, bias)
    _check(19, 264, BF16, F32, weight, bias)


def test_no_rows():
    print("[case] layer norm without rows", flush=True)
    x = torch.zeros(0, 12, device="cuda", requires_grad=True)
    w, b = torch.ones(12, device="cuda", requires_grad=True), torch.ones(12, device="cuda", requires_grad=True)
    y = sparc_amd.layer_norm(x, w, b)
    dx, dw, db = torch.autograd.grad(y.sum(), [x, w, b])
    assert y.shape == dx.shape == (0, 12) and not dw.any() and not db.any()


def test_strides_and_alignment():
    """A transposed input, an incoming gradient that is an expanded row, and
    tensors that begin off a 16-byte boundary."""
    print("[case] layer norm strides", flush=True)
    x, w, b, dy = _case(40, 96, BF16, BF16, 3)
    xt = x.t().contiguous().cuda().t()
    assert not xt.is_contiguous()
    xt.requires_grad_()
    wd, bd = (torch.cat((t.new_zeros(1), t)).cuda()[1:].requires_grad_() for t in (w, b))
    y = sparc_amd.layer_norm(xt, wd, bd)
    row = dy[:1].cuda().expand(40, 96)
    got = torch.autograd.grad(y, [xt, wd, bd], row)
    _close(y, L.layer_norm(x, w, b, 1e-5), "y")
    for a, ref, name in zip(got, L.layer_norm_grads(x, w, 1e-5, dy[:1].expand(40, 96)), ("dx", "dw", "db")):
        _close(a, ref, name, scale=4.0)


def test_large_mean_keeps_its_precision():
    """A mean of 1000 standard deviations: the differences from it, and so the
    variance, are off by the mean's own rounding (1000 2^-24 of a deviation),
    not by that of squares."""
    print("[case] layer norm large mean", flush=True)
    x, w, b, _ = _case(16, 1000, F32, F32, 4, mean=0.0)
    x = x + 1700.0
    y = sparc_amd.layer_norm(x.cuda(), w.cuda(), b.cuda())
    want = L.layer_norm(x, w, b, 1e-5)
    assert (y.cpu().double() - want).abs().max() <= 4 * 1000 * 2.0 ** -24 * want.abs().max()


def test_constant_rows_and_nan():
    """A constant row has no variance: y is the bias; NaN stays in its row."""
    print("[case] layer norm constant rows, NaN", flush=True)
    x = torch.full((3, 320), 2.5, device="cuda")
    x[1] = torch.randn(320)
    x[1, 7] = float("nan")
    b = torch.randn(320, device="cuda")
    y = sparc_amd.layer_norm(x, torch.ones(320, device="cuda"), b)
    assert torch.equal(y[0], b) and torch.equal(y[2], b) and y[1].isnan().all()


def test_gradient_against_differences():
    """<gradient, u> against (L(p + h u) - L(p - h u)) / 2h of the kernel's own
    forward, L = <dy, y> in fp64.  y is off by up to 2^-20 per value, at random:
    over sqrt(n) values of |dy| ~ 1 and 1 / 2h = 64 that is 0.01; the formula's
    third derivative adds h^2 ~ 6e-5 of the gradient."""
    print("[case] layer norm differences", flush=True)
    x, w, b, dy = (t.cuda() for t in _case(24, 500, F32, F32, 6))
    leaves = [t.requires_grad_() for t in (x, w, b)]
    grads = torch.autograd.grad(sparc_amd.layer_norm(*leaves), leaves, dy)
    g = torch.Generator().manual_seed(1)
    h = 2.0 ** -7
    for at, (leaf, grad) in enumerate(zip(leaves, grads)):
        u = torch.randn(leaf.shape, generator=g).cuda()
        loss = []
        for s in (1, -1):
            args = [t.detach() + s * h * u if i == at else t.detach() for i, t in enumerate(leaves)]
            loss.append((sparc_amd.layer_norm(*args).double() * dy.double()).sum())
        diff, want = float(loss[0] - loss[1]) / (2 * h), float((grad.double() * u.double()).sum())
        assert abs(diff - want) <= 0.01 + 1e-3 * float(grad.norm() * u.norm()) / leaf.numel() ** 0.5 + 1e-3 * abs(want)


def test_equal_calls_give_equal_bits_on_any_stream():
    print("[case] layer norm determinism", flush=True)
    x, w, b, dy = (t.cuda() for t in _case(3000, 768, BF16, BF16, 8))
    leaves = [t.requires_grad_() for t in (x, w, b)]
    first = torch.autograd.grad(sparc_amd.layer_norm(*leaves), leaves, dy)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        again = torch.autograd.grad(sparc_amd.layer_norm(*leaves), leaves, dy)
    torch.cuda.current_stream().wait_stream(side)
    assert all(torch.equal(p, q) for p, q in zip(first, again))


@pytest.mark.parametrize("given", ["xwb", "xw", "xb", "x"])
def test_gradients_of_some_inputs_only(given):
    """Every choice of inputs that want a gradient, with parameters that are there
    and not, and a gradient of y that is one row expanded."""
    print(f"[case] layer norm gradients of some of {given}", flush=True)
    x, w, b, _ = _case(9, 40, F32, F32, 3)
    dy = torch.linspace(-1.0, 2.0, 40).expand(9, 40)
    dx, dw, db = L.layer_norm_grads(x, w if "w" in given else None, 1e-5, dy)
    want = {"x": dx, "w": dw, "b": db}
    for pick in range(1, 1 << len(given)):
        wanted = [n for i, n in enumerate(given) if pick >> i & 1]
        t = {n: v.cuda().requires_grad_(n in wanted) for n, v in zip("xwb", (x, w, b)) if n in given}
        y = sparc_amd.layer_norm(t["x"], t.get("w"), t.get("b"))
        grads = torch.autograd.grad(y, [t[n] for n in wanted], dy[0].cuda().expand(9, 40))
        for n, g in zip(wanted, grads):
            _close(g, want[n], f"d{n} of {wanted}", scale=1.0 if n == "x" else 4.0)


@pytest.mark.parametrize("dtype", [F32, BF16], ids=["f32", "bf16"])
@pytest.mark.parametrize("D", [1, 2, 3, 5, 7])
def test_short_rows_of_large_values(D, dtype):
    """mean * rstd overflows: nothing of that comes from behind a row's end.
    Rows whose mean is exact are taken, so that xhat is 0."""
    print(f"[case] layer norm short rows of large values D={D} {dtype}", flush=True)
    x = torch.tensor([2.0 ** 121, -2.0 ** 122, 1.0])[:, None].expand(3, D).to(dtype).contiguous()
    _, w, b, dy = _case(3, D, dtype, F32, D)
    leaves = [t.cuda().requires_grad_() for t in (x, w, b)]
    y = sparc_amd.layer_norm(*leaves)
    assert torch.equal(y, leaves[2].detach().to(dtype).expand_as(y))
    dx, dw, db = torch.autograd.grad(y, leaves, dy.cuda())
    assert not dw.any()
    _close(dx, L.layer_norm_grads(x, w, 1e-5, dy)[0], "dx")
    _close(db, dy.double().sum(0), "db", scale=4.0)


def _off_by_the_mean(x, rstd):
    """How far xhat may be off where the mean is rounded to fp32: half a unit in
    its last place, and as much again for the sums behind it."""
    return 2.0 ** -23 * x.double().mean(-1, keepdim=True).abs() * rstd


@pytest.mark.parametrize("D", [3, 64, 200, 768, 1001, 5000, 16388, 24577, 33001, 50001])
@pytest.mark.parametrize("dtype", [F32, BF16], ids=["f32", "bf16"])
def test_constant_rows_of_any_value(D, dtype):
    """The mean of a constant row is its value, to the last bit: xhat and the
    weight's gradient are 0, y is the bias, and rstd is 1 / sqrt(eps).  (A sum of
    D values and a product with 1 / D, each rounded, are some units off.)"""
    print(f"[case] layer norm constant rows D={D} {dtype}", flush=True)
    values = [1000.7, 12345.67, 1e6 + 0.3, -1e6 - 0.3, 1e-3, 0.0, torch.finfo(dtype).min]
    x = torch.tensor(values, dtype=torch.float64).to(dtype)[:, None].expand(len(values), D).contiguous()
    _, w, b, dy = _case(len(values), D, dtype, F32, D)
    leaves = [t.cuda().requires_grad_() for t in (x, w, b)]
    y = sparc_amd.layer_norm(*leaves)
    dx, dw, db = torch.autograd.grad(y, leaves, dy.cuda())
    assert torch.equal(y, leaves[2].detach().to(dtype).expand_as(y))
    assert torch.equal(y, sparc_amd.layer_norm(*[t.detach() for t in leaves]))
    assert not dw.any()
    _close(dx, L.layer_norm_grads(x, w, 1e-5, dy)[0], "dx")
    _close(db, dy.double().sum(0), "db", scale=4.0)


@pytest.mark.parametrize("D", [200, 768, 1001, 5000, 16388, 33001])
@pytest.mark.parametrize("mean", [1000.7, 12345.67, 1e6 + 0.3])
def test_nearly_constant_rows(D, mean):
    """A spread of some units in the values' last place: the variance is that of
    the values, and xhat is off by no more than the mean's rounding to fp32.
    dx = rstd (g - mean(g) - xhat mean(g xhat)) is then off by rstd e (|mean(g
    xhat)| + |xhat| mean|g|), e the error of xhat, and dw by e times the sum of
    |dy|."""
    print(f"[case] layer norm nearly constant rows D={D} mean={mean}", flush=True)
    _, w, b, dy = _case(8, D, F32, F32, D)
    g = torch.Generator().manual_seed(D)
    x = (mean + mean * 2.0 ** -21 * torch.randn(8, D, generator=g, dtype=torch.float64)).float()
    x[0, 1:] = x[0, 0]
    x[0, D // 2] = x[0, 0] * (1.0 + 2.0 ** -20)  # one value off
    leaves = [t.cuda().requires_grad_() for t in (x, w, b)]
    y = sparc_amd.layer_norm(*leaves)
    dx, dw, _ = torch.autograd.grad(y, leaves, dy.cuda())
    x64, g64 = x.double(), dy.double() * w.double()
    rstd = 1.0 / torch.sqrt(x64.var(-1, correction=0, keepdim=True) + 1e-5)
    xhat = (x64 - x64.mean(-1, keepdim=True)) * rstd
    e = _off_by_the_mean(x, rstd)
    want, (want_x, want_w, _) = L.layer_norm(x, w, b, 1e-5), L.layer_norm_grads(x, w, 1e-5, dy)

    def held(got, ref, bound):
        off = (got.detach().cpu().double() - ref).abs() - bound - 2.0 ** -17 * ref.abs().max()
        assert off.max() <= 0.0, f"{off.max().item():.3g} over the bound"

    held(y, want, e * w.double().abs())
    along = (g64 * xhat).mean(-1, keepdim=True).abs()
    held(dx, want_x, rstd * e * (along + xhat.abs() * g64.abs().mean(-1, keepdim=True)))
    held(dw, want_w, (e * dy.double().abs()).sum(0))


@pytest.mark.parametrize("D", [768, 16388, 32768, 40001])
def test_one_value_far_from_the_others(D):
    """At either end of the row and between: no sum about a value that is far off."""
    print(f"[case] layer norm one far value D={D}", flush=True)
    x, w, b, _ = _case(3, D, F32, F32, D)
    x[0, 0] = x[1, D // 2] = x[2, D - 1] = 1e4
    y = sparc_amd.layer_norm(x.cuda(), w.cuda(), b.cuda()).cpu().double()
    want = L.layer_norm(x, w, b, 1e-5)
    xhat = L.layer_norm(x, None, None, 1e-5)
    assert ((y - want).abs() <= 2.0 ** -17 * (w.double().abs() * (1.0 + xhat.abs()) + b.double().abs())).all()


@pytest.mark.parametrize("pdtype", ["same", F32], ids=["same", "f32"])
@pytest.mark.parametrize("D,dtype", [(28000, F32), (32768, F32), (32769, F32), (40001, F32), (49152, BF16), (49153, BF16),
                                     (60007, BF16)])
def test_the_widest_rows(D, dtype, pdtype):
    """On both sides of what a workgroup holds in registers."""
    print(f"[case] layer norm D={D} {dtype} {pdtype}", flush=True)
    _check(5, D, dtype, dtype if pdtype == "same" else pdtype, seed=D)
    _check(70, D, dtype, F32, bias=False, seed=D + 1)
