"""qk_norm_rotary against its formula in 64 bits.

Tolerances.  With r the size of a head's largest normed value: the sum of squares is
a sum of D terms that are not negative (D 2^-24 relative at most, half of it in
rstd), and the rest a dozen roundings of values of at most twice that size; a
gradient has two such sums.  A result in bfloat16 is rounded once: 2^-8 of its
value.  The weights' gradients are sums over n heads: (n + D + 16) 2^-24 of the sum
of the terms' sizes."""
import pytest
import torch

import sparc_amd
from oracle import block_oracle as O

pytestmark = pytest.mark.gpu
F32, BF16 = torch.float32, torch.bfloat16
IDS = dict(ids=lambda d: str(d).replace("torch.", ""))
EPS = 1e-6


def _half(dtype):
    return 2.0 ** -8 if dtype == BF16 else 2.0 ** -24


def _case(B, T, H, G, D, R, dtype, pdtype, seed, layout="plain"):
    g = torch.Generator().manual_seed(seed)
    r = lambda *s: torch.randn(*s, generator=g)
    if layout == "fused":
        both = (r(B, T, (H + 2 * G) * D) * 1.3).to(dtype)
        q, k = both[..., :H * D].unflatten(-1, (H, D)), both[..., H * D:(H + G) * D].unflatten(-1, (G, D))
    elif layout == "heads first":
        q, k = ((r(B, n, T, D) * 1.3).to(dtype).transpose(1, 2) for n in (H, G))
    else:
        q, k = ((r(B, T, n, D) * 1.3).to(dtype) for n in (H, G))
    w = [(1.0 + 0.3 * r(D)).to(pdtype) if pdtype else None for _ in range(2)]
    return q, k, *w, r(B, T, H, D).to(dtype), r(B, T, G, D).to(dtype)


def _on_gpu(x):
    if x is None:
        return None
    return torch.empty_strided(x.shape, x.stride(), dtype=x.dtype, device="cuda").copy_(x)


def _run(q, k, wq, wk, dq, dk, table, positions, interleaved):
    B, T = q.shape[:2]
    at = torch.arange(T).expand(B, T) if positions is None else positions.long().expand(B, T)
    leaves = [x.detach().double().requires_grad_() for x in (q, k, wq, wk) if x is not None]
    it = iter(leaves[2:])
    refs = [O.norm_rotary(x, next(it) if w is not None else None, table, at, interleaved, EPS)
            for x, w in ((leaves[0], wq), (leaves[1], wk))]
    grads = torch.autograd.grad(refs, leaves, (dq.double(), dk.double()))
    mine = [_on_gpu(x).requires_grad_() if x is not None else None for x in (q, k, wq, wk)]
    ys = sparc_amd.qk_norm_rotary(*mine, table.cuda(), None if positions is None else positions.cuda(),
                                  interleaved=interleaved, eps=EPS)
    got = torch.autograd.grad(ys, [x for x in mine if x is not None], (dq.cuda(), dk.cuda()))
    D = q.shape[-1]
    for y, ref, x in zip(ys, refs, (q, k)):
        assert y.dtype == x.dtype and y.is_contiguous()
        tol = _half(x.dtype) * ref.abs() + (D + 16) * 2.0 ** -24 * 2 * ref.abs().amax(-1, keepdim=True)
        assert ((y.detach().cpu().double() - ref).abs() <= tol).all()
    for x, dy, w, d, ref, dw, dw_ref in zip((q, k), (dq, dk), (wq, wk), got[:2], grads[:2],
                                            got[2:] or (None, None), grads[2:] or (None, None)):
        assert d.dtype == x.dtype and d.shape == x.shape
        x, dy = x.double(), dy.double()
        rstd = 1.0 / torch.sqrt(x.square().mean(-1, keepdim=True) + EPS)
        # sizes: |g| is at most the two values of a pair, |g w| and |xhat mean(g w xhat)|
        top = dy.abs().amax(-1, keepdim=True) * 2 * (1.0 if w is None else w.double().abs().max())
        size = rstd * (top + (x * rstd).abs().amax(-1, keepdim=True) ** 2 * top)
        tol = _half(d.dtype) * ref.abs() + (2 * D + 32) * 2.0 ** -24 * size
        assert ((d.cpu().double() - ref).abs() <= tol).all()
        if dw is not None:
            n = x.shape[0] * x.shape[1] * x.shape[2]
            terms = (2 * dy.abs().amax(-1, keepdim=True) * (x * rstd).abs()).sum((0, 1, 2))
            assert dw.dtype == w.dtype
            assert ((dw.cpu().double() - dw_ref).abs() <= _half(dw.dtype) * dw_ref.abs()
                    + (n + D + 16) * 2.0 ** -24 * terms).all()


SHAPES = [  # B, T, H, G, D, R
    (1, 1, 1, 1, 1, 0), (2, 3, 2, 1, 2, 2), (2, 5, 3, 2, 7, 4), (1, 40, 4, 4, 64, 64), (2, 9, 6, 1, 128, 128),
    (3, 17, 5, 2, 90, 42), (1, 6, 2, 2, 256, 64), (2, 3, 1, 1, 512, 512), (1, 7, 2, 1, 511, 510), (2, 4, 12, 3, 80, 32),
    (1, 11, 3, 3, 36, 20), (1, 300, 2, 2, 40, 40),
    (2, 10000, 5, 2, 20, 12),  # enough for several heads at once, with heads left over
]


@pytest.mark.parametrize("interleaved", [False, True], ids=["halves", "pairs"])
@pytest.mark.parametrize("dtype,pdtype", [(F32, F32), (BF16, BF16), (BF16, F32)], **IDS)
@pytest.mark.parametrize("shape", SHAPES, ids=str)
def test_against_the_formula(shape, dtype, pdtype, interleaved):
    print(f"[case] rotary {shape} {dtype} {pdtype} {interleaved}", flush=True)
    table = O.rotary_table(shape[1] + 5, shape[5]).float()
    _run(*_case(*shape, dtype, pdtype, seed=sum(shape)), table, None, interleaved)


@pytest.mark.parametrize("layout", ["fused", "heads first"])
@pytest.mark.parametrize("dtype", [F32, BF16], **IDS)
def test_strides_positions_and_no_weights(dtype, layout):
    table = O.rotary_table(200, 16).float()
    positions = torch.randint(0, 200, (3, 10), generator=torch.Generator().manual_seed(1))
    for at in (positions, positions[0], positions[:, :1], positions.int()):
        _run(*_case(3, 10, 4, 2, 24, 16, dtype, None, seed=5, layout=layout), table, at, False)


def test_the_table_is_that_of_the_angles():
    table = sparc_amd.rotary_table(5000, 8, device="cuda")
    want = O.rotary_table(5000, 8)
    # cosines and sines of angles in 64 bits (2^-40 for 5000 rad), rounded once
    assert table.dtype == F32 and ((table.cpu().double() - want).abs() <= 2.0 ** -24 + 2.0 ** -38).all()
    for bad in ((-1, 8), (4, 7)):
        with pytest.raises(ValueError):
            sparc_amd.rotary_table(*bad)


def test_a_position_outside_the_table_shows():
    q, k, wq, wk, dq, dk = _case(1, 4, 2, 1, 16, 8, F32, F32, seed=3)
    table = sparc_amd.rotary_table(10, 8, device="cuda")
    at = torch.tensor([0, 10, -1, 9], device="cuda")
    leaf = q.cuda().requires_grad_()
    yq, yk = sparc_amd.qk_norm_rotary(leaf, k.cuda(), wq.cuda(), wk.cuda(), table, at)
    assert yq[:, 1:3].isnan().all() and yk[:, 1:3].isnan().all()
    good, _ = sparc_amd.qk_norm_rotary(q.cuda(), k.cuda(), wq.cuda(), wk.cuda(), table, at.clamp(0, 9))
    assert torch.equal(good[:, ::3], yq[:, ::3])
    d, = torch.autograd.grad(yq, leaf, dq.cuda())
    assert d[:, 1:3].isnan().all() and d[:, ::3].isfinite().all()


def test_some_gradients_only():
    q, k, wq, wk, dq, dk = (x.cuda() for x in _case(2, 5, 3, 2, 32, 32, BF16, F32, seed=8))
    table = sparc_amd.rotary_table(5, 32, device="cuda")

    def grads(which):
        x = [t.detach().requires_grad_(n in which) for n, t in enumerate((q, k, wq, wk))]
        y = sparc_amd.qk_norm_rotary(*x, table)
        return dict(zip(which, torch.autograd.grad(y, [x[n] for n in which], (dq, dk))))

    every = grads((0, 1, 2, 3))
    for which in ((0,), (1,), (2,), (3,), (1, 2)):
        for n, g in grads(which).items():
            assert torch.equal(g, every[n])


def test_rows_of_zero_and_of_large_values():
    q, k, wq, wk, _, _ = _case(1, 3, 2, 2, 64, 64, F32, F32, seed=6)
    q[:, 0], q[:, 1] = 0.0, q[:, 1] * 1e15
    table = sparc_amd.rotary_table(3, 64, device="cuda")
    yq, _ = sparc_amd.qk_norm_rotary(q.cuda(), k.cuda(), wq.cuda(), wk.cuda(), table)
    ref = O.norm_rotary(q, wq, table.cpu(), torch.arange(3)[None], False, EPS)
    assert not yq[:, 0].any()
    assert ((yq.cpu().double() - ref).abs() <= (64 + 16) * 2.0 ** -23 * ref.abs().amax(-1, keepdim=True)).all()


def test_equal_calls_give_equal_bits_and_once_differentiable():
    q, k, wq, wk, dq, dk = (x.cuda().requires_grad_() for x in _case(4, 100, 8, 2, 64, 64, BF16, BF16, seed=4))
    table = sparc_amd.rotary_table(100, 64, device="cuda")
    runs = []
    for _ in range(2):
        y = sparc_amd.qk_norm_rotary(q, k, wq, wk, table)
        runs.append((*y, *torch.autograd.grad(y, (q, k, wq, wk), (dq.detach(), dk.detach()))))
    assert all(torch.equal(a, b) for a, b in zip(*runs))
    y, _ = sparc_amd.qk_norm_rotary(q, k, wq, wk, table)
    with pytest.raises(RuntimeError, match="not twice"):
        torch.autograd.grad(y, q, dq.detach(), create_graph=True)
    with pytest.raises(RuntimeError, match="no backward"):
        sparc_amd.qk_norm_rotary(q, k, wq, wk, table.requires_grad_())


def test_no_tokens():
    q, k, wq, wk, dq, dk = (x.cuda().requires_grad_() for x in _case(2, 0, 3, 2, 16, 16, F32, F32, seed=4))
    y = sparc_amd.qk_norm_rotary(q, k, wq, wk, sparc_amd.rotary_table(0, 16, device="cuda"))
    assert y[0].shape == q.shape and y[1].shape == k.shape
    g = torch.autograd.grad(y, (q, wq, wk), (dq.detach(), dk.detach()))
    assert g[0].shape == q.shape and not g[1].any() and not g[2].any()
