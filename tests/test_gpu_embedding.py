"""embedding on the GPU against float64: lookups and the table's gradient over
types, odd widths, alignments, and ids from all different to all the same.

Tolerances: an fp32 sum of c rows in pieces and slices is off by at most some
(16 + c / 128 + 20) roundings of 2^-24 of the summed magnitudes, held to 2^-17
of the largest here; bf16 results are one rounding (2^-8) of such a value."""
import math

import pytest
import torch

import sparc_amd
from oracle import lm_oracle as L

pytestmark = pytest.mark.gpu

F32, BF16 = torch.float32, torch.bfloat16


def _close(got, want, what):
    off = (got.detach().cpu().double() - want).abs()
    bound = 2.0 ** -17 * want.abs().max().clamp_min(1e-30)
    if got.dtype == BF16:
        bound = bound + want.abs() * 2.0 ** -8
    assert (off <= bound).all(), f"{what}: {(off - bound).max().item():.3g} over the bound"


def _ids(kind, n, vocab, g):
    if kind == "uniform":
        return torch.randint(0, vocab, (n,), generator=g)
    if kind == "same":
        return torch.full((n,), vocab - 1)
    if kind == "two":
        return torch.randint(0, 2, (n,), generator=g) * (vocab - 1)
    if kind == "runs":  # equal neighbours, runs of every length up to 40
        return torch.repeat_interleave(torch.arange(n) % vocab, torch.arange(n) % 40 + 1)[:n]
    rank = torch.exp(torch.rand(n, generator=g) * math.log(vocab + 1)).long() - 1
    return rank.clamp_(0, vocab - 1)


def _check(n, vocab, D, dtype, kind="zipf", scale=1.0, pad=None, ids=torch.int64, seed=0):
    print(f"[case] embedding n={n} V={vocab} D={D} {dtype} {kind} pad={pad}", flush=True)
    g = torch.Generator().manual_seed(seed)
    tokens = _ids(kind, n, vocab, g).to(ids)
    w = torch.randn(vocab, D, generator=g).to(dtype)
    dy = torch.randn(n, D, generator=g).to(dtype)
    wd = w.cuda().requires_grad_()
    y = sparc_amd.embedding(tokens.cuda(), wd, scale=scale, padding_idx=pad)
    dw, = torch.autograd.grad(y, [wd], dy.cuda())
    want = L.embedding(tokens, w, scale)
    # the scale rounded to fp32, one fp32 product, rounded to 8 bits in bf16
    one = 2.0 ** -23 + (2.0 ** -8 if dtype == BF16 else 0.0)
    assert ((y.detach().cpu().double() - want).abs() <= want.abs() * one).all()
    _close(dw, L.embedding_grad(tokens, vocab, dy, scale, pad), "dw")
    assert dw.dtype == dtype and y.dtype == dtype


@pytest.mark.parametrize("dtype", [F32, BF16], ids=["f32", "bf16"])
@pytest.mark.parametrize("D", [1, 3, 8, 20, 64, 100, 513, 768, 1001])
def test_widths(D, dtype):
    _check(300, 97, D, dtype, scale=math.sqrt(D), seed=D)


@pytest.mark.parametrize("n,vocab", [(1, 1), (1, 500), (15, 9), (16, 9), (17, 9), (100, 1), (127, 300), (128, 40),
                                     (129, 40), (2048, 511), (2049, 512),
                                     (5000, 32768), (5000, 300000)])
@pytest.mark.parametrize("kind", ["zipf", "uniform", "same", "two", "runs"])
def test_sizes_and_frequencies(n, vocab, kind):
    _check(n, vocab, 24, F32, kind, seed=n)


def test_many_tokens():
    """More positions than 64 tiles of the sort."""
    _check(70001, 1000, 8, F32, "zipf")
    _check(70001, 3, 8, F32, "same")


@pytest.mark.parametrize("n,vocab,D,dtype,kind", [(100003, 1000, 400, BF16, "zipf"), (100003, 5000, 337, F32, "runs"),
                                                  (60001, 3, 300, F32, "two"), (100003, 40, 336, BF16, "uniform"),
                                                  (1100001, 3000, 16, F32, "zipf"), (99001, 300000, 9, F32, "uniform")])
def test_long_batches(n, vocab, D, dtype, kind):
    """Longer pieces with more work, the tiles' counts summed beforehand, and
    past 2^20 positions larger tiles."""
    _check(n, vocab, D, dtype, kind, seed=n)


def test_few_tokens_of_a_large_vocabulary():
    """Ids and positions that do not fit into 32 bits together."""
    _check(3000, (1 << 21) + 5, 1, F32, "uniform")
    _check(4096, (1 << 19) + 5, 1, F32, "zipf")


@pytest.mark.parametrize("pad", [0, 5, -1])
def test_padding_and_id_types(pad):
    _check(700, 40, 33, F32, "zipf", pad=pad)
    _check(700, 40, 32, BF16, "same", pad=pad, ids=torch.int32)


def test_ids_outside_the_table():
    """They read nothing: a row of NaN, and no part in the gradient."""
    print("[case] embedding outside ids", flush=True)
    g = torch.Generator().manual_seed(1)
    tokens = torch.tensor([[3, -1, 7, 2 ** 40], [10, 9, -2 ** 62, 3]])
    w, dy = torch.randn(10, 48, generator=g), torch.randn(2, 4, 48, generator=g)
    wd = w.cuda().requires_grad_()
    y = sparc_amd.embedding(tokens.cuda(), wd)
    dw, = torch.autograd.grad(y, [wd], dy.cuda())
    want = L.embedding(tokens, w, 1.0)
    assert torch.equal(y.isnan().cpu(), want.isnan()) and torch.equal(y.detach().cpu().double().nan_to_num(),
                                                                      want.nan_to_num())
    _close(dw, L.embedding_grad(tokens, 10, dy, 1.0), "dw")


def test_no_tokens():
    print("[case] embedding without tokens", flush=True)
    w = torch.randn(70, 24, device="cuda", requires_grad=True)
    y = sparc_amd.embedding(torch.zeros(2, 0, dtype=torch.int64, device="cuda"), w)
    dw, = torch.autograd.grad(y.sum(), [w])
    assert y.shape == (2, 0, 24) and dw.shape == w.shape and not dw.any()


def test_strides_and_alignment():
    """Ids and gradients of other orders, and a table that begins off a 16-byte
    boundary."""
    print("[case] embedding strides", flush=True)
    g = torch.Generator().manual_seed(2)
    tokens = torch.randint(0, 50, (12, 30), generator=g)
    w, dy = torch.randn(50, 16, generator=g).bfloat16(), torch.randn(30, 12, 16, generator=g).bfloat16()
    wd = torch.cat((torch.zeros(1).bfloat16(), w.reshape(-1))).cuda()[1:].view(50, 16).requires_grad_()
    y = sparc_amd.embedding(tokens.cuda().t(), wd, scale=0.5)
    dyd = dy.cuda().transpose(0, 1).contiguous().transpose(0, 1)
    dw, = torch.autograd.grad(y, [wd], dyd)
    want = L.embedding(tokens.t(), w, 0.5)
    assert ((y.detach().cpu().double() - want).abs() <= want.abs() * 2.0 ** -8).all()
    _close(dw, L.embedding_grad(tokens.t(), 50, dy, 0.5), "dw")


def test_gradient_is_the_difference():
    """The lookup is linear in the table: <dw, u> is L(W + u) - L(W - u) over 2
    up to the sums' rounding, L = <dy, y> in fp64."""
    print("[case] embedding differences", flush=True)
    g = torch.Generator().manual_seed(3)
    tokens = _ids("zipf", 900, 130, g).cuda()
    w, u, dy = (torch.randn(*s, generator=g).cuda() for s in ((130, 40), (130, 40), (900, 40)))
    leaf = w.clone().requires_grad_()
    dw, = torch.autograd.grad(sparc_amd.embedding(tokens, leaf, scale=3.0), [leaf], dy)
    loss = [(sparc_amd.embedding(tokens, w + s * u, scale=3.0).double() * dy.double()).sum() for s in (1, -1)]
    want = float(loss[0] - loss[1]) / 2
    assert abs(float((dw.double() * u.double()).sum()) - want) <= 2.0 ** -20 * 3.0 * 900 * 40


def test_equal_calls_give_equal_bits():
    print("[case] embedding determinism", flush=True)
    g = torch.Generator().manual_seed(4)
    tokens = _ids("zipf", 20000, 5000, g).cuda()
    w, dy = torch.randn(5000, 136, generator=g).bfloat16().cuda(), torch.randn(20000, 136, generator=g).bfloat16().cuda()
    leaf = w.requires_grad_()
    grads = [torch.autograd.grad(sparc_amd.embedding(tokens, leaf), [leaf], dy)[0] for _ in range(3)]
    assert torch.equal(grads[0], grads[1]) and torch.equal(grads[0], grads[2])


@pytest.mark.parametrize("dtype", [F32, BF16], ids=["f32", "bf16"])
@pytest.mark.parametrize("D", [1, 7, 64, 513, 1001, 2056])
@pytest.mark.parametrize("n", [1, 5, 127, 128, 129])
def test_few_positions(n, D, dtype):
    """Rows of one and of several blocks of columns, whole vectors and not, with
    every kind of id."""
    _check(n, 90, D, dtype, "zipf", scale=math.sqrt(D), seed=n)
    _check(n, 90, D, dtype, "same", pad=-1, ids=torch.int32, seed=n)
    _check(n, 90, D, dtype, "same", pad=3, seed=n)
    _check(n, 4099, D, dtype, "uniform", pad=11, ids=torch.int32, seed=n)
    _check(n, 7, D, dtype, "runs", pad=2, seed=n)


def test_few_positions_outside_the_table():
    """And equal calls give equal bits."""
    print("[case] embedding few positions", flush=True)
    g = torch.Generator().manual_seed(6)
    for dtype in (F32, BF16):
        tokens = torch.randint(-3, 44, (100,), generator=g)
        w, dy = torch.randn(40, 1001, generator=g).to(dtype), torch.randn(100, 1001, generator=g).to(dtype)
        leaf = w.cuda().requires_grad_()
        grads = [torch.autograd.grad(sparc_amd.embedding(tokens.cuda(), leaf), leaf, dy.cuda())[0] for _ in range(3)]
        _close(grads[0], L.embedding_grad(tokens, 40, dy, 1.0), "dw")
        assert torch.equal(grads[0], grads[1]) and torch.equal(grads[0], grads[2])
