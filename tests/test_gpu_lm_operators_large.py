"""The operators around the stack where element offsets pass 2^31 (and byte
offsets 2^32): the rows at both ends against float64, the rest in bulk."""
import math

import pytest
import torch

import sparc_amd
from oracle import lm_oracle as L

pytestmark = pytest.mark.gpu

BF16 = torch.bfloat16


def _some(rows):
    """The first and last rows, and those on both sides of element 2^31."""
    return [0, 1, rows // 2, rows - 2, rows - 1]


def test_layer_norm_beyond_32_bits():
    """2^31 and more elements: y, dx by rows; the parameters' gradients against
    the same sums of the kernel's own xhat in fp64, block by block."""
    rows, D = 70_000, 32_768
    print(f"[case] layer norm {rows} x {D}", flush=True)
    x = torch.empty(rows, D, dtype=BF16, device="cuda").normal_(0.3, 1.5)
    dy = torch.empty_like(x).normal_()
    w, b = (torch.randn(D, device="cuda") for _ in range(2))
    leaves = [t.requires_grad_() for t in (x, w, b)]
    y = sparc_amd.layer_norm(*leaves)
    dx, dw, db = torch.autograd.grad(y, leaves, dy)
    at = _some(rows)
    xs, dys = x.detach()[at].cpu(), dy[at].cpu()
    want = L.layer_norm(xs, w.detach().cpu(), b.detach().cpu(), 1e-5)
    tol = 2.0 ** -17 * want.abs().max()
    assert ((y.detach()[at].cpu().double() - want).abs() <= want.abs() * 2.0 ** -8 + tol).all()
    want = L.layer_norm_grads(xs, w.detach().cpu(), 1e-5, dys)[0]
    assert ((dx[at].cpu().double() - want).abs() <= want.abs() * 2.0 ** -8 + 2.0 ** -17 * want.abs().max()).all()
    sum_w, sum_b = torch.zeros(D, dtype=torch.float64, device="cuda"), torch.zeros(D, dtype=torch.float64, device="cuda")
    for k in range(0, rows, 2_000):
        xk, dk = x.detach()[k:k + 2_000].double(), dy[k:k + 2_000].double()
        var, mu = torch.var_mean(xk, dim=1, correction=0, keepdim=True)
        sum_w += (dk * (xk - mu) / torch.sqrt(var + 1e-5)).sum(0)
        sum_b += dk.sum(0)
    for got, ref in ((dw, sum_w), (db, sum_b)):  # partial sums of 280 rows each, then 256 of them
        assert (got.double() - ref).abs().max() <= 2.0 ** -15 * ref.abs().max()


def test_embedding_beyond_32_bits():
    vocab, D, n = 300_001, 8_192, 300
    print(f"[case] embedding {vocab} x {D}", flush=True)
    w = torch.empty(vocab, D, dtype=BF16, device="cuda").normal_().requires_grad_()
    tokens = torch.randint(0, vocab, (n,), generator=torch.Generator().manual_seed(1))
    tokens[:4] = torch.tensor([0, vocab - 1, vocab - 1, 262_144])  # 262144 x 8192 = 2^31
    dy = torch.empty(n, D, dtype=BF16, device="cuda").normal_()
    y = sparc_amd.embedding(tokens.cuda(), w)
    dw, = torch.autograd.grad(y, [w], dy)
    assert torch.equal(y, w.detach()[tokens.cuda()])
    named = tokens.unique()
    want = torch.zeros(len(named), D, dtype=torch.float64)
    want.index_add_(0, torch.searchsorted(named, tokens), dy.cpu().double())
    got = dw[named.cuda()].cpu().double()
    assert ((got - want).abs() <= want.abs() * 2.0 ** -8 + 1e-6).all()
    assert int((dw != 0).any(dim=1).sum()) == len(named)


def test_clip_beyond_32_bits():
    n = (1 << 31) + 4_099
    print(f"[case] clip {n} values", flush=True)
    p = torch.nn.Parameter(torch.empty(n, dtype=BF16, device="cuda"))
    p.grad = torch.empty_like(p).normal_(0.0, 0.01)
    kept = p.grad[-5_000:].clone()
    want = math.sqrt(sum(float(c.double().square().sum()) for c in p.grad.split(1 << 28)))
    norm = sparc_amd.clip_grad_norm_([p], 0.5 * want)
    assert abs(float(norm) - want) <= 2.0 ** -22 * want
    ref = kept.double() * (0.5 * want / (want + 1e-6))
    assert ((p.grad[-5_000:].double() - ref).abs() <= ref.abs() * (2.0 ** -8 + 2.0 ** -21)).all()


def test_beam_and_states_beyond_32_bits():
    B, K, V = 4, 32, 17_000_003  # 2.2e9 logits
    print(f"[case] beam {B} x {K} x {V}", flush=True)
    logits = torch.full((B, K, V), -20.0, dtype=BF16, device="cuda")
    g = torch.Generator().manual_seed(2)
    best = {}
    for b in range(B):
        for k, tok, val in ((0, 0, 5.0), (31, V - 1, 9.0), (15, V // 2, 7.0)):
            logits[b, k, tok] = val
            best[b, k] = tok
    scores = torch.full((B, K), -50.0, device="cuda")
    scores[:, [0, 15, 31]] = 0.0
    step = sparc_amd.beam_search_step(logits, scores)
    assert step.parents[:, :3].tolist() == [[31, 15, 0]] * B
    assert step.tokens[:, :3].tolist() == [[V - 1, V // 2, 0]] * B
    lse = math.log((V - 1) * math.exp(-20.0) + math.exp(9.0))
    assert (step.scores[:, 0] - (9.0 - lse)).abs().max() <= 1e-5
    del logits
    plane = torch.empty(128, 10_000_000, device="cuda").normal_()  # 5.1 GB
    parents = torch.randint(0, 32, (4, 32), generator=g).cuda()
    rows = (parents + 32 * torch.arange(4, device="cuda")[:, None]).reshape(-1)
    out, = sparc_amd.reorder_states([plane], parents)
    for r in (0, 1, 64, 126, 127):
        assert torch.equal(out[r], plane[rows[r]])
    sparc_amd.reorder_states([plane], parents, out_states=[plane])
    assert torch.equal(out, plane)


def test_few_ids_of_a_table_beyond_32_bits():
    vocab, D, n = 300_001, 8_192, 100
    print(f"[case] embedding {n} of {vocab} x {D}", flush=True)
    w = torch.empty(vocab, D, dtype=BF16, device="cuda").normal_().requires_grad_()
    tokens = torch.randint(0, vocab, (n,), generator=torch.Generator().manual_seed(3))
    tokens[:5] = torch.tensor([0, vocab - 1, vocab - 1, 262_143, 262_144])
    dy = torch.empty(n, D, dtype=BF16, device="cuda").normal_()
    y = sparc_amd.embedding(tokens.cuda(), w)
    dw, = torch.autograd.grad(y, [w], dy)
    assert torch.equal(y, w.detach()[tokens.cuda()])
    named = tokens.unique()
    want = torch.zeros(len(named), D, dtype=torch.float64)
    want.index_add_(0, torch.searchsorted(named, tokens), dy.cpu().double())
    got = dw[named.cuda()].cpu().double()
    assert ((got - want).abs() <= want.abs() * 2.0 ** -8 + 1e-6).all()
    assert int((dw != 0).any(dim=1).sum()) == len(named)
