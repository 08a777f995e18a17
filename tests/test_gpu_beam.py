"""beam_search_step and reorder_states on the GPU against float64.

A candidate's score is off from its 64-bit value by the log-sum-exp's fp32 sum
(some 2^-22) and the roundings of three fp32 operations on values up to the
largest |logit| and |score|, 4 2^-24 of them; two candidates nearer to each other
than twice that may change places.  Where scores are equal by construction the
order is checked exactly."""
import math

import pytest
import torch

import sparc_amd
from oracle import lm_oracle as L

pytestmark = pytest.mark.gpu

F32, BF16 = torch.float32, torch.bfloat16
INF = math.inf


def _inputs(B, K, V, dtype, seed, spread=3.0):
    g = torch.Generator().manual_seed(seed)
    logits = (torch.randn(B, K, V, generator=g) * spread).to(dtype)
    scores = -torch.cumsum(torch.rand(B, K, generator=g) * 2.0, 1)
    return logits, scores, torch.rand(B, K, generator=g) < 0.2


def _check(logits, scores, finished=None, eos=None, step=None):
    """Every chosen candidate's 64-bit score is that of its place in the 64-bit
    order, no candidate is chosen twice, and what is returned for it is right."""
    B, K, V = logits.shape
    if step is None:
        step = sparc_amd.beam_search_step(logits.cuda(), scores.cuda(),
                                          finished=None if finished is None else finished.cuda(), eos_id=eos)
    tokens, parents, got = step.tokens.cpu(), step.parents.cpu(), step.scores.cpu().double()
    cand = L.beam_candidates(logits, scores, finished, eos).reshape(B, K * V)
    flat = parents * V + tokens
    assert ((tokens >= 0) & (tokens < V) & (parents >= 0) & (parents < K)).all()
    assert all(len(set(row)) == K for row in flat.tolist())
    best = torch.sort(cand, dim=-1, descending=True, stable=True).values[:, :K]
    mine = cand.gather(1, flat)
    finite = torch.isfinite(cand)
    reach = float(cand[finite].abs().max()) if finite.any() else 1.0
    reach = max(reach, float(logits.float()[logits.isfinite()].abs().max()) if logits.isfinite().any() else 0.0)
    tol = 2.0 ** -21 + 4 * 2.0 ** -24 * reach
    for a, b, what in ((mine, best, "the chosen candidates"), (got, mine, "the returned scores")):
        assert torch.equal(torch.isfinite(a), torch.isfinite(b)), what
        assert torch.equal(a[~torch.isfinite(a)].nan_to_num(7.0), b[~torch.isfinite(b)].nan_to_num(7.0)), what
        ok = torch.isfinite(a)
        assert ((a[ok] - b[ok]).abs() <= 2 * tol).all(), f"{what}: {(a[ok] - b[ok]).abs().max():.3g}"
    if eos is not None:
        was = torch.zeros(B, K, dtype=torch.bool) if finished is None else finished
        assert torch.equal(step.finished.cpu(), was.gather(1, parents) | (tokens == eos))
    return step


@pytest.mark.parametrize("dtype", [F32, BF16], ids=["f32", "bf16"])
@pytest.mark.parametrize("B,K,V", [(1, 1, 1), (1, 1, 5), (3, 2, 1), (2, 4, 3), (2, 32, 7), (5, 3, 64), (2, 5, 1001),
                                   (1, 8, 4099), (2, 16, 50001), (7, 32, 2050), (300, 4, 513), (1, 4, 131072)])
def test_sizes(B, K, V, dtype):
    print(f"[case] beam B={B} K={K} V={V} {dtype}", flush=True)
    logits, scores, finished = _inputs(B, K, V, dtype, V + K)
    _check(logits, scores)
    _check(logits, scores, finished, V // 2)
    _check(logits, scores, None, 0)


@pytest.mark.parametrize("dtype", [F32, BF16], ids=["f32", "bf16"])
def test_first_step(dtype):
    """One beam and K - 1 that are not there yet."""
    print(f"[case] beam first step {dtype}", flush=True)
    logits, scores, _ = _inputs(3, 6, 3001, dtype, 1)
    scores[:, 0], scores[:, 1:] = 0.0, -INF
    step = _check(logits, scores)
    assert not step.parents.any()


@pytest.mark.parametrize("dtype", [F32, BF16], ids=["f32", "bf16"])
@pytest.mark.parametrize("value", [0.0, -1.25, 80.0])
def test_equal_logits_take_the_lowest_tokens(dtype, value):
    """Every logit the same (an untrained model): ties everywhere, over several
    spans of the vocabulary, and beams that are better than others by far less
    than a token."""
    print(f"[case] beam equal logits {value} {dtype}", flush=True)
    logits = torch.full((2, 4, 9001), value, dtype=dtype)
    step = sparc_amd.beam_search_step(logits.cuda(), torch.zeros(2, 4, device="cuda"))
    assert step.parents.tolist() == [[0, 0, 0, 0]] * 2 and step.tokens.tolist() == [[0, 1, 2, 3]] * 2
    scores = torch.tensor([[-3.0, -1.0, -1.0, -2.0]] * 2)
    step = sparc_amd.beam_search_step(logits.cuda(), scores.cuda())
    assert step.parents.tolist() == [[1, 1, 1, 1]] * 2 and step.tokens.tolist() == [[0, 1, 2, 3]] * 2


def test_different_logits_of_equal_score_take_the_lowest_token():
    """Logits 2^-24 apart near 0 under a score of -1000 round to one score; the
    lowest token wins, not the largest logit, so the row is ranked by score."""
    print("[case] beam scores that round together", flush=True)
    V = 5003
    x = torch.full((1, 2, V), -30.0)
    x[0, 0, 4000:4040] = torch.arange(40).flip(0) * 2.0 ** -22  # the largest at the lowest token
    x[0, 1, 100:140] = torch.arange(40) * 2.0 ** -22            # the largest at the highest token
    for beam, first in ((0, 4000), (1, 100)):
        scores = torch.full((1, 2), -INF)
        scores[0, beam] = -1000.0
        step = sparc_amd.beam_search_step(x.cuda(), scores.cuda())
        assert step.parents.tolist() == [[beam, beam]] and step.tokens.tolist() == [[first, first + 1]]


@pytest.mark.parametrize("K", [1, 3, 11, 32])
@pytest.mark.parametrize("V", [67, 5003, 70001])
def test_rows_ranked_by_score(K, V):
    """Logits of three values, apart by less than 2^-20 within each, under a score
    of -4096 whose last place is 2^-11: three scores, the lowest tokens of the
    best first, wherever in the row they stand."""
    print(f"[case] beam ranked by score K={K} V={V}", flush=True)
    g = torch.Generator().manual_seed(K * V)
    level = (torch.randint(0, 3000, (2, K, V), generator=g) > 2990).float() + torch.randint(0, 2, (2, K, V), generator=g)
    logits = level + torch.rand(2, K, V, generator=g) * 2.0 ** -21
    scores = torch.full((2, K), -INF)
    scores[0, 0] = scores[1, K - 1] = -4096.0
    step = sparc_amd.beam_search_step(logits.cuda(), scores.cuda())
    for b, beam in ((0, 0), (1, K - 1)):
        assert step.parents[b].tolist() == [beam] * K
        assert step.tokens[b].tolist() == torch.sort(-level[b, beam], stable=True).indices[:K].tolist()


@pytest.mark.parametrize("dtype", [F32, BF16], ids=["f32", "bf16"])
def test_masked_tokens(dtype):
    """-inf and the type's lowest value over most or all of the vocabulary."""
    print(f"[case] beam masks {dtype}", flush=True)
    logits, scores, finished = _inputs(2, 4, 3000, dtype, 2)
    logits[0, :, 2:] = -INF                       # two tokens left
    logits[1, 1:, :] = -INF                       # one beam left
    logits[1, 0, 5:] = torch.finfo(dtype).min     # five tokens left, the others masked by value
    _check(logits, scores)
    _check(logits, scores, finished, 1)
    logits[0] = -INF                              # nothing left: the lowest tokens of the first beam, -inf
    step = _check(logits, scores)
    assert step.parents[0].tolist() == [0] * 4 and step.tokens[0].tolist() == [0, 1, 2, 3]
    assert torch.equal(step.scores[0].cpu(), torch.full((4,), -INF))


def test_all_beams_finished():
    print("[case] beam all finished", flush=True)
    logits, scores, _ = _inputs(2, 5, 600, BF16, 3)
    done = torch.ones(2, 5, dtype=torch.bool)
    step = _check(logits, scores, done, 17)
    assert step.tokens.eq(17).all() and step.finished.all()
    assert torch.equal(step.parents.cpu(), torch.arange(5).expand(2, 5)) and torch.equal(step.scores.cpu(), scores)


def test_nan_and_infinite_logits_rank_first():
    print("[case] beam NaN", flush=True)
    for bad in (math.nan, INF):
        logits, scores, _ = _inputs(1, 3, 5000, F32, 4)
        logits[0, 2, 4321] = bad
        step = sparc_amd.beam_search_step(logits.cuda(), scores.cuda())
        assert step.scores.isnan().all() and step.parents.tolist() == [[2, 2, 2]]
        assert step.tokens.tolist() == [[0, 1, 2]]
    logits, scores, _ = _inputs(1, 3, 5000, F32, 4)
    scores[0, 1] = math.nan
    step = sparc_amd.beam_search_step(logits.cuda(), scores.cuda())
    assert step.scores.isnan().all() and step.parents.tolist() == [[1, 1, 1]]


@pytest.mark.parametrize("order", ["rising", "falling"])
@pytest.mark.parametrize("K", [1, 32])
def test_sorted_logits(order, K):
    """Every logit larger than those before it, and the reverse."""
    print(f"[case] beam {order} K={K}", flush=True)
    row = torch.arange(9000.0) * 1e-2
    logits = (row if order == "rising" else row.flip(0)).expand(2, K, 9000).contiguous()
    _check(logits, -torch.arange(K).float().expand(2, K) * 100.0)


def test_logits_apart():
    """The last position of a sequence's logits, rows off 16-byte boundaries."""
    print("[case] beam strided logits", flush=True)
    g = torch.Generator().manual_seed(5)
    for dtype in (F32, BF16):
        seq = (torch.randn(2 * 3, 4, 1003, generator=g) * 3).to(dtype).cuda()
        last = seq[:, -1].view(2, 3, 1003)
        assert not last.is_contiguous()
        scores = -torch.rand(2, 3, generator=g)
        _check(last.cpu(), scores, step=sparc_amd.beam_search_step(last, scores.cuda()))
        shared = seq[:2, -1][:, None].expand(2, 3, 1003)  # every beam the same row
        _check(shared.cpu(), scores, step=sparc_amd.beam_search_step(shared, scores.cuda()))


@pytest.mark.parametrize("in_place", [False, True])
@pytest.mark.parametrize("K", [1, 3, 8, 11, 32])
def test_reorder(K, in_place):
    print(f"[case] reorder K={K} in_place={in_place}", flush=True)
    g = torch.Generator().manual_seed(K)
    B = 5
    parents = torch.randint(0, K, (B, K), generator=g)
    parents[0] = torch.arange(K)            # nothing moves
    parents[1] = torch.arange(K).flip(0)    # everything does
    shapes = [(B * K, 1), (B * K, 12), (B * K, 1001), (B * K, 3, 700)]
    states = [(torch.randn(s, generator=g).cuda(), torch.randn(s, generator=g).bfloat16().cuda()
               if s[-1] % 2 == 0 else torch.randn(s, generator=g).cuda()) for s in shapes]
    want = [tuple(L.reorder(p.cpu(), parents) for p in s) for s in states]
    kept = [tuple(p.clone() for p in s) for s in states]
    out = sparc_amd.reorder_states(states, parents.cuda(), out_states=states if in_place else None)
    for a, b, old, s in zip(out, want, kept, states):
        for x, y, o, q in zip(a, b, old, s):
            assert torch.equal(x.cpu(), y) and (x.data_ptr() == q.data_ptr()) is in_place
            assert in_place or torch.equal(o, q)


def test_reorder_many_planes_and_layouts():
    """More planes than one launch takes; planes of other strides and starts."""
    print("[case] reorder planes", flush=True)
    g = torch.Generator().manual_seed(9)
    parents = torch.randint(0, 4, (3, 4), generator=g)
    states = [torch.randn(12, 5 + i % 7, generator=g).cuda() for i in range(200)]
    states[3] = torch.randn(8, 12, generator=g).cuda().t()
    states[4] = torch.randn(12 * 6 + 1, generator=g).cuda()[1:].view(12, 6)
    out = sparc_amd.reorder_states(states, parents.cuda())
    assert all(torch.equal(o.cpu(), L.reorder(s.cpu(), parents)) for o, s in zip(out, states))


def test_reorder_refuses_and_bad_parents():
    print("[case] reorder refusals", flush=True)
    a, b = torch.randn(6, 8, device="cuda"), torch.randn(6, 8, device="cuda")
    parents = torch.tensor([[0, 1, 2], [2, 2, 2]], device="cuda")
    with pytest.raises(ValueError, match="another one"):
        sparc_amd.reorder_states([a, b], parents, out_states=[b, a])
    with pytest.raises(ValueError, match="another one"):
        sparc_amd.reorder_states([a, b], parents, out_states=[a, a])
    with pytest.raises(ValueError, match="another one"):
        sparc_amd.reorder_states([a, a], parents, out_states=[a, a])
    wide = torch.randn(7, 8, device="cuda")
    with pytest.raises(ValueError, match="another one"):
        sparc_amd.reorder_states([wide[:6]], parents, out_states=[wide[1:]])
    fresh = sparc_amd.reorder_states([a, a], parents)  # to other memory a state may come twice
    assert torch.equal(fresh[0], fresh[1])
    with pytest.raises(ValueError, match="out_states"):
        sparc_amd.reorder_states([a], parents, out_states=[b[:5]])
    with pytest.raises(ValueError, match="tensors for"):
        sparc_amd.reorder_states([a, b], parents, out_states=[a])
    out, = sparc_amd.reorder_states([a], torch.tensor([[0, -1, 2], [3, 2 ** 40, 1]], device="cuda"))
    assert out[[1, 3, 4]].isnan().all() and torch.equal(out[[0, 2, 5]], a[[0, 2, 4]])


def test_step_with_states_and_streams():
    """The whole step on a side stream, in place, against the parts."""
    print("[case] beam step with states", flush=True)
    logits, scores, finished = _inputs(2, 4, 2000, F32, 6)
    g = torch.Generator().manual_seed(6)
    states = [tuple(torch.randn(8, 320, generator=g).cuda() for _ in range(2)) for _ in range(3)]
    kept = [tuple(p.clone() for p in s) for s in states]
    x, s, f = logits.cuda(), scores.cuda(), finished.cuda()
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step = sparc_amd.beam_search_step(x, s, finished=f, eos_id=3, states=states, out_states=states)
    torch.cuda.current_stream().wait_stream(side)
    _check(logits, scores, finished, 3, step=step)
    again = sparc_amd.beam_search_step(x, s, finished=f, eos_id=3)
    assert torch.equal(step.tokens, again.tokens) and torch.equal(step.scores, again.scores) and again.states == []
    for new, old in zip(step.states, kept):
        for p, q in zip(new, old):
            assert torch.equal(p.cpu(), L.reorder(q.cpu(), step.parents.cpu()))
    empty = sparc_amd.beam_search_step(x[:0], s[:0])
    assert empty.tokens.shape == (0, 4)


@pytest.mark.parametrize("dtype,width", [(F32, 1028), (F32, 257), (BF16, 257)], ids=["16", "4", "2"])
@pytest.mark.parametrize("K", [1, 3, 4, 7, 8, 13, 16, 32])
def test_reorder_in_place_of_many_rows(K, dtype, width):
    """More workgroups than the GPU runs at once, at each width of access."""
    print(f"[case] reorder in place K={K} {dtype} {width}", flush=True)
    g = torch.Generator().manual_seed(K)
    B = 300
    parents = torch.randint(0, K, (B, K), generator=g)
    parents[0] = torch.arange(K)
    parents[1] = torch.arange(K).flip(0)
    states = [tuple(torch.randn(B * K, width, generator=g).to(dtype).cuda() for _ in range(2)) for _ in range(2)]
    want = [tuple(L.reorder(p.cpu(), parents) for p in s) for s in states]
    out = sparc_amd.reorder_states(states, parents.cuda(), out_states=states)
    for a, b, s in zip(out, want, states):
        for x, y, q in zip(a, b, s):
            assert x.data_ptr() == q.data_ptr() and torch.equal(x.cpu(), y)
    bad = parents.clone()
    bad[5, K - 1], bad[7, 0] = K, -1
    kept = states[0][0].clone()
    sparc_amd.reorder_states(states, bad.cuda(), out_states=states)
    ok = ((bad >= 0) & (bad < K)).reshape(-1)
    rows = L.reorder(torch.arange(B * K), bad.clamp(0, K - 1))
    assert torch.equal(states[0][0][ok.cuda()], kept[rows[ok].cuda()]) and states[0][0][~ok.cuda()].isnan().all()
