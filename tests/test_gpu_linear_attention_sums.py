"""linear_attention in bfloat16 where a sum nearly cancels, so that the rounding of the
result does not hide what its terms lose: a state or a score that enters a product as
two bfloat16 values, both rounded to nearest, is off by at most 2^-17: of a value from 1
to 2 the first leaves 2^-8 at most, and half a step of what is below that is 2^-17.

Fifteen terms of 1 + 2^-7 - 2^-23, whose 24 bits are all needed, all but cancel one of
15.125, which bfloat16 holds.  With A the sum of the terms' sizes a result may be off by
2^-17 A, by 64 2^-24 A for the fp32 sums of 16 terms and the factors' few roundings, and
by its own rounding, 2^-8 of its value."""
import pytest
import torch

import sparc_amd
from oracle import block_oracle as O

pytestmark = pytest.mark.gpu
LONG = 1 + 2.0 ** -7 - 2.0 ** -23


def _check(s):
    g = {n: x.cuda() for n, x in s.items()}
    o = sparc_amd.linear_attention(**g, scale=1.0)[0].cpu().double()
    want = O.linear_attention(**s, scale=1.0)[0]
    size = O.linear_attention(**{n: x if n == "log_decay" else x.abs() for n, x in s.items()}, scale=1.0)[0]
    assert want[:, -1].abs().max() < 0.01 and size[:, -1].min() > 30.0  # it does cancel
    tol = (2.0 ** -17 + 64 * 2.0 ** -24) * size + 2.0 ** -8 * want.abs()
    off = ((o - want).abs() - tol).max().item()
    assert off <= 0.0, f"{off} over a tolerance of up to {tol.max().item()}"


@pytest.mark.parametrize("K,V", [(16, 16), (64, 64), (128, 128), (100, 72)])
def test_of_a_state(K, V):
    q, state = torch.zeros(1, 1, 1, K), torch.zeros(1, 1, K, V)
    q[..., 0], q[..., 1:16] = -1.0, 1.0
    state[:, :, 0], state[:, :, 1:16] = 15.125, LONG
    none = lambda d: torch.zeros(1, 1, 1, d, dtype=torch.bfloat16)
    _check(dict(q=q.bfloat16(), k=none(K), v=none(V), log_decay=torch.zeros(1), state=state))


@pytest.mark.parametrize("K,V", [(16, 16), (64, 64), (128, 128), (100, 72)])
def test_of_scores(K, V):
    """A score of these bits is the sum of three products."""
    q, k, v = torch.zeros(1, 16, 1, K), torch.zeros(1, 16, 1, K), torch.ones(1, 16, 1, V)
    q[..., :3] = 1.0
    k[..., 0], k[..., 1], k[..., 2] = 1.0, 2.0 ** -7 - 2.0 ** -15, 2.0 ** -15 - 2.0 ** -23
    k[:, 0], v[:, 0] = 0.0, -1.0
    k[:, 0, :, 0] = 15.125
    assert k[0, 1].sum().item() == LONG and torch.equal(k, k.bfloat16().float())
    _check(dict(q=q.bfloat16(), k=k.bfloat16(), v=v.bfloat16(), log_decay=torch.zeros(1)))
