"""GPU: the clipped policy loss at the ends of its range."""

import math

import pytest
import torch

from genrec_amd.policy import policy_loss

pytestmark = pytest.mark.gpu

U = 2.0 ** -24


def _column(value, T, dev="cuda"):
    """[2, T] zeros with `value` at (1, 2)."""
    x = torch.zeros((2, T), device=dev)
    x[1, 2] = value
    return x


@pytest.mark.parametrize("T", [5, 200, 1500])  # rows in registers (of one wave, of a workgroup), rows in passes
@pytest.mark.parametrize("level,gap", [("token", 200.0), ("token", 700.0), ("sequence", 300000.0)])
@pytest.mark.parametrize("delta", [None, 1.5])
def test_no_advantage_and_a_ratio_that_overflows(T, level, gap, delta):
    """exp(200) is past fp32 and 0 times it is 0: the loss is -1 for the first row's tokens, 0 for the second's."""
    x = _column(gap, T).requires_grad_()
    adv = torch.tensor([1.0, 0.0], device="cuda")
    res = policy_loss(x, adv, torch.ones_like(x), torch.zeros_like(x), delta=delta, importance_sampling_level=level)
    (g,) = torch.autograd.grad(res.loss, x)
    assert float(res.loss) == -0.5
    want = torch.zeros_like(g)
    want[0] = -0.5 / T
    assert (g[1] == 0).all() and (g - want).abs().max() <= 2 * U * 0.5 / T
    assert float(res.clip_low) == 0 and float(res.clip_high) == 0
    # without a finite ratio there is nothing to multiply
    bad = policy_loss(_column(math.inf, T), adv, torch.ones_like(x), torch.zeros_like(x), delta=None)
    assert torch.isnan(bad.loss)


@pytest.mark.parametrize("level", ["token", "sequence"])
@pytest.mark.parametrize("T", [5, 200, 1500])
def test_no_old_policy_and_a_token_ruled_out(T, level):
    """Without an old policy the ratio is 1 whatever the log-probability is, -inf (a token that the policy rules out) too."""
    x = (_column(-math.inf, T) - 1.0).requires_grad_()
    adv = torch.tensor([1.0, -3.0], device="cuda")
    res = policy_loss(x, adv, torch.ones_like(x), importance_sampling_level=level)
    (g,) = torch.autograd.grad(res.loss, x)
    assert float(res.loss) == 1.0  # (-1 + 3) / 2
    want = -adv[:, None].expand(2, T) / (2 * T)
    assert (g - want).abs().max() <= 2 * U * 1.5 / T
    assert float(res.clip_low) == 0 and float(res.clip_high) == 0 and float(res.kl) == 0
