"""GPU: how finely the logits' gradient G reaches the two gradients of ``policy.lm_head_token_logps``.

Hidden states of -1, 0 and 1 and weights of whole eighths make every logit exact in fp32, so what is left is G's own error
and the sums'.  u = 2^-24.  An element of G is p times fp32 factors: the row's sum of exponentials carries
(V / 256 + 160) u, the argument of the exponential 3 u (|log p| + 20), the factors 12 u; it is held in two bf16 pieces, the
second within half a step (2^-8) of what the first leaves (at most 2^-8 of the element), 2^-16 in all; products are added
in fp32, off by (terms) u of the sum of their sizes, and the result is rounded to bf16 once (2^-8)."""

import math

import pytest
import torch

from genrec_amd.policy import lm_head_token_logps

pytestmark = pytest.mark.gpu

U = 2.0 ** -24
HALF = 2.0 ** -8


def _exact_inputs(groups, K, H, V, seed):
    """Groups of K rows that share a hidden state, gradients that add up to 0 within a group, tokens below V / 2."""
    dev = torch.device("cuda", 0)
    gen = torch.Generator(device=dev).manual_seed(seed)
    states = torch.randint(-1, 2, (groups, 1, H), generator=gen, device=dev)
    hidden = states.expand(groups, K, H).reshape(-1, H).to(torch.bfloat16)
    weight = (torch.randint(-4, 5, (V, H), generator=gen, device=dev) / 8).to(torch.bfloat16)
    ids = torch.randint(0, max(1, V // 2), (groups * K,), generator=gen, device=dev)
    g = torch.randint(-300, 301, (groups, K), generator=gen, device=dev).float() / 1024
    g[:, -1] = -g[:, :-1].sum(1)  # exact: whole 1024ths
    return hidden, weight, ids, g.reshape(-1)


def _definition(hidden, weight, ids, g, h):
    x = hidden.double() @ weight.double().T
    lp = x - x.max(1, keepdim=True).values
    lp = lp - lp.exp().sum(1, keepdim=True).log()
    p = lp.exp()
    G = -p * g.double()[:, None]
    if h is not None:
        G = G - h.double()[:, None] * p * (lp - (p * lp).sum(1, keepdim=True))
    G.scatter_add_(1, ids[:, None], g.double()[:, None])
    return G, p, lp


@pytest.mark.parametrize("groups,K,H,V", [(1, 3, 64, 40), (5, 4, 128, 1000), (20, 16, 64, 777), (33, 8, 192, 300), (300, 7, 64, 513)])
@pytest.mark.parametrize("entropy", [False, True])
@pytest.mark.parametrize("keep_bytes", [8 << 30, 0])
def test_gradients_that_cancel(groups, K, H, V, entropy, keep_bytes):
    hidden, weight, ids, g = _exact_inputs(groups, K, H, V, seed=groups + V)
    x, w = hidden.detach().requires_grad_(), weight.detach().requires_grad_()
    lp, ent = lm_head_token_logps(x, w, ids, return_entropy=True, keep_bytes=keep_bytes)
    h = g.flip(0) * 0.125 if entropy else None
    dh, dw = torch.autograd.grad([lp, ent] if entropy else lp, [x, w], [g, h] if entropy else g)
    G, p, lp_all = _definition(hidden, weight, ids, g, h)
    rel = (V / 256 + 160) * U
    size = g.double().abs()[:, None]
    if entropy:
        size = size + h.double().abs()[:, None] * (2 * lp_all.abs() + math.log(V) + 4)
    dG = p * size * (rel + 3 * U * (lp_all.abs() + 20) + 12 * U) + HALF * HALF * G.abs()
    if entropy:  # the row's entropy in the factor: its own error
        dG = dG + p * h.double().abs()[:, None] * 2 * rel * (math.log(V) + 2)
    dG.scatter_add_(1, ids[:, None], 4 * U * g.double().abs()[:, None])
    flat, wd = hidden.double(), weight.double()
    N = flat.shape[0]
    want = G.T @ flat
    bound = HALF * want.abs() + (1 + HALF) * (dG.T @ flat.abs() + 2 * N * U * (G.abs().T @ flat.abs())) + 1e-37
    off = (dw.double() - want).abs() - bound
    assert (off <= 0).all(), float(off.max())
    want = G @ wd
    bound = HALF * want.abs() + (1 + HALF) * (dG @ wd.abs() + 2 * V * U * (G.abs() @ wd.abs())) + 1e-37
    off = (dh.double() - want).abs() - bound
    assert (off <= 0).all(), float(off.max())
    if not entropy:  # nobody chose these tokens: their rows of d weight are 0 but for the errors
        free = torch.ones(V, dtype=torch.bool, device=ids.device)
        free[ids] = False
        assert free.any() and float((G.T @ flat)[free].abs().max()) <= 1e-12
