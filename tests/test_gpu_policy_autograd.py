"""GPU: what autograd may ask of ``genrec_amd.policy`` besides a gradient: a second derivative is refused however it is
reached, and so is a derivative in forward mode; the statistics of a loss are the caller's."""

import pytest
import torch
import torch.autograd.forward_ad as forward_ad

from genrec_amd.policy import lm_head_token_logps, policy_loss, token_logps

pytestmark = pytest.mark.gpu


def _logits(B=4, T=5, V=301, seed=1):
    dev = torch.device("cuda", 0)
    gen = torch.Generator(device=dev).manual_seed(seed)
    x = torch.randn((B, T, V), generator=gen, device=dev, requires_grad=True)
    return x, torch.randint(0, V, (B, T), generator=gen, device=dev), torch.randn((B,), generator=gen, device=dev)


def _head(N=40, H=128, V=301, seed=2):
    dev = torch.device("cuda", 0)
    gen = torch.Generator(device=dev).manual_seed(seed)
    h = torch.randn((N, H), generator=gen, device=dev).to(torch.bfloat16).requires_grad_()
    w = (torch.randn((V, H), generator=gen, device=dev) * 0.1).to(torch.bfloat16).requires_grad_()
    return h, w, torch.randint(0, V, (N,), generator=gen, device=dev)


def _first(kind):
    """(a value, its leaves)"""
    if kind == "logits":
        x, ids, _ = _logits()
        return token_logps(x, ids).sum(), [x]
    if kind == "entropy":
        x, ids, _ = _logits()
        return token_logps(x, ids, return_entropy=True)[1].sum(), [x]
    if kind == "loss":
        x = torch.zeros((4, 5), device="cuda", requires_grad=True)
        return policy_loss(x, torch.ones(4, device="cuda"), torch.ones((4, 5), device="cuda")).loss, [x]
    if kind == "loss of logits":
        x, ids, adv = _logits()
        return policy_loss(token_logps(x, ids), adv, torch.ones_like(ids)).loss, [x]
    h, w, ids = _head()
    if kind == "head":
        return lm_head_token_logps(h, w, ids).sum(), [h, w]
    return lm_head_token_logps(h, w.detach(), ids).sum(), [h]


KINDS = ["logits", "entropy", "loss", "loss of logits", "head", "head, frozen weight"]


@pytest.mark.parametrize("kind", KINDS)
def test_second_derivative_of_a_plain_sum_is_refused(kind):
    """The incoming gradient is a constant, and the result still depends on the leaves."""
    value, leaves = _first(kind)
    first = torch.autograd.grad(value, leaves, create_graph=True)
    for d in first:
        assert d.requires_grad
        with pytest.raises(RuntimeError, match="differentiate twice"):
            torch.autograd.grad(d.float().pow(2).sum(), leaves, retain_graph=True)
        with pytest.raises(RuntimeError, match="differentiate twice"):
            torch.autograd.grad(d.float().pow(2).sum(), leaves, retain_graph=True, allow_unused=True)
    with pytest.raises(RuntimeError, match="differentiate twice"):  # a penalty on the gradient, beside the loss
        (value + sum(d.float().pow(2).sum() for d in first)).backward()


@pytest.mark.parametrize("kind", KINDS)
def test_a_graph_of_the_gradient_changes_nothing_else(kind):
    value, leaves = _first(kind)
    want = torch.autograd.grad(value, leaves, retain_graph=True)
    got = torch.autograd.grad(value, leaves, create_graph=True)
    assert all(torch.equal(a, b) for a, b in zip(want, got))
    assert not any(d.requires_grad for d in want)
    for d in got:  # a constant made of it is fine
        assert not d.detach().requires_grad and torch.isfinite(d.detach().float()).all()


def test_second_derivative_with_respect_to_the_incoming_gradient_is_refused():
    x, ids, _ = _logits()
    lp = token_logps(x, ids)
    g = torch.ones_like(lp).requires_grad_()
    (d,) = torch.autograd.grad(lp, x, g, create_graph=True)
    with pytest.raises(RuntimeError, match="differentiate twice"):
        torch.autograd.grad(d.sum(), g)


@pytest.mark.parametrize("grad", [True, False])
@pytest.mark.parametrize("kind", ["logits", "logits, transposed vocabulary", "hidden", "weight", "loss"])
def test_forward_mode_is_refused(kind, grad):
    """A dual tensor must not come back without its tangent, whether a gradient is recorded or not."""
    x, ids, adv = (t.detach() for t in _logits())
    h, w, tokens = (t.detach() for t in _head())

    def call(t):
        if kind == "logits":
            return token_logps(t(x), ids, return_entropy=True)
        if kind == "logits, transposed vocabulary":
            return token_logps(t(x.transpose(1, 2)).transpose(1, 2), ids)
        if kind == "hidden":
            return lm_head_token_logps(t(h), w, tokens)
        if kind == "weight":
            return lm_head_token_logps(h, t(w), tokens)
        return policy_loss(t(x[..., 0].contiguous()), adv, torch.ones_like(ids)).loss

    call(lambda t: t)  # the same call without a tangent
    with forward_ad.dual_level(), torch.set_grad_enabled(grad):
        with pytest.raises((RuntimeError, NotImplementedError), match="jvp"):
            call(lambda t: forward_ad.make_dual(t, torch.ones_like(t)))


@pytest.mark.parametrize("kind", ["grpo", "bnpo"])  # the gradient's factor known beforehand, and only at the end
def test_statistics_may_be_written_over_before_the_backward_pass(kind):
    gen = torch.Generator(device="cuda").manual_seed(3)
    old = torch.randn((30, 7), generator=gen, device="cuda") - 2
    mask = torch.ones_like(old)
    mask[::3, 4:] = 0

    def step():
        x = (old + 0.3).requires_grad_()
        return x, policy_loss(x, torch.ones(30, device="cuda"), mask, old, old, beta=0.1, loss_type=kind)

    x, res = step()
    (want,) = torch.autograd.grad(res.loss, x)
    values = res.kl.clone(), res.clip_low.clone(), res.clip_high.clone()
    x, res = step()
    res.kl.div_(2)
    res.clip_low.fill_(9)
    res.clip_high.neg_()
    assert torch.equal(res.kl, values[0] / 2) and torch.equal(res.clip_high, -values[2]) and float(res.clip_low) == 9
    (got,) = torch.autograd.grad(res.loss, x)
    assert torch.equal(got, want)
    with torch.inference_mode():
        assert torch.equal(step()[1].kl, values[0])


@pytest.mark.parametrize("L,T", [(6, 5), (40, 5), (17, 16)])
def test_whole_logits_with_padding_where_a_slice_would_cut(L, T):
    """The same log-probabilities and gradient as from the slice: two runs of a row differ by the order of its sums, twice
    (V / 256 + 160) u of a probability, and by 8 u of what is multiplied with it."""
    B, V = 6, 1003
    x, _, _ = _logits(B, L, V)
    ids = torch.randint(0, V, (B, T), device=x.device)
    ids[0, 2:] = -1
    g = torch.randn((B, T), device=x.device)
    cut = token_logps(x[:, -T - 1 : -1], ids)
    every = ids.new_full((B, L), -1)
    every[:, -T - 1 : -1] = ids
    whole = token_logps(x, every)[:, -T - 1 : -1]
    bound = (2 * (V / 256 + 160) + 12) * 2.0 ** -24
    assert ((cut - whole).abs() <= bound + 2.0 ** -23 * cut.abs()).all()
    (want,), (got,) = torch.autograd.grad(cut, x, g), torch.autograd.grad(whole, x, g)
    assert (got[:, : L - T - 1] == 0).all() and (got[:, -1] == 0).all()
    off = (got - want).abs()[:, -T - 1 : -1]
    assert (off <= bound * 2 * g.abs()[..., None]).all()


@pytest.mark.parametrize("keep_bytes", [8 << 30, 0])
def test_entropies_alone_and_other_integer_types(keep_bytes):
    """No gradient of the log-probabilities is a gradient of 0; token ids of any integer type are the same tokens."""
    h, w, ids = _head()
    ids[::5] = -1
    g = torch.randn(ids.shape, device=ids.device)
    lp, ent = lm_head_token_logps(h, w, ids, 0.9, True, keep_bytes)
    want = torch.autograd.grad([lp, ent], [h, w], [torch.zeros_like(g), g], retain_graph=True)
    got = torch.autograd.grad(ent, [h, w], g, retain_graph=True)
    assert all(torch.equal(a, b) for a, b in zip(got, want)) and got[1].any()
    half = torch.autograd.grad(lp[::2], [h, w], g[::2], retain_graph=True)  # an incoming gradient with gaps
    some = torch.where(torch.arange(ids.numel(), device=ids.device) % 2 == 0, g, 0.0)
    assert all(torch.equal(a, b) for a, b in zip(half, torch.autograd.grad(lp, [h, w], some)))
    for kind in (torch.int32, torch.int16):
        assert torch.equal(lm_head_token_logps(h, w, ids.to(kind), 0.9, keep_bytes=keep_bytes), lp)


@pytest.mark.parametrize("shape", [(5, 1), (1, 1), (1, 4097), (4097, 1), (3, 1025)])
def test_advantages_of_single_positions_and_rows(shape):
    """[R, T] and [R] say the same where a row's advantages are equal, at the borders between the kernels."""
    gen = torch.Generator(device="cuda").manual_seed(4)
    x = (torch.randn(shape, generator=gen, device="cuda") - 2).requires_grad_()
    old = x.detach() + 0.1 * torch.randn(shape, generator=gen, device="cuda")
    adv = torch.randn(shape[:1], generator=gen, device="cuda")
    mask = torch.ones(shape, device="cuda")
    for level in ("token", "sequence"):
        made = []
        for a in (adv, adv[:, None].expand(shape), adv[:, None].expand(shape).contiguous()):
            loss = policy_loss(x, a, mask, old, importance_sampling_level=level).loss
            made.append((loss.detach(), torch.autograd.grad(loss, x)[0]))
        assert all(torch.equal(p, q) for m in made[1:] for p, q in zip(m, made[0]))
