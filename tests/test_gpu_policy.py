"""GPU: log-probabilities of tokens and the clipped policy loss (``genrec_amd.policy``), against their definitions
in 64 bits, in both directions.

Tolerances.  u = 2^-24 is fp32's rounding.  A row's sum of V exponentials is added up by at least 256 threads and
joined over a tree: relative error at most (V / 256 + 64) u.  The argument (x - m) log2(e) / T of an exponential of
weight w carries at most 3 roundings: |t| 3 u ln 2, and 2^t |t| <= 2^t 24 + 2^-20 for any t, so the sum is off by
at most another 64 u; the exponential itself by 2 u.  All of it together: ``_row_rel(V)``.  A gradient element is
such an exponential over the sum times fp32 factors, rounded once to its type (half a step, eps / 2)."""

import math

import pytest
import torch

from genrec_amd.policy import policy_loss, token_logps

pytestmark = pytest.mark.gpu

U = 2.0 ** -24
DTYPES = [torch.float32, torch.bfloat16, torch.float16]


def _row_rel(V):
    return (V / 256 + 160) * U


def _definition(logits, ids, temperature, g=None, h=None):
    """(logps, entropy, gradient of the logits) in 64 bits; rows with a negative id give 0."""
    shape = ids.shape
    V = logits.shape[-1]
    x = logits.double().reshape(-1, V) / temperature
    t = ids.reshape(-1)
    use = t >= 0
    at = t.clamp(min=0)[:, None]
    # the maximum is taken out first: max + log(sum) rounds the logarithm away beside a row of 3e38
    x = x - x.detach().max(1, keepdim=True).values
    lp = x - x.exp().sum(1, keepdim=True).log()
    p = lp.exp()
    plp = torch.where(p > 0, p * lp, torch.zeros_like(p))
    logps = torch.where(use, lp.gather(1, at)[:, 0], 0.0)
    ent = torch.where(use, -plp.sum(1), 0.0)
    grad = None
    if g is not None or h is not None:
        gg = torch.zeros_like(logps) if g is None else g.double().reshape(-1)
        hh = torch.zeros_like(logps) if h is None else h.double().reshape(-1)
        d = -p * gg[:, None] - hh[:, None] * (plp + p * ent[:, None])
        d.scatter_add_(1, at, gg[:, None])
        grad = (torch.where(use[:, None], d, 0.0) / temperature).reshape(logits.shape)
    return logps.reshape(shape), ent.reshape(shape), grad


def _check(logits, ids, temperature=1.0, entropy=True, g=None, h=None, seed=0):
    dev = logits.device
    gen = torch.Generator(device=dev).manual_seed(seed)
    if g is None:
        g = torch.randn(ids.shape, generator=gen, device=dev)
    if h is None and entropy:
        h = torch.randn(ids.shape, generator=gen, device=dev) * 0.3
    x = logits.detach().requires_grad_()
    made = token_logps(x, ids, temperature, return_entropy=entropy)
    logps, ent = made if entropy else (made, None)
    assert logps.dtype == torch.float32 and logps.shape == ids.shape
    (grad,) = torch.autograd.grad([logps] + ([ent] if entropy else []), x, [g] + ([h] if entropy else []))
    want, want_ent, want_grad = _definition(logits, ids, temperature, g, h if entropy else None)
    V = logits.shape[-1]
    rel = _row_rel(V)
    assert ((logps.double() - want).abs() <= rel + 6 * U * want.abs()).all()
    if entropy:  # log2 of the sum, and a weighted sum of t over it: |t| averages below log2(V) + 2
        assert ((ent.double() - want_ent).abs() <= 2 * rel * (math.log(V) + 2)).all()
    assert grad.shape == logits.shape and grad.dtype == logits.dtype
    eps = torch.finfo(logits.dtype).eps / 2
    size = (g.double().abs() + (h.double().abs() * (3 * math.log(V) + 8) if entropy else 0.0)) / temperature
    lp_all = logits.double() / temperature
    lp_all = lp_all - lp_all.max(-1, keepdim=True).values
    lp_all = lp_all - lp_all.exp().sum(-1, keepdim=True).log()
    p = lp_all.exp()
    hit = torch.zeros_like(p).scatter_(-1, ids.clamp(min=0)[..., None], 1.0)
    # |t| of an element with weight p is up to -log2 p + log2 V: its own argument error, on top of the row's
    arg = 3 * U * (torch.where(p > 0, -lp_all, torch.zeros_like(p)) + math.log(V) + 2)
    spread = p * (rel + arg + 8 * U) * size[..., None] * 2 + hit * 4 * U * size[..., None]
    if entropy:  # the entropy's slope grows with |log p|
        spread = spread + p * torch.where(p > 0, -lp_all, torch.zeros_like(p)) * (rel + arg) * 2 * (h.double().abs() / temperature)[..., None]
    tiny = torch.finfo(logits.dtype).tiny * eps * 2 + 2.0 ** -126
    off = (grad.double() - want_grad).abs()
    bound = spread * (1 + eps) + eps * want_grad.abs() + tiny
    assert (off <= bound).all(), float((off - bound).max())
    return logps, ent, grad


def _case(shape, V, dtype, seed, scale=3.0, pad=0.2):
    dev = torch.device("cuda", 0)
    g = torch.Generator(device=dev).manual_seed(seed)
    logits = (torch.randn((*shape, V), generator=g, device=dev) * scale).to(dtype)
    ids = torch.randint(0, V, shape, generator=g, device=dev)
    ids[torch.rand(shape, generator=g, device=dev) < pad] = -1
    return logits, ids


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("shape,V", [((1,), 1), ((1, 1), 2), ((3,), 7), ((2, 3), 8), ((5, 4), 63), ((3, 2), 1001),
                                     ((2, 5), 4096), ((7, 3), 8191), ((1, 2), 152640), ((3, 1), 151669)])
def test_logps_and_gradient(shape, V, dtype):
    logits, ids = _case(shape, V, dtype, seed=V)
    for temperature in (1.0, 0.7):
        _check(logits, ids, temperature, entropy=True, seed=V)
    _check(logits, ids, 1.3, entropy=False, seed=V + 1)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("rows,V", [(2500, 517), (9, 33003), (130, 40001), (400, 33003)])
def test_rows_whole_and_split(rows, V, dtype):
    """Many rows (one workgroup each) and few (several workgroups each)."""
    _check(*_case((rows,), V, dtype, seed=rows), seed=rows)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
def test_strided_logits(dtype):
    """Views: positions cut off, rows that start at any element, an expanded row, a transposed vocabulary."""
    buf, _ = _case((4, 6), 1003, dtype, seed=1)
    ids = torch.randint(0, 900, (4, 5), device=buf.device)
    for view in (buf[:, :-1], buf[:, 1:, 1:902], buf[:1, 1:].expand(4, 5, 1003), buf[::2, 1:].repeat(2, 1, 1)[:, :, 3:]):
        use = ids.clamp(max=view.shape[-1] - 1)
        got = token_logps(view, use)
        assert torch.equal(got, token_logps(view.contiguous(), use)) or (
            (got - token_logps(view.contiguous(), use)).abs().max() <= 2 * _row_rel(1003))
        _check(view, use)
    swapped = buf.reshape(-1, 1003).t().contiguous().t()  # last dimension not contiguous
    _check(swapped, torch.randint(0, 1003, (24,), device=buf.device))
    wide = torch.randint(0, 1003, (4, 10), device=buf.device)[:, ::2]  # strided ids, int32 ids
    assert torch.equal(token_logps(buf[:, :5], wide), token_logps(buf[:, :5], wide.to(torch.int32)))


@pytest.mark.parametrize("dtype", DTYPES)
def test_masked_vocabulary_and_extreme_rows(dtype):
    dev = torch.device("cuda", 0)
    V = 2050
    low = torch.finfo(dtype).min
    logits, ids = _case((6, 2), V, dtype, seed=3, pad=0.0)
    logits[0, :, 100:] = -math.inf                    # most of the vocabulary masked
    ids[0] = torch.tensor([5, 500])                   # the second token is a masked one
    logits[1] = low                                   # a row at the type's lowest value: uniform
    logits[2, :, :-1] = low
    logits[2, :, -1] = 0.0
    ids[2] = V - 1
    logits[3, :, 7] = 300.0 if dtype != torch.float16 else 60000.0  # one token takes everything
    ids[3] = torch.tensor([7, 8])
    logits[4, 1] = -math.inf                          # nothing is allowed: no log-probability
    logits[5, 0, 9] = math.nan
    x = logits.clone().requires_grad_()
    lp, ent = token_logps(x, ids, return_entropy=True)
    want, want_ent, _ = _definition(logits, ids, 1.0)
    assert lp[0, 1] == -math.inf and torch.isnan(lp[4, 1]) and torch.isnan(lp[5, 0])
    assert torch.isnan(ent[4, 1]) and torch.isnan(ent[5, 0])
    keep = torch.isfinite(want)
    assert ((lp - want).abs()[keep] <= (_row_rel(V) + 6 * U * want.abs())[keep]).all()
    assert abs(float(lp[1, 0]) + math.log(V)) <= _row_rel(V) + 6 * U * 8
    assert ((ent - want_ent).abs()[keep] <= 2 * _row_rel(V) * 10).all()
    g = torch.ones_like(lp)
    g[4, 1] = g[5, 0] = 0.0                           # the loss leaves those two out: gradient 0, not NaN
    (grad,) = torch.autograd.grad(lp, x, g)
    assert torch.isfinite(grad).all() and (grad[4, 1] == 0).all() and (grad[5, 0] == 0).all()
    assert (grad[0, 0, 100:] == 0).all() and float(grad[0, 1, 500]) == 1.0
    sums = grad.double().sum(-1)                      # a row's gradient adds up to 0 unless the token is masked
    assert sums[1:4].abs().max() <= V * 2 * torch.finfo(dtype).eps and abs(float(sums[0, 0])) <= 200 * torch.finfo(dtype).eps
    # entropies are smooth there too
    (grad,) = torch.autograd.grad(token_logps(x, ids, return_entropy=True)[1], x, g)
    assert torch.isfinite(grad).all()


def test_padding_is_not_read_and_bad_ids_are_nan():
    dev = torch.device("cuda", 0)
    logits = torch.randn((3, 2, 515), device=dev)
    logits[0] = math.nan
    ids = torch.tensor([[-1, -100], [4, 515], [514, 1 << 40]], device=dev)
    x = logits.clone().requires_grad_()
    lp, ent = token_logps(x, ids, return_entropy=True)
    assert (lp[0] == 0).all() and (ent[0] == 0).all()
    assert torch.isnan(lp[1, 1]) and torch.isnan(lp[2, 1]) and torch.isfinite(lp[1, 0]) and torch.isfinite(lp[2, 0])
    (grad,) = torch.autograd.grad(lp, x, torch.ones_like(lp))
    assert (grad[0] == 0).all() and torch.isfinite(grad[1, 0]).all() and torch.isnan(grad[1, 1, 0])
    for shape in ((0, 4), (4, 0)):
        e = torch.zeros((*shape, 515), device=dev, requires_grad=True)
        out = token_logps(e, torch.zeros(shape, dtype=torch.int64, device=dev))
        assert out.shape == shape
        out.sum().backward()
        assert e.grad.shape == e.shape


def test_gradient_against_differences():
    """Central differences of the definition in 64 bits at a few elements, step 1e-4: the cut-off of the third
    derivative is below 1e-8, far inside the tolerance of the gradient itself."""
    logits, ids = _case((2, 2), 37, torch.float32, seed=8, pad=0.0)
    g = torch.tensor([[0.5, -1.0], [2.0, 0.25]], device=logits.device)
    h = torch.tensor([[0.1, 0.3], [-0.2, 0.0]], device=logits.device)
    x = logits.clone().requires_grad_()
    lp, ent = token_logps(x, ids, 0.8, return_entropy=True)
    (grad,) = torch.autograd.grad([lp, ent], x, [g, h])

    def value(z):
        a, b, _ = _definition(z, ids, 0.8)
        return float((a * g).sum() + (b * h).sum())

    for at in [(0, 0, int(ids[0, 0])), (0, 1, 3), (1, 0, int(ids[1, 0])), (1, 1, 36), (1, 0, 0)]:
        up, down = logits.double(), logits.double()
        up[at] += 1e-4
        down[at] -= 1e-4
        slope = (value(up) - value(down)) / 2e-4
        assert abs(float(grad[at]) - slope) <= 1e-6 + 4 * _row_rel(37) * 10


def test_what_autograd_may_ask():
    """One of two outputs, a graph kept for a second backward, a second derivative refused, no graph at all."""
    logits, ids = _case((6, 5), 701, torch.float32, seed=31)
    x = logits.clone().requires_grad_()
    lp, ent = token_logps(x, ids, return_entropy=True)
    g = torch.randn_like(lp)
    (a,) = torch.autograd.grad(lp, x, g, retain_graph=True)
    (b,) = torch.autograd.grad(ent, x, g, retain_graph=True)
    (both,) = torch.autograd.grad([lp, ent], x, [g, g], retain_graph=True)
    want = [_definition(logits, ids, 1.0, *w)[2] for w in ((g, None), (None, g), (g, g))]
    bound = (_row_rel(701) + 32 * U) * 8 * (3 * math.log(701) + 8) * float(g.abs().max())  # as _check, for the largest p = 1
    for got, w in zip((a, b, both), want):
        assert float((got.double() - w).abs().max()) <= bound
    (again,) = torch.autograd.grad(lp, x, g)
    assert torch.equal(a, again)
    lp = token_logps(x, ids)
    (d,) = torch.autograd.grad(lp, x, torch.ones_like(lp).requires_grad_(), create_graph=True)
    with pytest.raises(RuntimeError, match="differentia"):
        torch.autograd.grad(d.sum(), x)
    loss = policy_loss(lp, torch.ones(6, device=x.device), torch.ones_like(lp)).loss
    (d,) = torch.autograd.grad(loss, lp, torch.ones_like(loss).requires_grad_(), create_graph=True)
    with pytest.raises(RuntimeError, match="differentia"):
        d.sum().backward()
    with torch.no_grad():
        assert not token_logps(x, ids).requires_grad
        assert not policy_loss(lp, torch.ones(6, device=x.device), torch.ones_like(lp)).loss.requires_grad
    with torch.inference_mode():
        assert torch.equal(token_logps(x, ids), lp)


def test_more_rows_than_one_launch_and_offsets_past_32_bits():
    """2^23 rows of 4104: the gradient takes more workgroups than a launch may have, and 69 GB."""
    dev = torch.device("cuda", 0)
    if torch.cuda.mem_get_info(dev)[0] < 90 << 30:
        pytest.skip("needs 90 GB of free memory")
    N, V = 1 << 23, 4104
    g = torch.Generator(device=dev).manual_seed(33)
    one = (torch.randn((1, V), generator=g, device=dev) * 3).to(torch.bfloat16)
    x = one.expand(N, V).detach().requires_grad_()
    ids = torch.randint(0, V, (N,), generator=g, device=dev)
    rows = torch.tensor([0, 1, 77, 4194303, 4194304, 8388606, 8388607], device=dev)
    up = torch.zeros(N, device=dev)
    up[rows] = torch.randn(rows.shape, generator=g, device=dev)
    lp = token_logps(x, ids)
    (grad,) = torch.autograd.grad(lp, x, up)
    want, _, _ = _definition(one.expand(rows.numel(), V), ids[rows], 1.0)
    assert ((lp[rows].double() - want).abs() <= _row_rel(V) + 6 * U * want.abs()).all()
    _, _, d = _check(one.expand(rows.numel(), V), ids[rows], entropy=False, g=up[rows])
    assert torch.equal(grad[rows], d)
    assert not grad[2:77].any() and not grad[4194305:4194400].any() and not grad[8388500:8388606].any()
    far = grad[:: 1 << 22]  # rows 2^22 apart: 1.7e10 elements
    far.copy_((torch.randn((2, V), generator=g, device=dev) * 3).to(torch.bfloat16))
    _check(far, torch.tensor([5, 4103], device=dev))


def test_called_on_a_stream_of_its_own():
    """The call follows the current stream, and its backward pass the stream of the call."""
    logits, ids = _case((300, 4), 20011, torch.bfloat16, seed=35)
    g = torch.randn(ids.shape, device=logits.device)
    x = logits.clone().requires_grad_()
    want = torch.autograd.grad(token_logps(x, ids), x, g)[0]
    side = torch.cuda.Stream()
    for _ in range(3):
        y = logits.detach().requires_grad_()
        side.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(side):
            lp = token_logps(y, ids)
        torch.cuda.current_stream().wait_stream(side)
        (got,) = torch.autograd.grad(lp, y, g)  # called with another stream current
        assert torch.equal(got, want)


# ---- the loss ------------------------------------------------------------------------------------------------


def _loss_definition(logps, adv, mask, old=None, ref=None, low=0.2, high=0.2, delta=None, beta=0.0, kind="grpo",
                     level="token", length=None, items=None):
    x = logps.detach().double().requires_grad_()
    m = mask > 0
    md = m.double()
    n = md.sum(1)
    o = x.detach() if old is None else old.double()
    d = torch.where(m, x - torch.where(m, o, torch.zeros_like(o)), torch.zeros_like(x))
    if level == "sequence":
        d = (d.sum(1) / n.clamp(min=1))[:, None].expand_as(x)
    w = d.exp()
    A = adv.double() if adv.dim() == 2 else adv.double()[:, None]
    A = torch.where(m, A.expand_as(x), torch.zeros_like(x))
    first = (w if delta is None else w.clamp(max=delta)) * A
    second = w.clamp(1 - low, 1 + high) * A
    tok = -torch.min(first, second)
    kl = torch.zeros_like(x)
    if ref is not None:
        q = torch.where(m, torch.where(m, ref.double(), torch.zeros_like(x)) - x, torch.zeros_like(x))
        kl = q.exp() - 1 - q
    tok = torch.where(m, tok + beta * kl, torch.zeros_like(x))
    total = md.sum().clamp(min=1)
    loss = {"grpo": lambda: (tok.sum(1) / n.clamp(min=1)).sum() / max(1, x.shape[0]), "bnpo": lambda: tok.sum() / total,
            "dr_grpo": lambda: tok.sum() / (x.shape[0] * length), "dapo": lambda: tok.sum() / items}[kind]()
    (grad,) = torch.autograd.grad(loss, x)
    weight = {"grpo": md / n.clamp(min=1)[:, None] / max(1, x.shape[0]), "bnpo": md / total,
              "dr_grpo": md / (x.shape[0] * (length or 1)), "dapo": md / (items or 1)}[kind]
    size = (torch.where(m, w.abs() * A.abs(), torch.zeros_like(x)) + abs(beta) * (kl + 1)).detach() * weight
    return dict(loss=loss.detach(), grad=grad, kl=(kl.detach() * md).sum() / total, clip_low=((w < 1 - low) & (A < 0) & m).sum() / total,
                clip_high=((w > 1 + high) & (A > 0) & m).sum() / total, size=size, n=n)


def _loss_inputs(R, T, seed, tokenwise=False, mask_dtype=torch.int64, spread=0.2):
    dev = torch.device("cuda", 0)
    g = torch.Generator(device=dev).manual_seed(seed)
    lengths = torch.randint(0, T + 1, (R, 1), generator=g, device=dev)
    mask = (torch.arange(T, device=dev)[None] < lengths).to(mask_dtype)
    logps = -torch.rand((R, T), generator=g, device=dev) * 3
    old = logps + spread * torch.randn((R, T), generator=g, device=dev)
    ref = logps + 0.4 * torch.randn((R, T), generator=g, device=dev)
    adv = torch.randn((R, T) if tokenwise else (R,), generator=g, device=dev)
    return logps, adv, mask, old, ref


def _check_loss(logps, adv, mask, old=None, ref=None, upstream=None, **o):
    x = logps.detach().requires_grad_()
    res = policy_loss(x, adv, mask, old, ref, epsilon_low=o.get("low", 0.2), epsilon_high=o.get("high"), delta=o.get("delta"),
                      beta=o.get("beta", 0.0), loss_type=o.get("kind", "grpo"), importance_sampling_level=o.get("level", "token"),
                      max_completion_length=o.get("length"), num_items=o.get("items"))
    o["high"] = o.get("low", 0.2) if o.get("high") is None else o["high"]
    want = _loss_definition(logps, adv, mask, old, ref, **o)
    # a term: differences exact in 64 bits and rounded once, exp within 2 u, three products, the KL series within
    # 16 u of it: 24 u of the term's size; sums are 64-bit
    total = want["size"].sum()
    assert abs(float(res.loss.double() - want["loss"])) <= 24 * U * float(total) + U * abs(float(want["loss"])) + 1e-38
    (grad,) = torch.autograd.grad(res.loss, x, upstream)
    f = 1.0 if upstream is None else float(upstream)
    per = want["size"]
    if o.get("level") == "sequence":  # every token carries the row's sum
        per = per + per.sum(1, keepdim=True)
    off = (grad.double() - want["grad"] * f).abs()
    assert (off <= 28 * U * (per * abs(f)) + 1e-38).all(), float((off - 28 * U * per).max())
    assert (grad[mask <= 0] == 0).all()
    assert abs(float(res.kl.double() - want["kl"])) <= 16 * U * float(want["kl"]) + 1e-12
    assert abs(float(res.clip_low.double() - want["clip_low"])) <= 2 * U
    assert abs(float(res.clip_high.double() - want["clip_high"])) <= 2 * U
    assert not res.kl.requires_grad and not res.clip_low.requires_grad
    return res, grad


@pytest.mark.parametrize("R,T", [(1, 1), (3, 5), (64, 5), (7, 8), (5, 9), (33, 64), (16, 131), (900, 6), (200, 65),
                                 (2, 2049), (1, 5000), (3000, 33)])
@pytest.mark.parametrize("kind", ["grpo", "bnpo", "dr_grpo", "dapo"])
def test_loss_and_gradient(R, T, kind):
    for i, (level, tokenwise) in enumerate([("token", False), ("token", True), ("sequence", False), ("sequence", True)]):
        logps, adv, mask, old, ref = _loss_inputs(R, T, seed=R * 31 + T + i, tokenwise=tokenwise)
        beta = 0.04 * (i % 2)
        _check_loss(logps, adv, mask, old, ref if beta else None, kind=kind, level=level, beta=beta, high=0.28,
                    delta=1.5 if i >= 2 else None, length=T + 2, items=R * T * 0.5, upstream=torch.tensor(0.37, device=logps.device))


@pytest.mark.parametrize("mask_dtype", [torch.bool, torch.uint8, torch.int32, torch.int64, torch.float32, torch.float64, torch.int16])
def test_mask_types_and_strides(mask_dtype):
    logps, adv, mask, old, ref = _loss_inputs(6, 24, seed=5, tokenwise=True, mask_dtype=mask_dtype)
    _check_loss(logps, adv, mask, old, ref, beta=0.1)
    wide = torch.randn((6, 40), device=logps.device)
    views = [t.clone() for t in (wide, wide, wide)]
    for v, t in zip(views, (logps, old, ref)):
        v[:, 3:27] = t
    want, g = _check_loss(logps, adv, mask, old, ref, beta=0.1)
    m = torch.zeros((6, 31), dtype=mask_dtype, device=mask.device)
    m[:, 7:] = mask
    A = torch.randn((24, 6), device=logps.device)
    A.copy_(adv.t())
    got, g2 = _check_loss(views[0][:, 3:27], A.t(), m[:, 7:], views[1][:, 3:27], views[2][:, 3:27], beta=0.1)
    assert torch.equal(g, g2) and torch.equal(got.loss, want.loss)
    _check_loss(logps[:, ::2], adv[:, ::2], mask[:, ::2], old[:, ::2], None)


def test_first_step_reference_only_and_no_gradient():
    """No old policy: ratio 1, the gradient is that of -A logp; a reference without beta is reported, not added."""
    logps, adv, mask, old, ref = _loss_inputs(8, 12, seed=6)
    for level in ("token", "sequence"):
        _check_loss(logps, adv, mask, None, ref, beta=0.2, level=level)
    a, _ = _check_loss(logps, adv, mask, old, ref)
    b, _ = _check_loss(logps, adv, mask, old, None)
    assert torch.equal(a.loss, b.loss) and float(a.kl) > 0 and float(b.kl) == 0
    res = policy_loss(logps, adv, mask, old)
    assert not res.loss.requires_grad and torch.equal(res.loss, b.loss)
    half = policy_loss(logps.to(torch.bfloat16).requires_grad_(), adv, mask, old)
    half.loss.backward()


def test_nothing_valid_and_garbage_behind_the_mask():
    dev = torch.device("cuda", 0)
    for kind in ("grpo", "bnpo", "dr_grpo", "dapo"):
        logps, adv, mask, old, ref = _loss_inputs(5, 11, seed=7)
        _check_loss(logps, adv, torch.zeros_like(mask), old, ref, beta=0.1, kind=kind, length=11, items=3)
        want, g = _check_loss(logps, adv, mask, old, ref, beta=0.1, kind=kind, length=11, items=3)
        for bad in (math.nan, math.inf, -math.inf, torch.finfo(torch.float32).min):
            dirty = [torch.where(mask > 0, t, torch.full_like(t, bad)) for t in (logps, old, ref)]
            got, g2 = _check_loss(dirty[0], adv, mask, dirty[1], dirty[2], beta=0.1, kind=kind, length=11, items=3)
            assert torch.equal(got.loss, want.loss) and torch.equal(g, g2)
    for shape in ((0, 4), (4, 0), (0, 0)):
        x = torch.zeros(shape, device=dev, requires_grad=True)
        res = policy_loss(x, torch.zeros(shape[0], device=dev), torch.ones(shape, device=dev))
        res.loss.backward()
        assert float(res.loss) == 0.0 and x.grad.shape == shape


def test_bounds_and_extreme_ratios():
    """Ratios right next to a bound, exactly at it, far outside, and an overflowing one whose clipped term wins."""
    dev = torch.device("cuda", 0)
    hi, lo = math.log1p(0.2), math.log1p(-0.2)
    d = []
    for b in (hi, lo, math.log(1.5)):
        f = torch.tensor(b, dtype=torch.float32)
        d += [f, torch.nextafter(f, torch.tensor(9.0)), torch.nextafter(f, torch.tensor(-9.0))]
    d = torch.stack(d + [torch.tensor(v, dtype=torch.float32) for v in (0.0, 5.0, -5.0, 60.0, -90.0)]).to(dev)
    for sign in (1.0, -1.0):
        logps = d[None].clone()
        _check_loss(logps, torch.full((1,), sign, device=dev), torch.ones_like(logps), torch.zeros_like(logps), delta=1.5)
        _check_loss(logps, torch.full((1,), sign, device=dev), torch.ones_like(logps), torch.zeros_like(logps))
    x = torch.tensor([[200.0]], device=dev, requires_grad=True)
    res = policy_loss(x, torch.ones(1, device=dev), torch.ones_like(x), torch.zeros_like(x))
    res.loss.backward()
    assert float(res.loss) == pytest.approx(-1.2, abs=1e-6) and float(x.grad) == 0.0


@pytest.mark.parametrize("kind,level", [("grpo", "token"), ("bnpo", "sequence"), ("dapo", "token")])
def test_loss_gradient_against_differences(kind, level):
    """A step of h = 2^-6 either way, away from the bounds (|d| < 0.15 + h): off by h^2 / 6 of the third derivative
    (|w A| + beta e^q, below 3 here with its weight below 1) and by the rounding of two losses, 24 u of their size each."""
    logps, adv, mask, old, ref = _loss_inputs(3, 9, seed=23)
    old = logps + (old - logps).clamp(-0.15, 0.15)
    mask[:, 0] = 1
    o = dict(beta=0.1, loss_type=kind, importance_sampling_level=level, num_items=20)
    x = logps.clone().requires_grad_()
    (grad,) = torch.autograd.grad(policy_loss(x, adv, mask, old, ref, **o).loss, x)
    size = float((adv.abs().max() * 1.2 + 0.1 * 8))
    h = 2.0 ** -6
    for r, t in ((0, 0), (1, 0), (2, 0), (0, 4), (1, 3), (2, 8)):
        up, down = logps.clone(), logps.clone()
        up[r, t] += h
        down[r, t] -= h
        a, b = (float(policy_loss(v, adv, mask, old, ref, **o).loss) for v in (up, down))
        step = float(up[r, t].double() - down[r, t].double())
        assert abs((a - b) / step - float(grad[r, t])) <= h * h / 6 * size * 1.1 + 2 * 24 * U * 2 * size / step


def test_rows_without_positions_read_nothing():
    """An expanded view without elements has no memory behind it."""
    dev = torch.device("cuda", 0)
    x = torch.zeros((6, 0), device=dev, requires_grad=True)
    adv = torch.ones((6, 1), device=dev).expand(6, 4)[:, :0]
    assert adv.data_ptr() == 0 or adv.stride(1) == 0
    for kind in ("grpo", "bnpo"):
        res = policy_loss(x, adv, torch.ones((6, 0), device=dev), loss_type=kind)
        (g,) = torch.autograd.grad(res.loss, x)
        assert float(res.loss) == 0.0 and float(res.kl) == 0.0 and g.shape == (6, 0)


@pytest.mark.parametrize("T", [5, 200, 1500])
@pytest.mark.parametrize("level", ["token", "sequence"])
def test_reference_that_rules_a_token_out(T, level):
    """exp(q) - 1 - q with q = -inf: the KL is infinite, its slope is 1; without beta it does not reach the loss."""
    logps, adv, mask, old, ref = _loss_inputs(4, T, seed=21)
    mask = torch.ones_like(mask)
    clean, _ = _check_loss(logps, adv, mask, old, ref, level=level)
    _, want = _check_loss(logps, adv, mask, old, ref, level=level, beta=0.1)
    ref[2, 3] = -math.inf
    x = logps.clone().requires_grad_()
    res = policy_loss(x, adv, mask, old, ref, importance_sampling_level=level)
    (g,) = torch.autograd.grad(res.loss, x)
    assert torch.equal(res.loss, clean.loss) and torch.isinf(res.kl) and torch.isfinite(g).all()
    x = logps.clone().requires_grad_()
    res = policy_loss(x, adv, mask, old, ref, importance_sampling_level=level, beta=0.1)
    (g,) = torch.autograd.grad(res.loss, x)
    d = _loss_definition(logps, adv, mask, old, ref, level=level, beta=0.1)
    assert torch.isinf(res.loss) and float(res.loss) > 0
    keep = torch.ones_like(mask, dtype=torch.bool)
    keep[2, 3] = False
    assert torch.equal(g[keep], want[keep])
    # the formula's: 24 u of |w A| + beta, per the bound of the checks above (sequence: the row's sum)
    size = (d["grad"].abs().max() + 1.0) * 64 * U
    assert abs(float(g[2, 3]) - float(d["grad"][2, 3])) <= float(size)


def test_results_do_not_change_from_call_to_call():
    logits, ids = _case((40, 7), 5003, torch.bfloat16, seed=12)
    logps, adv, mask, old, ref = _loss_inputs(700, 90, seed=13)
    a = token_logps(logits, ids, return_entropy=True)
    l = policy_loss(logps, adv, mask, old, ref, beta=0.1, loss_type="bnpo")
    for _ in range(3):
        b = token_logps(logits, ids, return_entropy=True)
        assert torch.equal(a[0], b[0]) and torch.equal(a[1], b[1])
        assert torch.equal(l.loss, policy_loss(logps, adv, mask, old, ref, beta=0.1, loss_type="bnpo").loss)


# ---- together ------------------------------------------------------------------------------------------------


def _step(logits, ids, mask, adv, old, ref):
    x = logits.detach().requires_grad_()
    lp, ent = token_logps(x[:, :-1], ids.masked_fill(mask == 0, -1), 0.9, return_entropy=True)
    res = policy_loss(lp, adv, mask, old, ref, beta=0.04)
    (grad,) = torch.autograd.grad(res.loss - 0.01 * (ent * mask).sum() / mask.sum(), x)
    return res.loss.detach(), grad


def _step_inputs(seed, R=16, T=5, V=3001, K=4):
    from genrec_amd.advantage import group_advantages

    dev = torch.device("cuda", 0)
    g = torch.Generator(device=dev).manual_seed(seed)
    logits = (torch.randn((R, T + 1, V), generator=g, device=dev) * 3).to(torch.bfloat16)
    ids = torch.randint(0, V, (R, T), generator=g, device=dev)
    mask = (torch.arange(T, device=dev)[None] < torch.randint(1, T + 1, (R, 1), generator=g, device=dev)).long()
    rewards = torch.rand((R, 1), generator=g, device=dev)
    adv = group_advantages(rewards, torch.ones(1, device=dev), K)[1]
    with torch.no_grad():
        lp = token_logps(logits[:, :-1], ids, 0.9)
    noise = torch.randn((2, R, T), generator=g, device=dev)
    return logits, ids, mask, adv, lp + 0.1 * noise[0], lp + 0.2 * noise[1]


def test_a_whole_step():
    """Rewards -> group advantages -> log-probabilities -> loss -> gradient of the logits, against 64 bits."""
    logits, ids, mask, adv, old, ref = _step_inputs(1)
    loss, grad = _step(logits, ids, mask, adv, old, ref)
    x = logits.double().requires_grad_()
    lp_all = torch.log_softmax(x[:, :-1] / 0.9, -1)
    lp = lp_all.gather(-1, ids[..., None])[..., 0]
    m = mask.double()
    w = (lp - old.double()).exp()
    A = adv.double()[:, None]
    q = ref.double() - lp
    tok = -torch.min(w * A, w.clamp(0.8, 1.2) * A) + 0.04 * (q.exp() - 1 - q)
    want = ((tok * m).sum(1) / m.sum(1)).mean()
    ent = -(lp_all.exp() * lp_all).sum(-1)
    (want_grad,) = torch.autograd.grad(want - 0.01 * (ent * m).sum() / m.sum(), x)
    assert abs(float(loss) - float(want)) <= 1e-5  # log-probabilities within _row_rel(3001) = 1e-5
    big = want_grad.abs().max()
    assert (grad.double() - want_grad).abs().max() <= (2.0 ** -8 + 1e-4) * big
    assert (grad[:, -1] == 0).all()


def test_step_recorded_into_a_graph():
    """A step recorded once and replayed over refilled buffers equals the eager step, with eager work between replays."""
    bufs = _step_inputs(2)
    made = {}
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        _step(*bufs)
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        made["out"] = _step(*bufs)
    for seed in (3, 4, 5):
        new = _step_inputs(seed)
        for b, n in zip(bufs, new):
            b.copy_(n)
        loss, grad = _step(*new)
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(made["out"][0], loss) and torch.equal(made["out"][1], grad)


def test_recording_refuses_leaves_of_an_eager_graph():
    """A leaf that a living eager graph holds: the recorded backward pass is refused before anything waits for the other
    stream, and with that graph gone, or a leaf of the recording's own, the same pass is recorded."""
    logits, ids, mask, adv, old, ref = _step_inputs(8)
    x = token_logps(logits[:, :-1].contiguous(), ids).detach().requires_grad_()
    y = logits[:, :-1].contiguous().requires_grad_()
    g = torch.ones_like(x)

    def loss():
        return torch.autograd.grad(policy_loss(x, adv, mask, old).loss, x)[0]

    def logps():
        return torch.autograd.grad(token_logps(y, ids), y, g)[0]

    for step in (loss, logps):
        want = step()
        alive = (policy_loss(x, adv, mask, old).loss, token_logps(y, ids))
        with pytest.raises(RuntimeError, match="leaves of its own"):
            with torch.cuda.graph(torch.cuda.CUDAGraph()):
                step()
        torch.cuda.synchronize()
        assert torch.equal(step(), want)
        del alive
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            got = step()
        for _ in range(3):
            got.zero_()
            graph.replay()
            torch.cuda.synchronize()
            assert torch.equal(got, want) and torch.equal(step(), want)


def test_two_streams_at_once():
    a, b = _step_inputs(6, V=20011), _step_inputs(7, V=20011)
    want = [_step(*a), _step(*b)]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream(), torch.cuda.Stream()]
    got = [None, None]
    for _ in range(4):
        for i, s in enumerate(streams):
            s.wait_stream(torch.cuda.current_stream())
            with torch.cuda.stream(s):
                got[i] = _step(*(a, b)[i])
    torch.cuda.synchronize()
    for w, g in zip(want, got):
        assert torch.equal(w[0], g[0]) and torch.equal(w[1], g[1])
