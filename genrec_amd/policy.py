"""The policy-gradient step behind a rollout: log-probabilities of the completion tokens, and the clipped loss.

The reference's trainers hand their advantages (fixed_hint_grpo_trainer.py:382-408,
token_prefix_grpo_trainer.py:196-278) to the loss of their base class, which computes per-token
log-probabilities from the model's logits and a clipped surrogate with a KL term on them.  Here both are HIP
kernels with hand-written gradients, on autograd tensors:

    logps = token_logps(logits[:, :-1], completion_ids.masked_fill(completion_mask == 0, -1))
    res = policy_loss(logps, rollout.local_advantages, completion_mask, old_logps, ref_logps, beta=0.04)
    res.loss.backward()

Everything runs on the current stream; nothing is read back.
"""

from __future__ import annotations

import ctypes as C
from typing import Optional

import torch
from torch.autograd.function import once_differentiable

from . import _lib

_MASK_TYPES = {torch.bool: 0, torch.uint8: 0, torch.int32: 1, torch.int64: 2, torch.float32: 3}
MAX_ROWS = 1 << 23
_LOSS_TYPES = ("grpo", "bnpo", "dr_grpo", "dapo")


def _same_device(dev, **tensors) -> None:
    for name, t in tensors.items():
        if t is not None and t.device != dev:
            raise ValueError(f"{name} is on {t.device}, expected {dev}")


def _scratch(n: int, dev):
    return torch.empty(n, dtype=torch.uint8, device=dev) if n else None


def _ptr(t):
    return t.data_ptr() if t is not None else None


def _rows_2d(t: torch.Tensor, what: str) -> torch.Tensor:
    """[N] as [N, 1], [B, T] as it is, elements of a row next to each other."""
    if t.dim() == 1:
        return t.unsqueeze(1)
    if t.dim() != 2:
        raise ValueError(f"{what} must be [rows] or [rows, positions], got {tuple(t.shape)}")
    return t if t.shape[1] <= 1 or t.stride(1) == 1 else t.contiguous()


def _temperature(value) -> float:
    value = float(value)
    if not 0.0 < value < float("inf"):
        raise ValueError(f"temperature must be positive and finite, got {value}")
    return value


def _token_ids(ids: torch.Tensor, dev) -> torch.Tensor:
    if ids.is_floating_point() or ids.is_complex() or ids.dtype == torch.bool:
        raise TypeError(f"token_ids must be integers, got {ids.dtype}")
    _same_device(dev, token_ids=ids)
    if ids.numel() > MAX_ROWS:
        raise ValueError(f"at most {MAX_ROWS} rows per call, got {ids.numel()}")
    return _rows_2d(ids.detach().to(torch.int64), "token_ids")


def _aligned_rows(t: torch.Tensor) -> torch.Tensor:
    """[N, H] with rows of consecutive elements that start on 16 bytes."""
    if t.stride(1) == 1 and t.data_ptr() % 16 == 0 and (t.shape[0] <= 1 or (t.stride(0) % 8 == 0 and t.stride(0) >= t.shape[1])):
        return t
    t = t.contiguous()
    return t if t.data_ptr() % 16 == 0 else t.clone()


def _grad_rows(g: Optional[torch.Tensor]) -> Optional[torch.Tensor]:
    return None if g is None else g.to(torch.float32).contiguous()


class _TokenLogps(torch.autograd.Function):
    @staticmethod
    def forward(ctx, logits, ids, temperature, entropy):
        B, T = ids.shape
        dev = logits.device
        V = logits.shape[-1]
        a = _lib.GrxTokenLogpsArgs()
        a.logits = logits.data_ptr()
        a.row_stride, a.pos_stride = logits.stride(0), (logits.stride(1) if logits.dim() == 3 else 0)
        a.token_ids, a.ids_stride = ids.data_ptr(), ids.stride(0)
        a.B, a.T, a.V, a.dtype, a.temperature = B, T, V, _lib.torch_dtype_code(logits.dtype), temperature
        out = torch.empty((2, B, T) if entropy else (1, B, T), dtype=torch.float32, device=dev)
        stats = torch.empty((B, T, 2), dtype=torch.float32, device=dev)
        a.logps, a.row_stats = out.data_ptr(), stats.data_ptr()
        logps, ent = out[0], None
        if entropy:
            ent = out[1]
            a.entropy = ent.data_ptr()
        index = dev.index
        lib = _lib.lib()
        n = lib.grx_token_logps_scratch_bytes(B * T, V, a.dtype)
        scratch = _scratch(n, dev)
        with _lib.on_device(index):
            _lib.check(lib.grx_token_logps(C.byref(a), _ptr(scratch), n, _lib.current_stream_ptr(index)))
        ctx.save_for_backward(logits, ids, stats, *((ent,) if entropy else ()))
        ctx.temperature = temperature
        ctx.set_materialize_grads(False)
        return (logps, ent) if entropy else logps

    @staticmethod
    @once_differentiable
    def backward(ctx, g_logps, g_entropy=None):
        logits, ids, stats, *rest = ctx.saved_tensors
        B, T = ids.shape
        dev = logits.device
        grad = torch.empty(logits.shape, dtype=logits.dtype, device=dev)
        g_logps, g_entropy = _grad_rows(g_logps), _grad_rows(g_entropy)
        a = _lib.GrxTokenLogpsArgs()
        a.logits = logits.data_ptr()
        a.row_stride, a.pos_stride = logits.stride(0), (logits.stride(1) if logits.dim() == 3 else 0)
        a.token_ids, a.ids_stride = ids.data_ptr(), ids.stride(0)
        a.B, a.T, a.V, a.dtype, a.temperature = B, T, logits.shape[-1], _lib.torch_dtype_code(logits.dtype), ctx.temperature
        a.row_stats = stats.data_ptr()
        a.entropy = _ptr(rest[0]) if rest else None
        a.grad_logps, a.grad_entropy, a.grad_logits = _ptr(g_logps), _ptr(g_entropy), grad.data_ptr()
        index = dev.index
        with _lib.on_device(index):
            _lib.check(_lib.lib().grx_token_logps_backward(C.byref(a), _lib.current_stream_ptr(index)))
        return grad, None, None, None


def token_logps(logits: torch.Tensor, token_ids: torch.Tensor, temperature: float = 1.0, return_entropy: bool = False):
    """Log-probabilities of ``token_ids`` under ``softmax(logits / temperature)``, fp32, in the shape of
    ``token_ids``; with ``return_entropy`` the pair (log-probabilities, entropies of the rows).

    ``logits`` [B, T, V] or [N, V] on the GPU, fp32, bf16 or fp16, last dimension contiguous (a view such as
    ``outputs.logits[:, -T - 1 : -1]`` is read where it lies); ``token_ids`` [B, T] or [N], integers.  A negative
    id marks padding: its row of logits is not read, results and gradient are 0 whatever it holds.  An id that
    is not below V gives NaN.  Differentiable in ``logits`` (the gradient has their type); rows whose incoming
    gradient is 0 cost one write.  A pass recorded into a HIP graph needs leaves of its own: take
    ``logits.detach().requires_grad_()`` inside the recording."""
    temperature = _temperature(temperature)
    _lib.torch_dtype_code(logits.dtype)
    if logits.dim() not in (2, 3) or token_ids.shape != logits.shape[:-1]:
        raise ValueError(f"logits must be [..., V] with one row per token id: got {tuple(logits.shape)} for ids "
                         f"{tuple(token_ids.shape)}")
    if logits.shape[-1] < 1:
        raise ValueError("the vocabulary is empty")
    shape = token_ids.shape
    ids = _token_ids(token_ids, logits.device)
    _lib.require_cuda(logits, "logits")
    if logits.shape[-1] > 1 and logits.stride(-1) != 1:
        logits = logits.contiguous()
    out = _TokenLogps.apply(logits, ids, temperature, bool(return_entropy))
    if len(shape) == 2:
        return out
    return tuple(t.reshape(shape) for t in out) if return_entropy else out.reshape(shape)


class _LmTokenLogps(torch.autograd.Function):
    @staticmethod
    def _args(hidden, weight, ids, temperature):
        a = _lib.GrxLmTokenLogpsArgs()
        a.hidden, a.hidden_stride = hidden.data_ptr(), hidden.stride(0) if hidden.shape[0] > 1 else hidden.shape[1]
        a.weight, a.weight_stride = weight.data_ptr(), weight.stride(0) if weight.shape[0] > 1 else weight.shape[1]
        a.token_ids, a.temperature = ids.data_ptr(), temperature
        (a.N, a.H), a.V = hidden.shape, weight.shape[0]
        return a

    @staticmethod
    def forward(ctx, hidden, weight, ids, temperature, entropy):
        N = hidden.shape[0]
        dev = hidden.device
        a = _LmTokenLogps._args(hidden, weight, ids, temperature)
        out = torch.empty((2, N) if entropy else (1, N), dtype=torch.float32, device=dev)
        stats = torch.empty((N, 2), dtype=torch.float32, device=dev)
        a.logps, a.row_stats = out.data_ptr(), stats.data_ptr()
        logps, ent = out[0], None
        if entropy:
            ent = out[1]
            a.entropy = ent.data_ptr()
        index = dev.index
        lib = _lib.lib()
        n = lib.grx_lm_token_logps_scratch_bytes(N, a.H, a.V, int(entropy))
        scratch = _scratch(n, dev)
        with _lib.on_device(index):
            _lib.check(lib.grx_lm_token_logps(C.byref(a), _ptr(scratch), n, _lib.current_stream_ptr(index)))
        ctx.save_for_backward(hidden, weight, ids, stats, *((ent,) if entropy else ()))
        ctx.temperature = temperature
        ctx.set_materialize_grads(False)
        return (logps, ent) if entropy else logps

    @staticmethod
    @once_differentiable
    def backward(ctx, g_logps, g_entropy=None):
        hidden, weight, ids, stats, *rest = ctx.saved_tensors
        dev = hidden.device
        a = _LmTokenLogps._args(hidden, weight, ids, ctx.temperature)
        want_h, want_w = ctx.needs_input_grad[:2]
        grad_h = torch.empty(hidden.shape, dtype=hidden.dtype, device=dev) if want_h else None
        grad_w = torch.empty(weight.shape, dtype=weight.dtype, device=dev) if want_w else None
        if a.N == 0 and want_w:
            grad_w.zero_()
        g_logps, g_entropy = _grad_rows(g_logps), _grad_rows(g_entropy)
        a.row_stats, a.entropy = stats.data_ptr(), (_ptr(rest[0]) if rest else None)
        a.grad_logps, a.grad_entropy = _ptr(g_logps), _ptr(g_entropy)
        a.grad_hidden, a.grad_weight = _ptr(grad_h), _ptr(grad_w)
        index = dev.index
        lib = _lib.lib()
        n = lib.grx_lm_token_logps_backward_scratch_bytes(a.N, a.H, a.V, int(want_h), int(want_w))
        scratch = _scratch(n, dev)
        with _lib.on_device(index):
            _lib.check(lib.grx_lm_token_logps_backward(C.byref(a), _ptr(scratch), n, _lib.current_stream_ptr(index)))
        return grad_h, grad_w, None, None, None


def lm_head_token_logps(hidden: torch.Tensor, weight: torch.Tensor, token_ids: torch.Tensor, temperature: float = 1.0,
                        return_entropy: bool = False):
    """:func:`token_logps` of ``logits = hidden @ weight.T`` without the logits: the product runs on the matrix cores
    and is consumed tile by tile, forward and backward (the backward pass forms it again).

    ``hidden`` [B, T, H] or [N, H] and ``weight`` [V, H] (``lm_head.weight``, no bias), bf16, H a multiple of 64, on
    the GPU; ``token_ids`` [B, T] or [N], negative for padding.  Differentiable in both; a frozen weight costs
    nothing.  The logits' gradient passes through bf16 on its way to the two products, as it does under autograd.
    The backward pass takes a scratch tensor of about 1 GB at many rows.  A pass recorded into a HIP graph needs
    leaves of its own (``detach().requires_grad_()`` inside the recording)."""
    temperature = _temperature(temperature)
    if hidden.dtype != torch.bfloat16 or weight.dtype != torch.bfloat16:
        raise TypeError(f"hidden states and weight must be bfloat16, got {hidden.dtype} and {weight.dtype}")
    if hidden.dim() not in (2, 3) or token_ids.shape != hidden.shape[:-1]:
        raise ValueError(f"hidden must be [..., H] with one row per token id: got {tuple(hidden.shape)} for ids "
                         f"{tuple(token_ids.shape)}")
    if weight.dim() != 2 or weight.shape[1] != hidden.shape[-1] or weight.shape[0] < 1:
        raise ValueError(f"weight must be [V, {hidden.shape[-1]}], got {tuple(weight.shape)}")
    H = hidden.shape[-1]
    if H < 64 or H % 64 or H > 1 << 16 or weight.shape[0] > 1 << 24:
        raise ValueError(f"the hidden size must be a multiple of 64 up to 2^16 and the vocabulary at most 2^24, got "
                         f"{H}, {weight.shape[0]}")
    shape = token_ids.shape
    ids = _token_ids(token_ids, hidden.device).reshape(-1).contiguous()
    _same_device(hidden.device, weight=weight)
    _lib.require_cuda(hidden, "hidden")
    rows = _aligned_rows(hidden.reshape(-1, H))
    out = _LmTokenLogps.apply(rows, _aligned_rows(weight), ids, temperature, bool(return_entropy))
    if len(shape) == 1:
        return out
    return tuple(t.reshape(shape) for t in out) if return_entropy else out.reshape(shape)


class PolicyLoss:
    """Result of :func:`policy_loss`: ``loss`` (0-d, differentiable) and, as 0-d fp32 tensors without gradient,
    ``kl`` (mean of the KL estimate over valid tokens), ``clip_low`` and ``clip_high`` (shares of valid tokens cut
    at the lower and the upper bound)."""

    __slots__ = ("loss", "kl", "clip_low", "clip_high")

    def __init__(self, loss, stats):
        self.loss = loss
        self.kl, self.clip_low, self.clip_high, _ = stats.unbind(0)


class _PolicyLoss(torch.autograd.Function):
    @staticmethod
    def forward(ctx, logps, a, keep):
        dev = logps.device
        R, T = logps.shape
        out = torch.empty(5, dtype=torch.float32, device=dev)
        loss, stats = out[0], out[1:]
        unit = torch.empty((R, T), dtype=torch.float32, device=dev) if ctx.needs_input_grad[0] else None
        a.loss, a.stats, a.unit_grad = loss.data_ptr(), stats.data_ptr(), _ptr(unit)
        index = dev.index
        lib = _lib.lib()
        n = lib.grx_policy_loss_scratch_bytes(R, T)
        scratch = _scratch(n, dev)
        with _lib.on_device(index):
            _lib.check(lib.grx_policy_loss(C.byref(a), _ptr(scratch), n, _lib.current_stream_ptr(index)))
        ctx.mark_non_differentiable(stats)
        ctx.set_materialize_grads(False)
        if unit is not None:
            ctx.save_for_backward(unit, stats)
        return loss, stats

    @staticmethod
    @once_differentiable
    def backward(ctx, g_loss, _g_stats):
        if g_loss is None:
            return None, None, None
        unit, stats = ctx.saved_tensors
        grad = torch.empty_like(unit)
        g_loss = g_loss.to(torch.float32)
        index = unit.device.index
        with _lib.on_device(index):
            _lib.check(_lib.lib().grx_policy_loss_backward(unit.data_ptr(), stats.data_ptr(), g_loss.data_ptr(),
                                                           unit.numel(), grad.data_ptr(), _lib.current_stream_ptr(index)))
        return grad, None, None


def policy_loss(
    logps: torch.Tensor,
    advantages: torch.Tensor,
    mask: torch.Tensor,
    old_logps: Optional[torch.Tensor] = None,
    ref_logps: Optional[torch.Tensor] = None,
    *,
    epsilon_low: float = 0.2,
    epsilon_high: Optional[float] = None,
    delta: Optional[float] = None,
    beta: float = 0.0,
    loss_type: str = "grpo",
    importance_sampling_level: str = "token",
    max_completion_length: Optional[int] = None,
    num_items: Optional[float] = None,
) -> PolicyLoss:
    """Clipped policy loss of ``logps`` [R, T] (:func:`token_logps`), with its gradient.

    ``advantages`` [R] (``rollout_advantages``) or [R, T] (``token_prefix_advantages``); ``mask`` [R, T], valid
    where above 0 (bool, uint8, int32, int64 or float32); ``old_logps`` / ``ref_logps`` [R, T]: the policy that
    sampled (None: this one, ratio 1) and the reference policy (needed when ``beta`` is not 0; its KL estimate is
    reported whenever it is given).  Per valid token, with w the ratio of the new to the old probability, per token or
    (``importance_sampling_level="sequence"``) as the geometric mean over the row's valid tokens:

        l = -min(min(w, delta) A, clip(w, 1 - epsilon_low, 1 + epsilon_high) A) + beta (exp(ref - logp) - (ref - logp) - 1)

    ``loss_type`` weighs them: "grpo" averages each row over its valid tokens and then the rows, "bnpo" averages
    over the batch's valid tokens, "dr_grpo" divides the sum by R x ``max_completion_length``, "dapo" by
    ``num_items`` (the valid tokens of the whole step, e.g. over gradient accumulation).  ``epsilon_high`` defaults
    to ``epsilon_low``; ``delta`` must lie above 1 + ``epsilon_high``.  Masked positions are not read, whatever they
    hold, and get gradient 0; a batch without valid tokens has loss 0.  Only ``logps`` gets a gradient."""
    dev = logps.device
    if logps.dim() != 2:
        raise ValueError(f"logps must be [rows, positions], got {tuple(logps.shape)}")
    R, T = logps.shape
    if max(R, T) >= 1 << 31:
        raise ValueError("rows and positions must stay below 2^31")
    for name, t in (("mask", mask), ("old_logps", old_logps), ("ref_logps", ref_logps)):
        if t is not None and t.shape != logps.shape:
            raise ValueError(f"{name} must have the shape of logps {tuple(logps.shape)}, got {tuple(t.shape)}")
    if tuple(advantages.shape) not in ((R,), (R, T)):
        raise ValueError(f"advantages must be [{R}] or [{R}, {T}], got {tuple(advantages.shape)}")
    _same_device(dev, mask=mask, old_logps=old_logps, ref_logps=ref_logps, advantages=advantages)
    for name, t in (("logps", logps), ("old_logps", old_logps), ("ref_logps", ref_logps), ("advantages", advantages)):
        if t is not None and not t.is_floating_point():
            raise TypeError(f"{name} must be floating point, got {t.dtype}")
    if loss_type not in _LOSS_TYPES:
        raise ValueError(f"loss_type must be one of {_LOSS_TYPES}, got {loss_type!r}")
    if importance_sampling_level not in ("token", "sequence"):
        raise ValueError(f"importance_sampling_level must be 'token' or 'sequence', got {importance_sampling_level!r}")
    epsilon_high = epsilon_low if epsilon_high is None else epsilon_high
    if not (0.0 <= epsilon_low < 1.0 and 0.0 <= epsilon_high < float("inf")):
        raise ValueError(f"epsilon_low must lie in [0, 1) and epsilon_high must not be negative, got {epsilon_low}, {epsilon_high}")
    if delta is not None and not 1.0 + epsilon_high < delta < float("inf"):
        raise ValueError(f"delta must lie above 1 + epsilon_high, got {delta}")
    if not -float("inf") < beta < float("inf"):
        raise ValueError(f"beta must be finite, got {beta}")
    if beta != 0.0 and ref_logps is None:
        raise ValueError("a KL term (beta) needs ref_logps")
    normalizer = 0.0
    if loss_type in ("dr_grpo", "dapo"):
        given = max_completion_length if loss_type == "dr_grpo" else num_items
        if given is None or not 0.0 < float(given) < float("inf"):
            raise ValueError(f"loss_type {loss_type!r} needs a positive "
                             f"{'max_completion_length' if loss_type == 'dr_grpo' else 'num_items'}, got {given}")
        normalizer = float(given) * (max(R, 1) if loss_type == "dr_grpo" else 1)
    _lib.require_cuda(logps, "logps")
    f32 = torch.float32
    logps = logps if logps.dtype == f32 else logps.to(f32)
    logps = _rows_2d(logps, "logps")
    old, ref = (None if t is None else _rows_2d(t.detach().to(f32), "log-probabilities") for t in (old_logps, ref_logps))
    adv = advantages.detach().to(f32)
    if mask.dtype not in _MASK_TYPES:
        mask = mask > 0
    mask = _rows_2d(mask.detach(), "mask")
    a = _lib.GrxPolicyLossArgs()
    a.logps, a.logps_stride = logps.data_ptr(), logps.stride(0)
    if old is not None:
        a.old_logps, a.old_stride = old.data_ptr(), old.stride(0)
    if ref is not None:
        a.ref_logps, a.ref_stride = ref.data_ptr(), ref.stride(0)
    a.advantages = adv.data_ptr()
    a.adv_row_stride, a.adv_pos_stride = adv.stride(0), (adv.stride(1) if adv.dim() == 2 else 0)
    a.mask, a.mask_stride, a.mask_type = mask.data_ptr(), mask.stride(0), _MASK_TYPES[mask.dtype]
    a.R, a.T = R, T
    a.sequence_level, a.row_mean = int(importance_sampling_level == "sequence"), int(loss_type == "grpo")
    a.beta, a.epsilon_low, a.epsilon_high = beta, epsilon_low, epsilon_high
    a.delta, a.normalizer = delta or 0.0, normalizer
    return PolicyLoss(*_PolicyLoss.apply(logps, a, (old, ref, adv, mask)))
