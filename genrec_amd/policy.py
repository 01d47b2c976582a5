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
import math
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


def _ptr(t):
    return t.data_ptr() if t is not None else None


def _scratch(n: int, dev):
    return torch.empty(n, dtype=torch.uint8, device=dev) if n else None


def _run(call, index: int, *args) -> None:
    """``call(*args, current stream)`` with device ``index`` current."""
    with _lib.on_device(index):
        status = call(*args, _lib.current_stream_ptr(index))
    if status:
        _lib.check(status)


def _rows_2d(t: torch.Tensor, what: str) -> torch.Tensor:
    """[N] as [N, 1], [B, T] as it is, elements of a row next to each other."""
    if t.dim() == 1:
        return t.unsqueeze(1)
    if t.dim() != 2:
        raise ValueError(f"{what} must be [rows] or [rows, positions], got {tuple(t.shape)}")
    return t if t.stride(1) == 1 or t.shape[1] <= 1 else t.contiguous()


def _f32_rows(t: Optional[torch.Tensor], what: str) -> Optional[torch.Tensor]:
    if t is None:
        return None
    return _rows_2d(t if t.dtype is torch.float32 else t.detach().to(torch.float32), what)


def _temperature(value) -> float:
    value = float(value)
    if not 0.0 < value < math.inf:
        raise ValueError(f"temperature must be positive and finite, got {value}")
    return value


def _token_ids(ids: torch.Tensor, dev) -> torch.Tensor:
    if ids.is_floating_point() or ids.is_complex() or ids.dtype == torch.bool:
        raise TypeError(f"token_ids must be integers, got {ids.dtype}")
    if ids.device != dev:
        raise ValueError(f"token_ids is on {ids.device}, expected {dev}")
    if ids.numel() > MAX_ROWS:
        raise ValueError(f"at most {MAX_ROWS} rows per call, got {ids.numel()}")
    return _rows_2d(ids if ids.dtype is torch.int64 else ids.to(torch.int64), "token_ids")


def _aligned_rows(t: torch.Tensor) -> torch.Tensor:
    """[N, H] with rows of consecutive elements that start on 16 bytes."""
    if t.stride(1) == 1 and t.data_ptr() % 16 == 0 and (t.shape[0] <= 1 or (t.stride(0) % 8 == 0 and t.stride(0) >= t.shape[1])):
        return t
    t = t.contiguous()
    return t if t.data_ptr() % 16 == 0 else t.clone()


def _grad_rows(g: Optional[torch.Tensor]) -> Optional[torch.Tensor]:
    if g is None or (g.dtype is torch.float32 and g.is_contiguous()):
        return g
    return g.to(torch.float32).contiguous()


def _token_logps_args(logits, ids, temperature, logps, stats, entropy, g=None, h=None, grad=None):
    three = logits.dim() == 3
    return _lib.GrxTokenLogpsArgs(
        logits.data_ptr(), logits.stride(0), logits.stride(1) if three else 0, ids.data_ptr(), ids.stride(0), ids.shape[0],
        ids.shape[1], logits.shape[-1], _lib.torch_dtype_code(logits.dtype), temperature, 0, logps, stats, entropy, g, h, grad)


class _TokenLogps(torch.autograd.Function):
    @staticmethod
    def forward(ctx, logits, ids, temperature, entropy):
        shape, dev = ids.shape, logits.device
        logps = torch.empty(shape, dtype=torch.float32, device=dev)
        ent = torch.empty(shape, dtype=torch.float32, device=dev) if entropy else None
        stats = torch.empty((*shape, 2), dtype=torch.float32, device=dev)
        a = _token_logps_args(logits, ids, temperature, logps.data_ptr(), stats.data_ptr(), _ptr(ent))
        lib = _lib.lib()
        n = lib.grx_token_logps_scratch_bytes(a.B * a.T, a.V, a.dtype)
        scratch = _scratch(n, dev)
        _run(lib.grx_token_logps, dev.index, C.byref(a), _ptr(scratch), n)
        if ctx.needs_input_grad[0]:
            ctx.save_for_backward(logits, ids, stats, ent)
            ctx.temperature = temperature
            ctx.set_materialize_grads(False)
        return (logps, ent) if entropy else logps

    @staticmethod
    @once_differentiable
    def backward(ctx, g_logps, g_entropy=None):
        logits, ids, stats, ent = ctx.saved_tensors
        grad = torch.empty(logits.shape, dtype=logits.dtype, device=logits.device)
        g_logps, g_entropy = _grad_rows(g_logps), _grad_rows(g_entropy)
        a = _token_logps_args(logits, ids, ctx.temperature, None, stats.data_ptr(), _ptr(ent), _ptr(g_logps), _ptr(g_entropy),
                              grad.data_ptr())
        _run(_lib.lib().grx_token_logps_backward, logits.device.index, C.byref(a))
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


def _lm_token_logps_args(hidden, weight, ids, temperature, logps, stats, entropy, g=None, h=None, grad_h=None, grad_w=None):
    (N, H), V = hidden.shape, weight.shape[0]
    return _lib.GrxLmTokenLogpsArgs(
        hidden.data_ptr(), hidden.stride(0) if N > 1 else H, weight.data_ptr(), weight.stride(0) if V > 1 else H, ids.data_ptr(),
        N, H, V, temperature, logps, stats, entropy, g, h, grad_h, grad_w)


class _LmTokenLogps(torch.autograd.Function):
    @staticmethod
    def forward(ctx, hidden, weight, ids, temperature, entropy):
        N, dev = hidden.shape[0], hidden.device
        logps = torch.empty(N, dtype=torch.float32, device=dev)
        ent = torch.empty(N, dtype=torch.float32, device=dev) if entropy else None
        stats = torch.empty((N, 2), dtype=torch.float32, device=dev)
        a = _lm_token_logps_args(hidden, weight, ids, temperature, logps.data_ptr(), stats.data_ptr(), _ptr(ent))
        lib = _lib.lib()
        n = lib.grx_lm_token_logps_scratch_bytes(N, a.H, a.V, int(entropy))
        scratch = _scratch(n, dev)
        _run(lib.grx_lm_token_logps, dev.index, C.byref(a), _ptr(scratch), n)
        if ctx.needs_input_grad[0] or ctx.needs_input_grad[1]:
            ctx.save_for_backward(hidden, weight, ids, stats, ent)
            ctx.temperature = temperature
            ctx.set_materialize_grads(False)
        return (logps, ent) if entropy else logps

    @staticmethod
    @once_differentiable
    def backward(ctx, g_logps, g_entropy=None):
        hidden, weight, ids, stats, ent = ctx.saved_tensors
        dev, N = hidden.device, hidden.shape[0]
        want_h, want_w = ctx.needs_input_grad[:2]
        grad_h = torch.empty(hidden.shape, dtype=hidden.dtype, device=dev) if want_h else None
        grad_w = torch.empty(weight.shape, dtype=weight.dtype, device=dev) if want_w else None
        if N == 0 and want_w:
            grad_w.zero_()
        g_logps, g_entropy = _grad_rows(g_logps), _grad_rows(g_entropy)
        a = _lm_token_logps_args(hidden, weight, ids, ctx.temperature, None, stats.data_ptr(), _ptr(ent), _ptr(g_logps),
                                 _ptr(g_entropy), _ptr(grad_h), _ptr(grad_w))
        lib = _lib.lib()
        n = lib.grx_lm_token_logps_backward_scratch_bytes(N, a.H, a.V, int(want_h), int(want_w))
        scratch = _scratch(n, dev)
        _run(lib.grx_lm_token_logps_backward, dev.index, C.byref(a), _ptr(scratch), n)
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
    def forward(ctx, logps, a, stats):
        dev = logps.device
        loss = torch.empty((), dtype=torch.float32, device=dev)
        unit = torch.empty(logps.shape, dtype=torch.float32, device=dev) if ctx.needs_input_grad[0] else None
        a.loss, a.stats, a.unit_grad = loss.data_ptr(), stats.data_ptr(), _ptr(unit)
        lib = _lib.lib()
        n = lib.grx_policy_loss_scratch_bytes(a.R, a.T)
        scratch = _scratch(n, dev)
        _run(lib.grx_policy_loss, dev.index, C.byref(a), _ptr(scratch), n)
        if unit is not None:
            ctx.save_for_backward(unit, stats)
        return loss

    @staticmethod
    @once_differentiable
    def backward(ctx, g_loss):
        unit, stats = ctx.saved_tensors
        grad = torch.empty_like(unit)
        if g_loss.dtype is not torch.float32:
            g_loss = g_loss.to(torch.float32)
        _run(_lib.lib().grx_policy_loss_backward, unit.device.index, unit.data_ptr(), stats.data_ptr(), g_loss.data_ptr(),
             unit.numel(), grad.data_ptr())
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
    dev, shape = logps.device, logps.shape
    if len(shape) != 2:
        raise ValueError(f"logps must be [rows, positions], got {tuple(shape)}")
    R, T = shape
    if R >= 1 << 31 or T >= 1 << 31:
        raise ValueError("rows and positions must stay below 2^31")
    for name, t in (("mask", mask), ("old_logps", old_logps), ("ref_logps", ref_logps)):
        if t is not None and t.shape != shape:
            raise ValueError(f"{name} must have the shape of logps {tuple(shape)}, got {tuple(t.shape)}")
    if advantages.shape != shape and advantages.shape != shape[:1]:
        raise ValueError(f"advantages must be [{R}] or [{R}, {T}], got {tuple(advantages.shape)}")
    for name, t in (("mask", mask), ("old_logps", old_logps), ("ref_logps", ref_logps), ("advantages", advantages)):
        if t is not None and t.device != dev:
            raise ValueError(f"{name} is on {t.device}, expected {dev}")
    for name, t in (("logps", logps), ("old_logps", old_logps), ("ref_logps", ref_logps), ("advantages", advantages)):
        if t is not None and not t.is_floating_point():
            raise TypeError(f"{name} must be floating point, got {t.dtype}")
    if loss_type not in _LOSS_TYPES:
        raise ValueError(f"loss_type must be one of {_LOSS_TYPES}, got {loss_type!r}")
    if importance_sampling_level not in ("token", "sequence"):
        raise ValueError(f"importance_sampling_level must be 'token' or 'sequence', got {importance_sampling_level!r}")
    epsilon_high = epsilon_low if epsilon_high is None else epsilon_high
    if not (0.0 <= epsilon_low < 1.0 and 0.0 <= epsilon_high < math.inf):
        raise ValueError(f"epsilon_low must lie in [0, 1) and epsilon_high must not be negative, got {epsilon_low}, {epsilon_high}")
    if delta is not None and not 1.0 + epsilon_high < delta < math.inf:
        raise ValueError(f"delta must lie above 1 + epsilon_high, got {delta}")
    if not -math.inf < beta < math.inf:
        raise ValueError(f"beta must be finite, got {beta}")
    if beta != 0.0 and ref_logps is None:
        raise ValueError("a KL term (beta) needs ref_logps")
    normalizer = 0.0
    if loss_type == "dr_grpo" or loss_type == "dapo":
        given = max_completion_length if loss_type == "dr_grpo" else num_items
        if given is None or not 0.0 < float(given) < math.inf:
            raise ValueError(f"loss_type {loss_type!r} needs a positive "
                             f"{'max_completion_length' if loss_type == 'dr_grpo' else 'num_items'}, got {given}")
        normalizer = float(given) * (max(R, 1) if loss_type == "dr_grpo" else 1)
    _lib.require_cuda(logps, "logps")
    # without detach() where nothing is converted: only addresses are taken of these
    if logps.dtype is not torch.float32:
        logps = logps.to(torch.float32)
    logps = _rows_2d(logps, "logps")
    old, ref = _f32_rows(old_logps, "old_logps"), _f32_rows(ref_logps, "ref_logps")
    adv = advantages if advantages.dtype is torch.float32 else advantages.detach().to(torch.float32)
    if mask.dtype not in _MASK_TYPES:
        mask = mask > 0
    mask = _rows_2d(mask, "mask")
    stats = torch.empty(4, dtype=torch.float32, device=dev)
    a = _lib.GrxPolicyLossArgs(
        logps.data_ptr(), logps.stride(0), _ptr(old), old.stride(0) if old is not None else 0, _ptr(ref),
        ref.stride(0) if ref is not None else 0, adv.data_ptr(), adv.stride(0), adv.stride(1) if adv.dim() == 2 else 0,
        mask.data_ptr(), mask.stride(0), _MASK_TYPES[mask.dtype], R, T, importance_sampling_level == "sequence",
        loss_type == "grpo", beta, epsilon_low, epsilon_high, delta or 0.0, normalizer)
    return PolicyLoss(_PolicyLoss.apply(logps, a, stats), stats)
