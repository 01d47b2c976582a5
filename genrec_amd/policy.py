"""The policy-gradient step behind a rollout: log-probabilities of the completion tokens, and the clipped loss.

The reference's trainers hand their advantages (fixed_hint_grpo_trainer.py:382-408,
token_prefix_grpo_trainer.py:196-278) to the loss of their base class, which computes per-token
log-probabilities from the model's logits and a clipped surrogate with a KL term on them.  Here both are HIP
kernels with hand-written gradients, on autograd tensors:

    ids = input_ids.new_full(logits.shape[:2], -1)      # -1: padding, prompt and last position
    ids[:, -T - 1 : -1] = completion_ids.masked_fill(completion_mask == 0, -1)
    logps = token_logps(logits, ids)[:, -T - 1 : -1]
    res = policy_loss(logps, rollout.local_advantages, completion_mask, old_logps, ref_logps, beta=0.04)
    res.loss.backward()

Everything runs on the current stream; nothing is read back.
"""

from __future__ import annotations

import ctypes as C
from typing import Optional

import torch

from . import _lib

MAX_ROWS = 1 << 23  # token rows per call

_ops_module = None


def _ops():
    """The autograd side of the operators (csrc/policy_ops.cpp), bound to the loaded library."""
    global _ops_module
    if _ops_module is None:
        lib = _lib.lib()
        try:
            from . import _policy_ops
        except ImportError as e:
            raise _lib.GenrecHipError(f"genrec_amd/_policy_ops.so cannot be loaded ({e}): run `make -C genrec_amd/csrc`") from e
        built = tuple(lib.grx_policy_struct_bytes(i) for i in range(3))
        if _policy_ops.abi_version != lib.grx_abi_version() or _policy_ops.struct_bytes != built:
            raise _lib.GenrecHipError("genrec_amd/_policy_ops.so and libgenrec_hip.so are of different builds: run "
                                      "`make -C genrec_amd/csrc`")
        names = [n for n in _lib.EXPORTED_SYMBOLS if "token_logps" in n or "policy_loss" in n] + ["grx_last_error"]
        _policy_ops.bind(_lib.GenrecHipError, {n: C.cast(getattr(lib, n), C.c_void_p).value for n in names})
        _ops_module = _policy_ops
    return _ops_module


def token_logps(logits: torch.Tensor, token_ids: torch.Tensor, temperature: float = 1.0, return_entropy: bool = False):
    """Log-probabilities of ``token_ids`` under ``softmax(logits / temperature)``, fp32, in the shape of
    ``token_ids``; with ``return_entropy`` the pair (log-probabilities, entropies of the rows).

    ``logits`` [B, T, V] or [N, V] on the GPU, fp32, bf16 or fp16, last dimension contiguous (a view such as
    ``outputs.logits[:, -T - 1 : -1]`` is read where it lies); ``token_ids`` [B, T] or [N], integers.  A negative
    id marks padding: its row of logits is not read, results and gradient are 0 whatever it holds.  An id that
    is not below V gives NaN.  Where a gradient follows, hand over the whole logits with -1 at the positions that do not
    count: the gradient is then written in one pass.  That of a slice is autograd's, which fills the whole logits'
    gradient with 0 and copies this one's into it (bf16, V = 152,640, forward and gradient: 5 of 6 positions of 64 rows 72
    and 109 us, 128 of 129 1.18 and 2.38 ms, 5 of 40 211 and 226 us).  Differentiable in ``logits`` (the gradient has their type); rows
    whose incoming gradient is 0 cost one write.  A pass recorded into a HIP graph needs leaves of its own: take
    ``logits.detach().requires_grad_()`` inside the recording (gradients that would leave it are refused)."""
    return (_ops_module or _ops()).token_logps(logits, token_ids, temperature, return_entropy)


def lm_head_token_logps(hidden: torch.Tensor, weight: torch.Tensor, token_ids: torch.Tensor, temperature: float = 1.0,
                        return_entropy: bool = False, keep_bytes: int = 8 << 30):
    """:func:`token_logps` of ``logits = hidden @ weight.T``: the product runs on the matrix cores and is consumed tile
    by tile, forward and backward.  Where a backward pass follows, and N x V x 4 bytes (and the tiles' margins; all N rows,
    padding too) are at most ``keep_bytes`` and are to be had, the products are kept for it in fp32 until its graph is gone:
    by default this trades the memory that the operator saves for a tenth of the time and more.  **With ``keep_bytes=0`` no
    logits are ever held** and the backward pass forms them again (8192 rows of a vocabulary of 152,640, H = 2048, both
    gradients: 5 GB kept, 21.1 ms; nothing kept, 23.4 ms): the choice where memory is short or several graphs are alive at
    a time.

    ``hidden`` [B, T, H] or [N, H] and ``weight`` [V, H] (``lm_head.weight``, no bias), bf16, H a multiple of 64, on
    the GPU; ``token_ids`` [B, T] or [N], negative for padding.  Differentiable in both; a frozen weight costs
    nothing.  The logits' gradient reaches the two products in two bf16 pieces (16 bits of each element, where autograd's bf16
    logits would hold 8), so that rows whose gradients cancel leave nothing but the rounding of 32-bit sums.
    Rows of padding, and in the backward pass rows whose gradients are 0, take no part in the products.  Scratch
    tensors: forward, per row, V / 16 (many rows) to V / 4 bytes (few), half as much again with entropies; backward up to
    1 GB for a chunk of the logits' gradient (above 2^20 rows 1 KB a row), and up to 64 copies of ``hidden``'s gradient in
    fp32 where there are few rows, one where there are many; both a copy or two of ``hidden``.  A pass
    recorded into a HIP graph needs leaves of its own (``detach().requires_grad_()`` inside the recording)."""
    return (_ops_module or _ops()).lm_head_token_logps(hidden, weight, token_ids, temperature, return_entropy, keep_bytes)


class PolicyLoss:
    """Result of :func:`policy_loss`: ``loss`` (0-d, differentiable) and, as 0-d fp32 tensors without gradient,
    ``kl`` (mean of the KL estimate over valid tokens), ``clip_low`` and ``clip_high`` (shares of valid tokens cut
    at the lower and the upper bound).  They are the caller's: averaging them in place before ``loss.backward()`` is fine."""

    __slots__ = ("loss", "kl", "clip_low", "clip_high")

    def __init__(self, loss, kl, clip_low, clip_high):
        self.loss, self.kl, self.clip_low, self.clip_high = loss, kl, clip_low, clip_high


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
    return PolicyLoss(*(_ops_module or _ops()).policy_loss(
        logps, advantages, mask, old_logps, ref_logps, epsilon_low, epsilon_high, delta, beta, loss_type,
        importance_sampling_level, max_completion_length, num_items))
