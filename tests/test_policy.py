"""Policy-training operators: argument checks, on the host (no kernel is launched: every call here is refused
by the Python entry points or by the C entry points before they touch a device)."""

import ctypes as C

import pytest
import torch

from genrec_amd import _lib, policy


def _loss(**over):
    args = dict(logps=torch.zeros(2, 3), advantages=torch.zeros(2), mask=torch.ones(2, 3))
    args.update(over)
    return policy.policy_loss(args.pop("logps"), args.pop("advantages"), args.pop("mask"), **args)


@pytest.mark.parametrize("over,error,match", [
    (dict(logps=torch.zeros(6)), ValueError, "rows, positions"),
    (dict(mask=torch.ones(2, 4)), ValueError, "mask must have the shape"),
    (dict(old_logps=torch.zeros(2, 2)), ValueError, "old_logps must have the shape"),
    (dict(ref_logps=torch.zeros(3, 3)), ValueError, "ref_logps must have the shape"),
    (dict(advantages=torch.zeros(3)), ValueError, "advantages must be"),
    (dict(advantages=torch.zeros(2, dtype=torch.int64)), TypeError, "advantages must be floating"),
    (dict(loss_type="ppo"), ValueError, "loss_type"),
    (dict(importance_sampling_level="row"), ValueError, "importance_sampling_level"),
    (dict(epsilon_low=1.0), ValueError, "epsilon_low"),
    (dict(epsilon_low=float("nan")), ValueError, "epsilon_low"),
    (dict(epsilon_high=-0.1), ValueError, "epsilon_high"),
    (dict(delta=1.2), ValueError, "delta"),
    (dict(beta=float("inf")), ValueError, "beta"),
    (dict(beta=0.1), ValueError, "ref_logps"),
    (dict(loss_type="dr_grpo"), ValueError, "max_completion_length"),
    (dict(loss_type="dapo", num_items=0), ValueError, "num_items"),
    (dict(), _lib.GenrecHipError, "must live on the GPU"),
])
def test_policy_loss_refuses(over, error, match):
    with pytest.raises(error, match=match):
        _loss(**over)


@pytest.mark.parametrize("logits,ids,options,error,match", [
    (torch.zeros(2, 3, 8), torch.zeros(2, 2, dtype=torch.int64), {}, ValueError, "one row per token"),
    (torch.zeros(8), torch.zeros((), dtype=torch.int64), {}, ValueError, "one row per token"),
    (torch.zeros(2, 8), torch.zeros(2), {}, TypeError, "integers"),
    (torch.zeros(2, 8, dtype=torch.float64), torch.zeros(2, dtype=torch.int64), {}, TypeError, "unsupported logits dtype"),
    (torch.zeros(2, 0), torch.zeros(2, dtype=torch.int64), {}, ValueError, "empty"),
    (torch.zeros(2, 8), torch.zeros(2, dtype=torch.int64), {"temperature": 0.0}, ValueError, "temperature"),
    (torch.zeros(2, 8), torch.zeros(2, dtype=torch.int64), {"temperature": float("inf")}, ValueError, "temperature"),
    (torch.zeros(1, 8).expand(policy.MAX_ROWS + 1, 8), torch.zeros(1, dtype=torch.int64).expand(policy.MAX_ROWS + 1), {},
     ValueError, "at most"),
    (torch.zeros(2, 8), torch.zeros(2, dtype=torch.int64), {}, _lib.GenrecHipError, "must live on the GPU"),
])
def test_token_logps_refuses(logits, ids, options, error, match):
    with pytest.raises(error, match=match):
        policy.token_logps(logits, ids, **options)


def _token_args(**over):
    a = _lib.GrxTokenLogpsArgs()
    a.logits, a.token_ids, a.logps, a.row_stats, a.grad_logits = 0x10000, 0x20000, 0x30000, 0x40000, 0x50000
    a.B, a.T, a.V, a.dtype, a.temperature, a.row_stride, a.pos_stride, a.ids_stride = 2, 3, 100, 1, 1.0, 300, 100, 3
    for k, v in over.items():
        setattr(a, k, v)
    return a


@pytest.mark.parametrize("over,code,match", [
    (dict(V=0), -1, b"bad shape"),
    (dict(dtype=7), -3, b"dtype"),
    (dict(temperature=0.0), -1, b"temperature"),
    (dict(temperature=float("nan")), -1, b"temperature"),
    (dict(logits=None), -1, b"null buffer"),
    (dict(row_stats=None), -1, b"null buffer"),
    (dict(logits=0x10001), -1, b"misaligned"),
    (dict(row_stats=0x40004), -1, b"misaligned"),
    (dict(B=1 << 22, T=3), -3, b"rows"),
    (dict(V=(1 << 24) + 1), -3, b"vocabulary"),
])
def test_token_logps_c_entries_refuse(over, code, match):
    lib = _lib.lib()
    a = _token_args(**over)
    assert lib.grx_token_logps(C.byref(a), None, 0, None) == code and match in lib.grx_last_error()
    assert lib.grx_token_logps_backward(C.byref(a), None) == code and match in lib.grx_last_error()


def test_token_logps_c_entries_refuse_what_only_one_direction_needs():
    lib = _lib.lib()
    assert lib.grx_token_logps(None, None, 0, None) == -1
    a = _token_args(logps=None)
    assert lib.grx_token_logps(C.byref(a), None, 0, None) == -1 and b"null logps" in lib.grx_last_error()
    a = _token_args(V=152640)
    need = lib.grx_token_logps_scratch_bytes(6, 152640, 1)
    assert need > 0
    assert lib.grx_token_logps(C.byref(a), 0x60000, need - 1, None) == -4 and b"scratch" in lib.grx_last_error()
    assert lib.grx_token_logps(C.byref(a), 0x60008, need, None) == -1 and b"misaligned scratch" in lib.grx_last_error()
    a = _token_args(grad_logits=None)
    assert lib.grx_token_logps_backward(C.byref(a), None) == -1 and b"grad_logits" in lib.grx_last_error()
    a = _token_args(grad_entropy=0x60000)
    assert lib.grx_token_logps_backward(C.byref(a), None) == -1 and b"entropies" in lib.grx_last_error()
    a = _token_args(B=0)  # nothing to do: accepted without buffers
    a.logits = None
    assert lib.grx_token_logps(C.byref(a), None, 0, None) == 0 and lib.grx_token_logps_backward(C.byref(a), None) == 0


@pytest.mark.parametrize("over,code,match", [
    (dict(R=-1), -1, b"bad shape"),
    (dict(T=(1 << 30) + 1), -3, b"positions"),
    (dict(loss=None), -1, b"null output"),
    (dict(mask=None), -1, b"null input"),
    (dict(mask_type=4), -1, b"mask type"),
    (dict(epsilon_low=1.0), -1, b"epsilon_low"),
    (dict(epsilon_high=float("inf")), -1, b"epsilon_high"),
    (dict(delta=1.1), -1, b"delta"),
    (dict(beta=0.1), -1, b"reference"),
    (dict(normalizer=-1.0), -1, b"normalizer"),
    (dict(unit_grad=0x50004), -1, b"misaligned"),
    (dict(R=5000, T=5), -4, b"scratch"),
])
def test_policy_loss_c_entry_refuses(over, code, match):
    lib = _lib.lib()
    a = _lib.GrxPolicyLossArgs()
    a.logps, a.advantages, a.mask, a.loss, a.stats, a.unit_grad = 0x10000, 0x20000, 0x30000, 0x40000, 0x40010, 0x50000
    a.R, a.T, a.mask_type, a.epsilon_low, a.epsilon_high = 2, 3, 2, 0.2, 0.2
    for k, v in over.items():
        setattr(a, k, v)
    assert lib.grx_policy_loss(C.byref(a), None, 0, None) == code and match in lib.grx_last_error()


def test_policy_loss_backward_c_entry_refuses():
    lib = _lib.lib()
    assert lib.grx_policy_loss_backward(None, None, None, 0, None, None) == 0
    assert lib.grx_policy_loss_backward(0x10000, 0x20000, None, 5, 0x30000, None) == -1
    assert lib.grx_policy_loss_backward(0x10004, 0x20000, 0x20010, 5, 0x30000, None) == -1
    assert b"misaligned" in lib.grx_last_error()


def _bf(*shape):
    return torch.zeros(*shape, dtype=torch.bfloat16)


@pytest.mark.parametrize("hidden,weight,ids,error,match", [
    (torch.zeros(2, 64), _bf(8, 64), torch.zeros(2, dtype=torch.int64), TypeError, "bfloat16"),
    (_bf(2, 64), _bf(8, 64).float(), torch.zeros(2, dtype=torch.int64), TypeError, "bfloat16"),
    (_bf(2, 64), _bf(8, 64), torch.zeros(3, dtype=torch.int64), ValueError, "one row per token"),
    (_bf(2, 64), _bf(8, 128), torch.zeros(2, dtype=torch.int64), ValueError, "weight must be"),
    (_bf(2, 64), _bf(0, 64), torch.zeros(2, dtype=torch.int64), ValueError, "weight must be"),
    (_bf(2, 96), _bf(8, 96), torch.zeros(2, dtype=torch.int64), ValueError, "multiple of 64"),
    (_bf(2, 0), _bf(8, 0), torch.zeros(2, dtype=torch.int64), ValueError, "multiple of 64"),
    (_bf(2, 64), _bf(8, 64), torch.zeros(2), TypeError, "integers"),
    (_bf(2, 64), _bf(8, 64), torch.zeros(2, dtype=torch.int64), _lib.GenrecHipError, "must live on the GPU"),
])
def test_lm_head_token_logps_refuses(hidden, weight, ids, error, match):
    with pytest.raises(error, match=match):
        policy.lm_head_token_logps(hidden, weight, ids)


def test_lm_head_token_logps_refuses_a_negative_budget():
    with pytest.raises(ValueError, match="keep_bytes"):
        policy.lm_head_token_logps(_bf(2, 64), _bf(8, 64), torch.zeros(2, dtype=torch.int64), keep_bytes=-1)


@pytest.mark.parametrize("over,code,match", [
    (dict(V=0), -1, b"bad shape"),
    (dict(H=96), -3, b"multiple of 64"),
    (dict(H=1 << 17, hidden_stride=1 << 17, weight_stride=1 << 17), -3, b"2^16"),
    (dict(N=(1 << 23) + 1), -3, b"rows"),
    (dict(temperature=-1.0), -1, b"temperature"),
    (dict(hidden_stride=100), -1, b"operand rows"),
    (dict(weight_stride=56), -1, b"operand rows"),
    (dict(weight=None), -1, b"null buffer"),
    (dict(hidden=0x10008), -1, b"misaligned"),
    (dict(kept=0x70004), -1, b"misaligned"),
    (dict(N=(1 << 20) + 1, kept=0x70000), -3, b"kept"),
])
def test_lm_head_c_entries_refuse(over, code, match):
    lib = _lib.lib()
    a = _lib.GrxLmTokenLogpsArgs()
    a.hidden, a.weight, a.token_ids, a.logps, a.row_stats, a.grad_hidden = 0x10000, 0x20000, 0x30000, 0x40000, 0x50000, 0x60000
    a.N, a.H, a.V, a.temperature, a.hidden_stride, a.weight_stride = 4, 64, 100, 1.0, 64, 64
    for k, v in over.items():
        setattr(a, k, v)
    assert lib.grx_lm_token_logps(C.byref(a), None, 0, None) == code and match in lib.grx_last_error()
    assert lib.grx_lm_token_logps_backward(C.byref(a), None, 0, None) == code and match in lib.grx_last_error()


def test_lm_head_c_entries_refuse_short_scratch():
    lib = _lib.lib()
    a = _lib.GrxLmTokenLogpsArgs()
    a.hidden, a.weight, a.token_ids, a.logps, a.row_stats, a.grad_hidden = 0x10000, 0x20000, 0x30000, 0x40000, 0x50000, 0x60000
    a.N, a.H, a.V, a.temperature, a.hidden_stride, a.weight_stride = 4, 64, 100, 1.0, 64, 64
    n = lib.grx_lm_token_logps_scratch_bytes(4, 64, 100, 0)
    assert n > 0 and lib.grx_lm_token_logps(C.byref(a), 0x70000, n - 1, None) == -4
    n = lib.grx_lm_token_logps_backward_scratch_bytes(4, 64, 100, 1, 0)
    assert n > 0 and lib.grx_lm_token_logps_backward(C.byref(a), 0x70000, n - 1, None) == -4
    a.grad_entropy = 0x80000
    assert lib.grx_lm_token_logps_backward(C.byref(a), 0x70000, n, None) == -1 and b"entropies" in lib.grx_last_error()
