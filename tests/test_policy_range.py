"""Policy-training operators: arguments at the ends of their range, on the host (every call here is refused before it
touches a device), and libraries that do not belong together."""

import ctypes as C

import pytest
import torch

from genrec_amd import _lib, policy


@pytest.mark.parametrize("temperature", [1e-45, 1e-40, 1.1e-38, -1.0, float("nan"), 1e39])
def test_temperatures_without_a_finite_inverse_are_refused(temperature):
    ids = torch.zeros(2, dtype=torch.int64)
    with pytest.raises(ValueError, match="temperature"):
        policy.token_logps(torch.zeros(2, 8), ids, temperature)
    with pytest.raises(ValueError, match="temperature"):
        policy.lm_head_token_logps(torch.zeros(2, 64, dtype=torch.bfloat16), torch.zeros(8, 64, dtype=torch.bfloat16), ids, temperature)
    lib = _lib.lib()
    a = _lib.GrxTokenLogpsArgs()
    a.logits, a.token_ids, a.logps, a.row_stats, a.grad_logits = 0x10000, 0x20000, 0x30000, 0x40000, 0x50000
    a.B, a.T, a.V, a.dtype, a.temperature, a.row_stride, a.pos_stride, a.ids_stride = 2, 3, 100, 1, temperature, 300, 100, 3
    assert lib.grx_token_logps(C.byref(a), None, 0, None) == -1 and b"temperature" in lib.grx_last_error()
    assert lib.grx_token_logps_backward(C.byref(a), None) == -1 and b"temperature" in lib.grx_last_error()
    h = _lib.GrxLmTokenLogpsArgs()
    h.hidden, h.weight, h.token_ids, h.logps, h.row_stats, h.grad_hidden = 0x10000, 0x20000, 0x30000, 0x40000, 0x50000, 0x60000
    h.N, h.H, h.V, h.temperature, h.hidden_stride, h.weight_stride = 4, 64, 100, temperature, 64, 64
    assert lib.grx_lm_token_logps(C.byref(h), None, 0, None) == -1 and b"temperature" in lib.grx_last_error()
    assert lib.grx_lm_token_logps_backward(C.byref(h), None, 0, None) == -1 and b"temperature" in lib.grx_last_error()


def test_the_smallest_temperature_is_taken():
    with pytest.raises(_lib.GenrecHipError, match="must live on the GPU"):
        policy.token_logps(torch.zeros(2, 8), torch.zeros(2, dtype=torch.int64), 2.0 ** -126)


def test_libraries_of_different_builds_are_refused(monkeypatch):
    """The number of the C ABI stays where a struct only grew: the sizes tell."""
    lib = _lib.lib()
    sizes = tuple(lib.grx_policy_struct_bytes(i) for i in range(3))
    assert sizes == tuple(C.sizeof(s) for s in (_lib.GrxTokenLogpsArgs, _lib.GrxLmTokenLogpsArgs, _lib.GrxPolicyLossArgs))
    assert lib.grx_policy_struct_bytes(3) == 0 and lib.grx_policy_struct_bytes(-1) == 0
    ops = policy._ops()
    assert ops.struct_bytes == sizes
    monkeypatch.setattr(policy, "_ops_module", None)
    monkeypatch.setattr(ops, "struct_bytes", (sizes[0], sizes[1] - 8, sizes[2]))
    with pytest.raises(_lib.GenrecHipError, match="different builds"):
        policy.token_logps(torch.zeros(2, 8), torch.zeros(2, dtype=torch.int64))
