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


@pytest.mark.parametrize("N,H,V", [(1, 64, 1), (5, 2048, 152640), (64, 2048, 152640), (100, 128, 151669), (320, 2048, 152640), (400, 1536, 152640),
                                   (1403, 3584, 151669), (8192, 2048, 152640), (1 << 21, 64, 1000), (1 << 23, 64, 1000)])
def test_scratch_sizes_are_what_the_header_says(N, H, V):
    lib = _lib.lib()
    up = lambda n, to: (n + to - 1) // to * to
    columns, small = up(V, 256), 16 << 10  # small: what is rounded up to 256 bytes
    per_row = lambda bn: columns * {64: 1 / 4, 128: 1 / 8, 192: 1 / 8, 256: 1 / 16}[bn]
    for entropy in (0, 1):
        most = max(up(N, bn) * per_row(bn) for bn in (64, 128, 192, 256)) * (1.5 if entropy else 1)
        least = min(up(N, bn) * per_row(bn) for bn in (64, 128, 192, 256)) * (1.5 if entropy else 1)
        have = lib.grx_lm_token_logps_scratch_bytes(N, H, V, entropy) - 2 * N * H
        assert least <= have <= most + 16 * N + small
    chunk = max(1 << 30, 4 * up(N, 64) * 256)
    for want_h, want_w in ((1, 0), (0, 1), (1, 1)):
        copies = (2 + 2 * want_w) * up(N, 64) * H
        have = lib.grx_lm_token_logps_backward_scratch_bytes(N, H, V, want_h, want_w)
        assert have <= copies + chunk + want_h * 64 * up(N, 256) * H * 4 + 64 * N + small
    assert lib.grx_lm_token_logps_kept_bytes(N, V) <= up(N, 256) * columns * 4
