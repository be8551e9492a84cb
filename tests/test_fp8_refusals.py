"""What the 8-bit products refuse before anything reaches a device."""
import pytest
import torch


def test_tensors_of_the_host_are_refused():
    from mimirmind_b200.kernels import ops
    from mimirmind_b200.kernels.lib import KernelError
    x = torch.zeros((3, 64))
    values, scales = torch.zeros((40, 64), dtype=torch.uint8).view(torch.float8_e4m3fn), torch.zeros((1, 1))
    for call in (lambda: ops.quantize_fp8_rows(x), lambda: ops.quantize_fp8_weight(x), lambda: ops.Fp8Weight(values, scales),
                 lambda: ops.Fp8Rows(values, scales), lambda: ops.gemm_fp8(x, x), lambda: ops.glu_mlp_fp8(x, x, x),
                 lambda: ops.moe_experts_fp8(x, x, x, x, x)):
        with pytest.raises(KernelError):
            call()


def test_a_tensor_of_another_device_is_refused(monkeypatch):
    from types import SimpleNamespace

    from mimirmind_b200.kernels import ops
    from mimirmind_b200.kernels.lib import KernelError
    monkeypatch.setattr(ops.torch._C, "_cuda_getDevice", lambda: 1, raising=False)
    ops._here("op", None, SimpleNamespace(device=torch.device("cuda", 1), get_device=lambda: 1))
    with pytest.raises(KernelError, match="current device is cuda:1"):
        ops._here("op", SimpleNamespace(device=torch.device("cuda", 0), get_device=lambda: 0))


def test_sizes_whose_places_would_leave_an_int_are_refused():
    from mimirmind_b200.kernels import lib
    L, most = lib.load(verbose=False), 1 << 30
    calls = [
        lambda n: L.mm_fp8_quant_rows(None, 1, 16, None, None, 16, None, n, 16, None),
        lambda n: L.mm_fp8_quant_rows(None, 1, n, None, None, n, None, 1, n, None),
        lambda n: L.mm_fp8_quant_weight(None, 1, None, 16, None, 1, n, 16, None),
        lambda n: L.mm_fp8_linear(None, 1, 16, None, 1, None, 16, None, n, 16, None, 0, None, 1, None, None, None),
        lambda n: L.mm_fp8_linear(None, 1, 16, None, n, None, 16, None, 16, 16, None, 0, None, 1, None, None, None),
        lambda n: L.mm_fp8_linear(None, 1, n, None, 1, None, n, None, 16, n, None, 0, None, 1, None, None, None),
        lambda n: L.mm_fp8_glu_mlp(None, 1, 16, None, 1, None, 16, None, n, 16, None, n, None, 16, 0, 0.0, None, None, None, None),
        lambda n: L.mm_fp8_glu_mlp(None, 1, 16, None, 1, None, 16, None, 16, 16, None, 16, None, n, 0, 0.0, None, None, None, None),
    ]
    for call in calls:
        for n in (most, 2 ** 31 - 1):
            assert call(n) != 0
            assert b"bad sizes" in L.mm_last_error()
