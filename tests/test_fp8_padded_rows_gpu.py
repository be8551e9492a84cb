"""Rows in 8 bits made from others: a number that is no row's, as a padded batch has, gives noughts."""
import pytest
import torch

pytestmark = pytest.mark.gpu
DEV = "cuda"


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("k", [5, 256, 1003])
def test_numbers_that_are_no_rows(k, dtype):
    from mimirmind_b200.kernels import ops
    gen = torch.Generator(device=DEV).manual_seed(k)
    x = torch.randn((6, k), generator=gen, device=DEV).to(dtype)
    source = torch.tensor([5, -1, 0, 6, 2 ** 31 - 1, 0, -2 ** 31, 3], dtype=torch.int32, device=DEV)
    got = ops.quantize_fp8_rows(x, source)
    whole = ops.quantize_fp8_rows(x)
    for r, s in enumerate(source.tolist()):
        if 0 <= s < 6:
            assert torch.equal(got.values[r].view(torch.uint8), whole.values[s].view(torch.uint8)) and torch.equal(got.scales[r], whole.scales[s])
        else:
            assert not bool(got.values[r].view(torch.uint8).any()) and bool((got.scales[r] == 2.0 ** -126).all())
    assert ops.quantize_fp8_rows(x, source[:0]).shape == (0, k)
