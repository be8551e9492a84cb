"""Matrices of more tiles than the weight-streaming kernel has CTAs: a CTA walks over several tiles, with weights on their way across a tile's border."""
import pytest
import torch

import fp8_util as f8
import test_fp8_gpu as base

pytestmark = pytest.mark.gpu
CTAS = 2 * 148
TILED_BYTES = 24 << 20           # beyond it more than eight rows leave the streaming kernel


@pytest.mark.parametrize("k", [144, 256, 1040])
@pytest.mark.parametrize("m", [1, 3, 8, 9, 16])
def test_product_over_several_steps(m, k):
    from mimirmind_b200.kernels import ops
    n = 40003
    groups = [-(-(-(-n // 16)) // side) for side in (8, 4, 2, 1)]          # by how many tiles stand side by side in a CTA
    assert all(g > CTAS and g % CTAS for g in groups)                      # two steps at least, and not the same number for every CTA
    if m > 8:
        n = 40003 if k < 512 else 21003                                    # (of 1,040 numbers: one or two steps, by the tiles side by side)
        assert n * k <= TILED_BYTES
    gen = base._gen(m, k)
    x, w, bias = base._rows(m, k, gen), base._weight(n, k, gen=gen), torch.randn(n, generator=gen, device=base.DEV)
    y, err = f8.product(f8.quantised(x)[0], base._wide(w))
    got = ops.gemm_fp8(x, w, out_dtype=torch.float32)
    base._close(got, y, err)
    base._close(ops.gemm_fp8(x, w), y, err)
    rows = ops.quantize_fp8_rows(x)
    assert torch.equal(ops.gemm_fp8(rows, w, out_dtype=torch.float32), got)
    assert torch.equal(ops.gemm_fp8(x, w, bias, torch.float32), got + bias)
    for t in {0, m - 1}:
        assert torch.equal(ops.gemm_fp8(x[t:t + 1], w, out_dtype=torch.float32)[0], got[t])


@pytest.mark.parametrize("d", [144, 400])
@pytest.mark.parametrize("m", [1, 8, 9, 16])
def test_feed_forward_over_two_steps(m, d):
    """more than 148 blocks of hidden columns: a CTA has a block for itself, in two steps of eight tiles"""
    from mimirmind_b200.kernels import ops
    f = 19003
    assert -(-f // 128) * 2 > CTAS and 2 * f * d <= TILED_BYTES
    gen = base._gen(m, d)
    x, w_in, w_out = base._rows(m, d, gen), base._weight(2, f, d, gen=gen), base._weight(72, f, gen=gen)
    got = ops.glu_mlp_fp8(x, w_in, w_out)
    base._close(got, *base._mlp64(x, w_in, w_out, "silu", 0.0))
    assert torch.equal(ops.glu_mlp_fp8(ops.quantize_fp8_rows(x), w_in, w_out), got)
    assert torch.equal(ops.glu_mlp_fp8(x[:1], w_in, w_out), got[:1])
