"""The layer for a few tokens where their rows do not fit into shared memory: a cluster keeps its copy of them in memory."""
import pytest
import torch

import test_moe_few_gpu as base

pytestmark = pytest.mark.gpu
SHARED = 227 * 1024


def _shared_bytes(n, d, experts, top, fp8):
    """What the first launch takes with the rows in shared memory (csrc/moe_few.cu)"""
    pairs = n * top
    words = ((n * experts + 3) // 4 * 4 + 6 * pairs + 2 * 16 + 2 + 16 + 3) // 4 * 4
    row = 2 * (-(-d // 128) * 128 + 32) if fp8 else -(-d // 64) * 128 + 64
    return 16 * 3 * 2048 + 4 * ((2 if fp8 else 1) * 16 * 16 * 16 + words) + n * row


@pytest.mark.parametrize("fp8", [False, True])
@pytest.mark.parametrize("n,d,f,experts,top", [(16, 4096, 64, 8, 2), (16, 4104, 72, 40, 4), (13, 5000, 48, 128, 8), (8, 7424, 40, 6, 3), (3, 20000, 24, 5, 2)])
def test_rows_in_memory(n, d, f, experts, top, fp8):
    from mimirmind_b200.kernels import ops
    assert _shared_bytes(n, d, experts, top, fp8) > SHARED >= _shared_bytes(1, d, experts, top, fp8)
    gen = base._gen(n, d, f, experts, fp8)
    x, router, w_in, w_out = base._layer(n, d, f, experts, gen, fp8)
    idx, wts = base._choice64(x, router, top)
    got = ops.moe_few(x, router, w_in, w_out, top)
    base._close(got, *base._layer64(x, idx, wts, w_in, w_out, f, "silu", 0.0, False, fp8))
    for t in range(n):                       # a token alone has its row in shared memory: the same bits
        assert torch.equal(ops.moe_few(x[t:t + 1], router, w_in, w_out, top), got[t:t + 1])
    x[1, 7] = float("nan")
    beside = ops.moe_few(x, router, w_in, w_out, top)
    keep = [t for t in range(n) if t != 1]
    assert torch.equal(beside[keep], got[keep]) and not beside[1].isfinite().any()


@pytest.mark.parametrize("fp8", [False, True])
def test_rows_in_memory_captured_and_on_two_streams(fp8):
    from mimirmind_b200.kernels import ops
    gen = base._gen(fp8)
    x, router, w_in, w_out = base._layer(16, 4104, 64, 16, gen, fp8)
    want = ops.moe_few(x, router, w_in, w_out, 4)
    graphs, outs = [], []
    for _ in range(2):
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            outs.append(ops.moe_few(x, router, w_in, w_out, 4))
        graphs.append(g)
    for g in graphs:
        s = torch.cuda.Stream()
        s.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(s):
            g.replay()
            outs.append(ops.moe_few(x, router, w_in, w_out, 4))
            g.replay()
    torch.cuda.synchronize()
    assert all(torch.equal(o, want) for o in outs)
