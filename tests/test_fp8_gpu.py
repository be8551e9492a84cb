"""Layer weights in 8 bits: quantised rows and weights, products, the gated feed-forward, experts, against the formulas in 64 bits."""
import zlib

import pytest
import torch

import fp8_util as f8

pytestmark = pytest.mark.gpu
DEV = "cuda"


def _gen(*key):
    return torch.Generator(device=DEV).manual_seed(zlib.crc32(repr(key).encode()))


def _rows(m, k, gen, dtype=torch.bfloat16):
    return (torch.randn((m, k), generator=gen, device=DEV) * (1 + 7 * (torch.rand(k, generator=gen, device=DEV) < 0.02))).to(dtype)


def _weight(*shape, gen):
    from mimirmind_b200.kernels import ops
    return ops.quantize_fp8_weight(0.05 * torch.randn(shape, generator=gen, device=DEV))


def _close(got, y, err):
    tol = f8.rounded(y, err, got.dtype)
    off = (got.double() - y).abs()
    assert bool((off <= tol).all()), f"{(off - tol).max().item():.3g} over, at {off.argmax().item()} of {tuple(y.shape)}; worst share {(off / tol).max().item():.3g}"


def _wide(w):
    return w.values.float().double() * w.scales.double().repeat_interleave(128, -2)[..., :w.shape[-2], :].repeat_interleave(128, -1)[..., :w.shape[-1]]


def _quantise_plain(x):
    """torch's own arithmetic on the same formula: bit for bit"""
    m, k = x.shape
    kb = -(-k // 128)
    pad = torch.nn.functional.pad(x.float(), (0, kb * 128 - k)).view(m, kb, 128)
    s = f8.scale(pad.abs().amax(dim=2))
    return (pad / s.unsqueeze(2)).to(torch.float8_e4m3fn).view(torch.uint8).view(m, -1)[:, :k], s


# ---- quantisation ----------------------------------------------------------------------------------------------------------
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("m,k", [(1, 1), (3, 127), (5, 129), (2, 16), (17, 1000), (300, 256), (2, 4096), (1, 18944)])
def test_rows_are_quantised_as_the_formula_says(m, k, dtype):
    from mimirmind_b200.kernels import ops
    x = _rows(m, k, _gen(m, k), dtype)
    got = ops.quantize_fp8_rows(x)
    q, s = _quantise_plain(x)
    assert torch.equal(got.scales, s) and torch.equal(got.values.view(torch.uint8), q)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("start", [0, 1, 3, 4])
def test_rows_with_a_stride_and_an_odd_start(dtype, start):
    from mimirmind_b200.kernels import ops
    wide = _rows(9, 411, _gen(start), dtype)
    x = wide[:, start:start + 300]
    q, s = _quantise_plain(x)
    got = ops.quantize_fp8_rows(x)
    assert torch.equal(got.scales, s) and torch.equal(got.values.view(torch.uint8), q)
    source = torch.tensor([8, 0, 0, 3], dtype=torch.int32, device=DEV)
    got = ops.quantize_fp8_rows(x, source)
    assert torch.equal(got.scales, s[source.long()]) and torch.equal(got.values.view(torch.uint8), q[source.long()])
    same = ops.quantize_fp8_rows(wide[2:3].expand(5, 411))            # one row for all: a stride of nought
    assert torch.equal(same.values.view(torch.uint8)[4], _quantise_plain(wide[2:3])[0][0])


def test_rows_at_the_ends_of_the_range():
    from mimirmind_b200.kernels import ops
    x = torch.zeros((7, 200), device=DEV)
    x[1] = 1e-45
    x[2] = 2.0 ** -126
    x[3, 5] = 3.4e38
    x[4, 130] = float("nan")
    x[5, 1] = float("inf")
    x[6] = -448.0
    got = ops.quantize_fp8_rows(x)
    q, s = _quantise_plain(x)
    assert torch.equal(got.scales.isnan(), s.isnan()) and torch.equal(got.scales.nan_to_num(1.0, 2.0), s.nan_to_num(1.0, 2.0))
    assert torch.equal(got.values.float().nan_to_num(1000.0), q.view(torch.float8_e4m3fn).float().nan_to_num(1000.0))
    assert ops.quantize_fp8_rows(x[:0]).shape == (0, 200)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("shape", [(1, 1), (130, 257), (3, 128, 128), (2, 2, 40, 176), (257, 1000)])
def test_weights_are_quantised_by_blocks(shape, dtype):
    from mimirmind_b200.kernels import ops
    w = (0.05 * torch.randn(shape, generator=_gen(shape), device=DEV)).to(dtype)
    got = ops.quantize_fp8_weight(w)
    n, k = shape[-2:]
    pad = torch.nn.functional.pad(w.float(), (0, -k % 128, 0, -n % 128))
    pad = pad.view(*shape[:-2], -(-n // 128), 128, -(-k // 128), 128)
    s = f8.scale(pad.abs().amax(dim=(-3, -1)))
    q = (pad / s[..., :, None, :, None]).to(torch.float8_e4m3fn).view(torch.uint8).reshape(*shape[:-2], -(-n // 128) * 128, -(-k // 128) * 128)[..., :n, :k]
    assert torch.equal(got.scales, s) and torch.equal(got.values.view(torch.uint8), q)
    assert (got.float() - w.float()).abs().max() <= 2.0 ** -4 * w.float().abs().max()


# ---- the product -----------------------------------------------------------------------------------------------------------
ROWS = [1, 2, 7, 8, 9, 16, 17, 31, 33, 64, 65, 127, 128, 129, 200, 256, 257, 400, 1000]
SIZES = [(1, 16), (130, 112), (64, 128), (257, 912), (640, 1040), (1001, 50), (3585, 272), (16, 4096)]


@pytest.mark.parametrize("n,k", SIZES)
@pytest.mark.parametrize("m", ROWS)
def test_product(m, n, k):
    from mimirmind_b200.kernels import ops
    gen = _gen(m, n, k)
    x, w = _rows(m, k, gen), _weight(n, k, gen=gen)
    y, err = f8.product(f8.quantised(x)[0], _wide(w))
    for dtype in (torch.bfloat16, torch.float32):
        _close(ops.gemm_fp8(x, w, out_dtype=dtype), y, err)
    ops.check_tcgen05_errors(torch.device(DEV))


def test_whole_rounds_of_tiles_and_a_split_rest():
    from mimirmind_b200.kernels import ops
    gen = _gen(2000)
    m, n, k = 2000, 5115, 4080              # 320 tiles of 128 x 256: two rounds of 148 and 24 more
    x, w, bias = _rows(m, k, gen), _weight(n, k, gen=gen), torch.randn(n, generator=gen, device=DEV)
    y, err = f8.product(f8.quantised(x)[0], _wide(w))
    y = y + bias.double()
    _close(ops.gemm_fp8(x, w, bias), y, err + y.abs() * 2.0 ** -24)
    _close(ops.gemm_fp8(x, w, bias, torch.float32), y, err + y.abs() * 2.0 ** -24)
    w_in, w_out = _weight(2, n // 2, k, gen=gen), _weight(200, n // 2, gen=gen)
    _close(ops.glu_mlp_fp8(x, w_in, w_out, "silu", 0.0), *_mlp64(x, w_in, w_out, "silu", 0.0))
    ops.check_tcgen05_errors(torch.device(DEV))


@pytest.mark.parametrize("m", [8, 9, 16])
def test_large_matrices_and_few_rows(m):
    from mimirmind_b200.kernels import ops
    gen = _gen(m)
    n, k = 16411, 1616                      # beyond what the weight-streaming kernel takes of more than eight rows
    x, w = _rows(m, k, gen), _weight(n, k, gen=gen)
    _close(ops.gemm_fp8(x, w), *f8.product(f8.quantised(x)[0], _wide(w)))
    w_in, w_out = _weight(2, n // 2, k, gen=gen), _weight(k, n // 2, gen=gen)
    _close(ops.glu_mlp_fp8(x, w_in, w_out, "silu", 0.0), *_mlp64(x, w_in, w_out, "silu", 0.0))
    ops.check_tcgen05_errors(torch.device(DEV))


@pytest.mark.parametrize("bias", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("m", [1, 5, 20, 130, 300, 700])
def test_product_with_a_bias_and_quantised_or_fp32_rows(m, bias):
    from mimirmind_b200.kernels import ops
    gen = _gen(m, str(bias))
    x, w = _rows(m, 400, gen, torch.float32), _weight(333, 400, gen=gen)
    b = torch.randn(333, generator=gen, device=DEV).to(bias)
    y, err = f8.product(f8.quantised(x)[0], _wide(w), b)
    got = ops.gemm_fp8(x, w, b)
    _close(got, y, err)
    assert torch.equal(ops.gemm_fp8(ops.quantize_fp8_rows(x), w, b), got)


@pytest.mark.parametrize("m", [3, 40, 200, 600])
def test_rows_that_are_no_numbers_stay_in_their_rows(m):
    from mimirmind_b200.kernels import ops
    gen = _gen(m)
    x, w = _rows(m, 528, gen), _weight(300, 528, gen=gen)
    want = ops.gemm_fp8(x, w)
    x[1, 7], x[m - 1, 527] = float("nan"), float("inf")
    got = ops.gemm_fp8(x, w)
    assert got[1].isnan().all() and got[m - 1].isnan().all()
    keep = torch.ones(m, dtype=torch.bool, device=DEV)
    keep[[1, m - 1]] = False
    assert torch.equal(got[keep], want[keep])


@pytest.mark.parametrize("m", [1, 12, 50, 140, 300])
def test_what_stands_behind_a_row_is_not_read_as_numbers(m):
    """weights cut out of a wider matrix: the bytes between rows are NaN"""
    from mimirmind_b200.kernels import ops
    gen = _gen(m)
    n, k = 200, 150
    w = _weight(n, k, gen=gen)
    wide = torch.full((n, 192), 0x7f, dtype=torch.uint8, device=DEV)
    wide[:, :k] = w.values.view(torch.uint8)
    strided = ops.Fp8Weight(wide.view(torch.float8_e4m3fn)[:, :k], w.scales)
    x = _rows(m, k, gen)
    assert torch.equal(ops.gemm_fp8(x, strided), ops.gemm_fp8(x, w))
    rows = ops.quantize_fp8_rows(x)
    wide = torch.full((m, 208), 0x7f, dtype=torch.uint8, device=DEV)
    wide[:, :k] = rows.values.view(torch.uint8)
    assert torch.equal(ops.gemm_fp8(ops.Fp8Rows(wide.view(torch.float8_e4m3fn)[:, :k], rows.scales), strided), ops.gemm_fp8(x, w))


def test_products_of_no_rows_and_of_rows_of_noughts():
    from mimirmind_b200.kernels import ops
    w = _weight(70, 130, gen=_gen(1))
    assert ops.gemm_fp8(torch.zeros((0, 130), device=DEV), w).shape == (0, 70)
    for m in (1, 40, 300):
        assert (ops.gemm_fp8(torch.zeros((m, 130), device=DEV), w) == 0).all()


@pytest.mark.parametrize("m", [1, 6, 16, 30, 100, 300, 900])
def test_a_row_does_not_depend_on_its_neighbours_or_on_the_run(m):
    """bit for bit: the same rows among others of the same step, and once more"""
    from mimirmind_b200.kernels import ops
    gen = _gen(m)
    x, w = _rows(m, 1536 + 48, gen), _weight(700, 1536 + 48, gen=gen)
    first = ops.gemm_fp8(x, w, out_dtype=torch.float32)
    other = _rows(m, 1536 + 48, gen)
    other[m // 2] = x[m // 2]
    assert torch.equal(ops.gemm_fp8(other, w, out_dtype=torch.float32)[m // 2], first[m // 2])
    assert torch.equal(ops.gemm_fp8(x, w, out_dtype=torch.float32), first)


# ---- the gated feed-forward ------------------------------------------------------------------------------------------------
def _mlp64(x, w_in, w_out, act, limit):
    gate, up = _wide(w_in)
    h, err = f8.hidden64(f8.quantised(x)[0], gate, up, act, limit)
    h, off = f8.quantised(h, err)
    return f8.product(h, _wide(w_out), off=off)


@pytest.mark.parametrize("act,limit", [("silu", 0.0), ("gelu_tanh", 0.0), ("clamped", 0.5)])
@pytest.mark.parametrize("d,f", [(64, 176), (400, 128), (272, 333), (1000, 640)])
@pytest.mark.parametrize("m", [1, 8, 16, 17, 40, 64, 128, 130, 300, 700])
def test_feed_forward(m, d, f, act, limit):
    from mimirmind_b200.kernels import ops
    gen = _gen(m, d, f)
    x, w_in, w_out = _rows(m, d, gen), _weight(2, f, d, gen=gen), _weight(d, f, gen=gen)
    _close(ops.glu_mlp_fp8(x, w_in, w_out, act, limit), *_mlp64(x, w_in, w_out, act, limit))
    ops.check_tcgen05_errors(torch.device(DEV))


# ---- experts over a prompt -------------------------------------------------------------------------------------------------
def _experts64(x, idx, wts, w_in, w_out, act, limit, on_input, quantise=True):
    m, top = idx.shape
    y = torch.zeros((m, x.shape[1]), dtype=torch.float64, device=DEV)
    err = torch.zeros_like(y)
    rows = f8.quantised(x)[0] if quantise else x.double()
    wide_in, wide_out = (_wide(w) if not isinstance(w, torch.Tensor) else w.double() for w in (w_in, w_out))
    for c in range(top):
        for e in idx[:, c].unique().tolist():
            at = (idx[:, c] == e).nonzero().flatten()
            weight = wts[at, c].double().unsqueeze(1)
            gate, up = wide_in[e][0] if wide_in.dim() == 4 else wide_in[e][:wide_in.shape[1] // 2], wide_in[e][1] if wide_in.dim() == 4 else wide_in[e][wide_in.shape[1] // 2:]
            h, off = f8.hidden64(rows[at], gate, up, act, limit, weight if on_input else None)
            if quantise:
                h, off = f8.quantised(h, off)
            part, part_err = f8.product(h, wide_out[e], off=off)
            if not on_input:
                part, part_err = part * weight, (part_err + part.abs() * 2.0 ** -22) * weight.abs()
            y[at] += part
            err[at] += part_err + part.abs() * top * 2.0 ** -22
    return y, err


@pytest.mark.parametrize("how", ["uneven", "one expert", "twice", "each its own", "input", "clamped"])
@pytest.mark.parametrize("m,d,f,experts,top", [(1, 64, 48, 4, 2), (17, 272, 176, 6, 2), (130, 400, 128, 3, 3), (300, 128, 336, 40, 4), (700, 512, 256, 5, 1)])
def test_experts_over_a_prompt(m, d, f, experts, top, how):
    from mimirmind_b200.kernels import ops
    gen = _gen(m, d, f, how)
    x, w_in, w_out = _rows(m, d, gen), _weight(experts, 2, f, d, gen=gen), _weight(experts, d, f, gen=gen)
    liking = torch.randn((m, experts), generator=gen, device=DEV)
    if how == "uneven":
        liking[:, 0] += 2.0
    idx = liking.topk(top, dim=1).indices.to(torch.int32).contiguous()
    if how == "one expert":
        idx = (torch.zeros_like(idx) + torch.arange(top, device=DEV, dtype=torch.int32)).contiguous()
    if how == "twice":
        idx[:, -1] = idx[:, 0]
    if how == "each its own":
        idx = ((torch.arange(m, device=DEV)[:, None] + torch.arange(top, device=DEV)) % experts).to(torch.int32).contiguous()
    wts = torch.rand((m, top), generator=gen, device=DEV) + 0.1
    act, limit = ("clamped", 0.7) if how == "clamped" else ("silu", 0.0)
    got = ops.moe_experts_fp8(x, idx, wts, w_in, w_out, act, limit, "input" if how == "input" else "output")
    _close(got, *_experts64(x, idx.long(), wts, w_in, w_out, act, limit, how == "input"))
    ops.check_tcgen05_errors(torch.device(DEV))


@pytest.mark.parametrize("m,d,f,experts,top", [(9, 64, 48, 4, 2), (300, 136, 64, 5, 3), (2500, 128, 64, 7, 2), (40, 100, 33, 6, 4)])
def test_a_choice_that_is_no_expert_adds_nothing(m, d, f, experts, top):
    from mimirmind_b200.kernels import ops
    gen = _gen(m, d, f)
    x, w_in, w_out = _rows(m, d, gen), _weight(experts, 2, f, d, gen=gen), _weight(experts, d, f, gen=gen)
    idx = torch.randn((m, experts), generator=gen, device=DEV).topk(top, dim=1).indices.to(torch.int32).contiguous()
    wts = torch.rand((m, top), generator=gen, device=DEV) + 0.1
    none = torch.rand((m, top), generator=gen, device=DEV) < 0.3
    none[m // 3] = True
    none[-2:] = True
    strange = torch.tensor([-1, experts, 2 ** 31 - 1, -2 ** 31], dtype=torch.int32, device=DEV)
    bad = torch.where(none, strange[torch.randint(4, (m, top), generator=gen, device=DEV)], idx).contiguous()
    x[-1] = float("nan")                    # a padded row may hold anything
    got = ops.moe_experts_fp8(x, bad, torch.where(none, torch.full_like(wts, float("nan")), wts), w_in, w_out)
    assert not bool(got[none.all(dim=1)].any())
    want, err = _experts64(x[:-1], idx[:-1].long(), wts[:-1].masked_fill(none[:-1], 0.0), w_in, w_out, "silu", 0.0, False)
    _close(got[:-1], want, err)
    nobody = torch.full_like(idx, experts)
    assert not bool(ops.moe_experts_fp8(x, nobody, wts, w_in, w_out).any())
    ops.check_tcgen05_errors(torch.device(DEV))


# ---- streams, graphs, refusals ---------------------------------------------------------------------------------------------
@pytest.mark.parametrize("m", [1, 12, 60, 300])
def test_captured_and_on_a_stream_of_its_own(m):
    from mimirmind_b200.kernels import ops
    gen = _gen(m)
    d, f, experts, top = 384, 272, 5, 2
    x = _rows(m, d, gen)
    w, w_in, w_out = _weight(500, d, gen=gen), _weight(2, f, d, gen=gen), _weight(d, f, gen=gen)
    e_in, e_out = _weight(experts, 2, f, d, gen=gen), _weight(experts, d, f, gen=gen)
    idx = torch.randn((m, experts), generator=gen, device=DEV).topk(top, dim=1).indices.to(torch.int32).contiguous()
    wts = torch.rand((m, top), generator=gen, device=DEV)

    def run():
        return ops.gemm_fp8(x, w), ops.glu_mlp_fp8(x, w_in, w_out), ops.moe_experts_fp8(x, idx, wts, e_in, e_out)

    want = run()
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        got = run()
        again = run()
    torch.cuda.current_stream().wait_stream(side)
    graphs, outs = [], []
    for _ in range(2):
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            outs.append(run())
        graphs.append(g)
    new = _rows(m, d, gen)
    x.copy_(new)
    later = run()
    for g in graphs:
        g.replay()
    graphs[0].replay()
    torch.cuda.synchronize()
    for a, b, c in zip(want, got, again):
        assert torch.equal(a, b) and torch.equal(a, c)
    for out in outs:
        for a, b in zip(later, out):
            assert torch.equal(a, b)
    ops.check_tcgen05_errors(torch.device(DEV))


FIRST_CALLS = """
import torch
from mimirmind_b200.kernels import ops
def w(*s):
    return ops.quantize_fp8_weight((0.02 * torch.randn(s, device="cuda")).bfloat16())
a, w_in, w_out, e_in, e_out = w(512, 1024), w(2, 256, 1024), w(1024, 256), w(4, 2, 64, 1024), w(4, 1024, 64)
x, router = torch.randn((40, 1024), device="cuda").bfloat16(), torch.randn((4, 1024), device="cuda")
idx, wts = torch.arange(80, device="cuda", dtype=torch.int32).view(40, 2) % 4, torch.rand((40, 2), device="cuda")
def run():
    return (ops.gemm_fp8(x, a), ops.gemm_fp8(x[:3], a), ops.glu_mlp_fp8(x, w_in, w_out), ops.glu_mlp_fp8(x[:5], w_in, w_out),
            ops.moe_experts_fp8(x, idx, wts, e_in, e_out), ops.moe_few(x[:7], router, e_in, e_out, 2))
torch.cuda.synchronize()
g = torch.cuda.CUDAGraph()
with torch.cuda.graph(g):
    got = run()
eager = run()
ops.check_tcgen05_errors("cuda")
g.replay()
torch.cuda.synchronize()
assert all(torch.equal(p, q) for p, q in zip(got, eager))
ops.check_tcgen05_errors("cuda")
print("the same")
"""


def test_first_calls_of_a_process_may_be_captured():
    import os
    import subprocess
    import sys
    root = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
    run = subprocess.run([sys.executable, "-c", FIRST_CALLS], capture_output=True, text=True, timeout=300, cwd=root, env={**os.environ, "PYTHONPATH": root})
    assert run.returncode == 0 and "the same" in run.stdout, run.stderr[-2000:]


def test_refusals():
    from mimirmind_b200.kernels import ops
    from mimirmind_b200.kernels.lib import KernelError
    w, w_in, w_out = _weight(40, 64, gen=_gen(0)), _weight(2, 48, 64, gen=_gen(1)), _weight(64, 48, gen=_gen(2))
    x = torch.zeros((3, 64), device=DEV)
    idx, wts = torch.zeros((3, 2), dtype=torch.int32, device=DEV), torch.zeros((3, 2), device=DEV)
    e_in, e_out = _weight(4, 2, 48, 64, gen=_gen(3)), _weight(4, 64, 48, gen=_gen(4))
    bad = [
        lambda: ops.gemm_fp8(x[:, :63], w),
        lambda: ops.gemm_fp8(x.half(), w),
        lambda: ops.gemm_fp8(x.cpu(), w),
        lambda: ops.gemm_fp8(x, w, out_dtype=torch.float16),
        lambda: ops.gemm_fp8(x, w, torch.zeros(39, device=DEV)),
        lambda: ops.gemm_fp8(x, w_in),
        lambda: ops.gemm_fp8(x, w.float()),
        lambda: ops.gemm_fp8(x.t().contiguous().t(), w),
        lambda: ops.Fp8Weight(w.values, w.scales[:, :0]),
        lambda: ops.Fp8Weight(w.values, w.scales.double()),
        lambda: ops.Fp8Weight(w.values.view(torch.uint8), w.scales),
        lambda: ops.Fp8Weight(w.values.view(torch.uint8).flatten()[1:1 + 39 * 64].view(torch.float8_e4m3fn).view(39, 64), w.scales),
        lambda: ops.Fp8Weight(torch.zeros((40, 60), dtype=torch.uint8, device=DEV).view(torch.float8_e4m3fn), w.scales),
        lambda: ops.Fp8Weight(e_out.values[::2], e_out.scales[::2].contiguous()),
        lambda: ops.quantize_fp8_rows(torch.zeros((2, 0), device=DEV)),
        lambda: ops.quantize_fp8_rows(x, torch.zeros(2, dtype=torch.int64, device=DEV)),
        lambda: ops.quantize_fp8_weight(x.t()),
        lambda: ops.glu_mlp_fp8(x, w_in, w_out, "relu"),
        lambda: ops.glu_mlp_fp8(x, w, w_out),
        lambda: ops.glu_mlp_fp8(x, w_in, _weight(64, 47, gen=_gen(5))),
        lambda: ops.moe_experts_fp8(x, idx, wts, e_in, w_out),
        lambda: ops.moe_experts_fp8(x, idx[:2], wts, e_in, e_out),
        lambda: ops.moe_experts_fp8(x, idx.long(), wts, e_in, e_out),
        lambda: ops.moe_experts_fp8(x, idx, wts, e_in, e_out, weight_on="both"),
    ]
    for i, call in enumerate(bad):
        with pytest.raises(KernelError):
            call()
            print("not refused:", i)
