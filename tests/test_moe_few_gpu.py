"""A routed-experts layer for a few tokens in two launches, against its formula in 64 bits and against the layer's five kernels."""
import zlib

import pytest
import torch

import fp8_util as f8

pytestmark = pytest.mark.gpu
DEV = "cuda"


def _gen(*key):
    return torch.Generator(device=DEV).manual_seed(zlib.crc32(repr(key).encode()))


def _layer(n, d, f, experts, gen, fp8, spread=1.5):
    from mimirmind_b200.kernels import ops
    x = (torch.randn((n, d), generator=gen, device=DEV) * (1 + 7 * (torch.rand(d, generator=gen, device=DEV) < 0.02))).to(torch.bfloat16)
    router = torch.randn((experts, d), generator=gen, device=DEV) * (spread / d ** 0.5)
    w_in, w_out = 0.05 * torch.randn((experts, 2, f, d), generator=gen, device=DEV), 0.05 * torch.randn((experts, d, f), generator=gen, device=DEV)
    if fp8:
        return x, router, ops.quantize_fp8_weight(w_in), ops.quantize_fp8_weight(w_out)
    return x, router, w_in.to(torch.bfloat16).view(experts, 2 * f, d), w_out.to(torch.bfloat16)


def _wide(w):
    if isinstance(w, torch.Tensor):
        return w.double()
    return w.values.float().double() * w.scales.double().repeat_interleave(128, -2)[..., :w.shape[-2], :].repeat_interleave(128, -1)[..., :w.shape[-1]]


def _choice64(x, router, top, groups=1, keep=1, scoring="softmax", renorm=True, scale=1.0, correction=None, pair_sum=False):
    z = x.double() @ router.double().t()
    s = torch.softmax(z, 1) if scoring == "softmax" else torch.sigmoid(z)
    c = s if correction is None else s + correction.double()
    if keep < groups:
        runs = c.view(c.shape[0], groups, -1)
        best = runs.topk(2, dim=2).values.sum(2) if pair_sum and runs.shape[2] > 1 else runs.amax(2)
        kept = torch.zeros_like(best).scatter_(1, torch.sort(best, dim=1, descending=True, stable=True).indices[:, :keep], 1.0)
        c = torch.where(kept.repeat_interleave(runs.shape[2], 1) > 0, c, torch.full_like(c, -float("inf")))
    idx = torch.sort(c, dim=1, descending=True, stable=True).indices[:, :top]
    w = s.gather(1, idx)
    if renorm:
        w = w / (w.sum(1, keepdim=True) + 1e-20)
    return idx, w * scale


def _layer64(x, idx, wts, w_in, w_out, f, act, limit, on_input, fp8):
    """The result and what it may be off by: the sums' errors (f8.sum_error; its 128 a block covers the products' own order), x in two e4m3 parts (2^-21
    of its largest), hidden rows in two bf16 parts (2^-17) or fp16 (half a step is 2^-12 of a number; 2^-38 of the row's largest below), weights and score in fp32
    (2^-18 with the router's sums)."""
    y = torch.zeros(x.shape, dtype=torch.float64, device=DEV)
    err = torch.zeros_like(y)
    wide_in, wide_out = _wide(w_in).view(-1, 2, f, x.shape[1]), _wide(w_out)
    for t in range(x.shape[0]):
        for c in range(idx.shape[1]):
            e, w = idx[t, c], wts[t, c]
            row = x[t:t + 1].double()
            h, off = f8.hidden64(row, wide_in[e][0], wide_in[e][1], act, limit, w.view(1, 1) if on_input else None,
                                off=torch.full_like(row, row.abs().max().item() * 2.0 ** -21) if fp8 else None)
            off = off + (h.abs() * 2.0 ** -12 + h.abs().amax() * 2.0 ** -38 if fp8 else h.abs() * 2.0 ** -17) + (h.abs() + off) * (2.0 ** -18 if on_input else 0.0)
            part, part_err = f8.product(h, wide_out[e], off=off)
            if not on_input:
                part, part_err = part * w, part_err * w.abs() + (part * w).abs() * 2.0 ** -18
            y[t] += part[0]
            err[t] += part_err[0] + part[0].abs() * idx.shape[1] * 2.0 ** -22
    return y, err


def _close(got, y, err):
    tol = f8.rounded(y, err, got.dtype)
    off = (got.double() - y).abs()
    assert bool((off <= tol).all()), f"{(off - tol).max().item():.3g} over; worst share {(off / tol).max().item():.3g}"


SHAPES = [(64, 48, 4, 2), (128, 136, 8, 1), (272, 176, 6, 6), (520, 64, 40, 8), (2048, 256, 128, 8), (1024, 72, 300, 3), (24, 8, 2, 1)]


@pytest.mark.parametrize("fp8", [False, True])
@pytest.mark.parametrize("d,f,experts,top", SHAPES)
@pytest.mark.parametrize("n", [1, 2, 5, 8, 9, 16])
def test_layer(n, d, f, experts, top, fp8):
    from mimirmind_b200.kernels import ops
    gen = _gen(n, d, f, experts, top, fp8)
    x, router, w_in, w_out = _layer(n, d, f, experts, gen, fp8)
    idx, wts = _choice64(x, router, top)
    _close(ops.moe_few(x, router, w_in, w_out, top), *_layer64(x, idx, wts, w_in, w_out, f, "silu", 0.0, False, fp8))


OPTIONS = {
    "sigmoid": dict(scoring="sigmoid"), "renormed sigmoid": dict(scoring="sigmoid", renorm=True, scale=2.5), "plain softmax": dict(renorm=False),
    "groups": dict(groups=4, keep=2), "pairs": dict(groups=4, keep=1, group_score="top2_sum"), "correction": dict(correction=True, scoring="sigmoid"),
    "gelu": dict(activation="gelu_tanh"), "clamped": dict(activation="clamped", limit=0.7), "input": dict(weight_on="input", scoring="sigmoid", renorm=False),
}


@pytest.mark.parametrize("fp8", [False, True])
@pytest.mark.parametrize("what", sorted(OPTIONS))
@pytest.mark.parametrize("n", [3, 13])
def test_options(n, what, fp8):
    from mimirmind_b200.kernels import ops
    d, f, experts, top = 256, 144, 16, 3
    gen = _gen(n, what, fp8)
    x, router, w_in, w_out = _layer(n, d, f, experts, gen, fp8)
    opt = dict(OPTIONS[what])
    if opt.get("correction"):
        opt["correction"] = 0.3 * torch.randn(experts, generator=gen, device=DEV)
    scoring = opt.get("scoring", "softmax")
    idx, wts = _choice64(x, router, top, opt.get("groups", 1), opt.get("keep", 1), scoring, opt.get("renorm", scoring == "softmax"), opt.get("scale", 1.0),
                         opt.get("correction"), opt.get("group_score") == "top2_sum")
    got = ops.moe_few(x, router, w_in, w_out, top, **opt)
    _close(got, *_layer64(x, idx, wts, w_in, w_out, f, opt.get("activation", "silu"), opt.get("limit", 0.0), opt.get("weight_on") == "input", fp8))


def test_interleaved_gate_and_up_rows():
    from mimirmind_b200.kernels import ops
    n, d, f, experts = 7, 192, 64, 6
    x, router, w_in, w_out = _layer(n, d, f, experts, _gen(3), False)
    woven = w_in.view(experts, 2, f // 8, 8, d).transpose(1, 2).reshape(experts, 2 * f, d).contiguous()
    assert torch.equal(ops.moe_few(x, router, woven, w_out, 2, interleaved=True), ops.moe_few(x, router, w_in, w_out, 2))


@pytest.mark.parametrize("fp8", [False, True])
@pytest.mark.parametrize("n", [2, 16])
def test_everyone_on_one_expert_and_experts_that_are_no_numbers(n, fp8):
    from mimirmind_b200.kernels import ops
    d, f, experts = 256, 80, 12
    x, router, w_in, w_out = _layer(n, d, f, experts, _gen(n, fp8), fp8)
    x[:, 0] = 1.0
    router.zero_()
    router[5, 0] = 9.0                      # every token's first choice is expert 5, the second (all alike) the lowest number
    got = ops.moe_few(x, router, w_in, w_out, 2)
    idx, wts = _choice64(x, router, 2)
    assert idx.tolist() == [[5, 0]] * n
    _close(got, *_layer64(x, idx, wts, w_in, w_out, f, "silu", 0.0, False, fp8))
    # the experts that nobody chose are not looked at
    for w in (w_in, w_out):
        if fp8:
            w.values.view(torch.uint8)[[1, 2, 3, 4, 6, 7, 8, 9, 10, 11]] = 0x7f
        else:
            w[[1, 2, 3, 4, 6, 7, 8, 9, 10, 11]] = float("nan")
    assert torch.equal(ops.moe_few(x, router, w_in, w_out, 2), got)


@pytest.mark.parametrize("fp8", [False, True])
@pytest.mark.parametrize("n", [4, 16])
def test_a_token_does_not_depend_on_its_neighbours(n, fp8):
    """bit for bit: alone, and beside one whose row is no number"""
    from mimirmind_b200.kernels import ops
    x, router, w_in, w_out = _layer(n, 512, 272, 24, _gen(n, fp8), fp8)
    whole = ops.moe_few(x, router, w_in, w_out, 4)
    for t in range(n):
        assert torch.equal(ops.moe_few(x[t:t + 1], router, w_in, w_out, 4), whole[t:t + 1])
    x[1, 3] = float("nan")
    x[2, 9] = float("inf")
    got = ops.moe_few(x, router, w_in, w_out, 4)
    assert not got[1].isfinite().any() and not got[2].isfinite().any()
    keep = [t for t in range(n) if t not in (1, 2)]
    assert torch.equal(got[keep], whole[keep])


@pytest.mark.parametrize("size", [1e-30, 1e-4, 1e4, 1e18])
def test_rows_of_any_size_in_8_bit_experts(size):
    """the powers of two in front of the parts follow the rows: scaling x and the router's rows against one another changes nothing but the scale of a linear layer"""
    from mimirmind_b200.kernels import ops
    n, d, f, experts = 5, 128, 64, 4
    x, router, w_in, w_out = _layer(n, d, f, experts, _gen(11), True)
    x = (x.float() * size).to(torch.bfloat16)
    router = router / size
    idx, wts = _choice64(x, router, 2)
    got = ops.moe_few(x, router, w_in, w_out, 2, activation="gelu_tanh")
    y, err = _layer64(x, idx, wts, w_in, w_out, f, "gelu_tanh", 0.0, False, True)
    fine = y.abs() < 1e37
    tol = f8.rounded(y, err, got.dtype) + 2.0 ** -133          # (bf16's own smallest step)
    assert bool(((got.double() - y).abs() <= tol)[fine].all())


def test_captured_twice_and_on_a_stream_of_its_own():
    from mimirmind_b200.kernels import ops
    x, router, w_in, w_out = _layer(6, 256, 144, 16, _gen(1), True)
    x2, router2, v_in, v_out = _layer(11, 256, 144, 16, _gen(2), False)

    def run():
        return ops.moe_few(x, router, w_in, w_out, 3), ops.moe_few(x2, router2, v_in, v_out, 3)

    want = run()
    side, other = torch.cuda.Stream(), torch.cuda.Stream()
    graphs, outs = [], []
    for _ in range(2):
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            outs.append(run())
        graphs.append(g)
    for s, g in zip((side, other), graphs):
        s.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(s):
            for _ in range(3):
                g.replay()
            eager = run()
    torch.cuda.synchronize()
    for out in outs + [eager]:
        for a, b in zip(want, out):
            assert torch.equal(a, b)


def test_no_rows_and_strided_rows():
    from mimirmind_b200.kernels import ops
    x, router, w_in, w_out = _layer(4, 256, 64, 8, _gen(5), True)
    assert ops.moe_few(x[:0], router, w_in, w_out, 2).shape == (0, 256)
    wide = torch.full((4, 280), float("nan"), dtype=torch.bfloat16, device=DEV)
    wide[:, 8:264] = x
    assert torch.equal(ops.moe_few(wide[:, 8:264], router, w_in, w_out, 2), ops.moe_few(x, router, w_in, w_out, 2))


def test_one_row_of_any_stride_and_two_streams_at_once():
    from mimirmind_b200.kernels import ops
    x, router, w_in, w_out = _layer(3, 256, 64, 8, _gen(8), True)
    want = ops.moe_few(x, router, w_in, w_out, 2)
    row = x[1].clone().as_strided((1, 256), (7, 1))              # a single row's stride is nobody's business
    assert torch.equal(ops.moe_few(row, router, w_in, w_out, 2)[0], want[1])
    streams = [torch.cuda.Stream() for _ in range(2)]
    outs = []
    for s in streams:
        s.wait_stream(torch.cuda.current_stream())
    for _ in range(5):
        for s in streams:
            with torch.cuda.stream(s):
                outs.append(ops.moe_few(x, router, w_in, w_out, 2))
    torch.cuda.synchronize()
    assert all(torch.equal(o, want) for o in outs)


def test_refusals():
    from mimirmind_b200.kernels import ops
    from mimirmind_b200.kernels.lib import KernelError
    x, router, w_in, w_out = _layer(4, 64, 32, 8, _gen(6), False)
    q, _, q_in, q_out = _layer(4, 64, 32, 8, _gen(6), True)
    big = torch.zeros((17, 64), dtype=torch.bfloat16, device=DEV)
    for i, call in enumerate([
        lambda: ops.moe_few(big, router, w_in, w_out, 2),
        lambda: ops.moe_few(x.float(), router, w_in, w_out, 2),
        lambda: ops.moe_few(x, router.bfloat16(), w_in, w_out, 2),
        lambda: ops.moe_few(x, router[:, :32].contiguous(), w_in, w_out, 2),
        lambda: ops.moe_few(x, router, w_in, w_out, 0),
        lambda: ops.moe_few(x, router, w_in, w_out, 9),
        lambda: ops.moe_few(x, router, w_in, w_out, 3, groups=4, keep=1),
        lambda: ops.moe_few(x, router, w_in, w_out, 2, groups=3, keep=1),
        lambda: ops.moe_few(x, router, w_in, q_out, 2),
        lambda: ops.moe_few(x, router, q_in, w_out, 2),
        lambda: ops.moe_few(x, router, q_in, q_out, 2, interleaved=True),
        lambda: ops.moe_few(x, router, w_in, w_out, 2, activation="relu"),
        lambda: ops.moe_few(x, router, w_in, w_out, 2, scoring="max"),
        lambda: ops.moe_few(x, router, w_in, w_out, 2, weight_on="both"),
        lambda: ops.moe_few(x, router, w_in, w_out, 2, correction=torch.zeros(7, device=DEV)),
        lambda: ops.moe_few(big.flatten()[1:257].view(4, 64), router, w_in, w_out, 2),
        lambda: ops.moe_few(x, router, w_in.transpose(1, 2), w_out, 2),
    ]):
        with pytest.raises(KernelError):
            call()
            print("not refused:", i)


@pytest.mark.parametrize("rows,top,experts", [(4095, 1, 64), (4096, 2, 64), (5001, 3, 7), (20000, 8, 300), (90000, 6, 128), (9000, 4, 1), (70000, 8, 600)])
def test_rows_sorted_by_expert_over_a_cluster(rows, top, experts):
    """many rows: the lists that torch's stable sort gives"""
    from mimirmind_b200.kernels import ops
    n = rows // top
    gen = _gen(rows, top)
    idx = (torch.randint(0, experts, (n, top), generator=gen, device=DEV) * torch.randint(0, 2, (n, top), generator=gen, device=DEV)).to(torch.int32)      # half on expert 0
    got = ops.moe_sort(idx, experts, with_tiles=True)
    flat = idx.flatten().long()
    order = torch.sort(flat, stable=True).indices
    counts = torch.bincount(flat, minlength=experts)
    starts = torch.cumsum(counts, 0) - counts
    assert torch.equal(got.order[:n * top].long(), order) and torch.equal(got.offsets[:-1].long(), starts) and int(got.offsets[-1]) == n * top
    assert torch.equal(got.row_token.long(), order // top) and torch.equal(got.place.long()[order], torch.arange(n * top, device=DEV))
    want = [(s + i, min(s + i + 128, s + c), e) for e, (s, c) in enumerate(zip(starts.tolist(), counts.tolist())) for i in range(0, c, 128)]
    assert int(got.n_tiles) == len(want) and [tuple(t) for t in got.tiles[:len(want)].tolist()] == want
