"""Layer weights in 8 bits, and routed experts for a few tokens: cases that can be timed and compared.

Weights are held as e4m3 numbers with one 32-bit scale for every block of 128 x 128; the rows that meet them are quantised per
row and block of 128 (``s = max(fl32(largest / 448), 2^-126)``, ``q = e4m3(fl32(x / s))``).  Four operators: the product of
rows with such weights; a gated feed-forward of two of them, whose hidden rows are quantised from their 32-bit values; a whole
routed-experts layer for a few tokens (its rows are not quantised; weights in bf16 or 8 bits); routed experts in 8 bits over a prompt.

``run`` is either the plain form in elementary torch operations, or (``own``) the calls that a user of the engine's kernels makes.
"""
import math

import torch

own = False

BLOCK = 128
TOP_E4M3 = 448.0
SMALLEST = 2.0 ** -126
DEV = "cuda"


def listed():
    return [
        # the query, key and value product of a 7B decoder for one request's next token: the smallest call, latency and one weight stream
        dict(name="product-1", kind="product", m=1, n=4608, k=3584),
        # the output product of the same decoder for a serving batch
        dict(name="product-48", kind="product", m=48, n=3584, k=3584),
        # the head of a small decoder over a ragged portion: an odd number of rows, depth that ends inside a block
        dict(name="product-ragged", kind="product", m=333, n=19001, k=912),
        # the first feed-forward product of a 7B decoder over a long prompt, the largest product
        dict(name="product-4096", kind="product", m=4096, n=18944, k=3584),
        # the feed-forward of a 7B decoder for a decode step of eight requests
        dict(name="feedforward-8", kind="feedforward", m=8, d=3584, f=18944, act="silu"),
        # the same of a small decoder for one token
        dict(name="feedforward-1", kind="feedforward", m=1, d=896, f=4864, act="silu"),
        # the feed-forward of a 14B decoder over a prompt of a length that fits no tile
        dict(name="feedforward-2000", kind="feedforward", m=2000, d=5120, f=13824, act="silu"),
        # many small experts, one token: what a lone request's decode step waits for
        dict(name="few-1", kind="few", m=1, d=2048, f=768, experts=128, top=8, weights="fp8", scoring="softmax", act="silu"),
        # larger experts in bf16, a batch of eight
        dict(name="few-8-bf16", kind="few", m=8, d=2048, f=1408, experts=16, top=4, weights="bf16", scoring="softmax", act="silu"),
        # the most tokens that the layer for a few takes, nearly every expert chosen by someone
        dict(name="few-16", kind="few", m=16, d=2048, f=768, experts=128, top=8, weights="fp8", scoring="sigmoid", act="silu"),
        # routed experts over an ordinary prompt
        dict(name="experts-1500", kind="experts", m=1500, d=2048, f=1408, experts=16, top=4, act="silu"),
        # many small experts over a long prompt: unequal numbers of rows per expert, a clamped activation
        dict(name="experts-3001", kind="experts", m=3001, d=2048, f=768, experts=64, top=6, act="clamped"),
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    kind = rng.choice(["product", "product", "feedforward", "few", "few", "experts"])
    act = rng.choice(["silu", "silu", "gelu_tanh", "clamped"])
    while True:
        if kind == "product":
            case = dict(kind=kind, m=_log(rng, 1, 8192), n=_log(rng, 64, 32768), k=16 * _log(rng, 4, 1184))
        elif kind == "feedforward":
            case = dict(kind=kind, m=_log(rng, 1, 4096), d=16 * _log(rng, 4, 320), f=16 * _log(rng, 8, 1728), act=act)
        elif kind == "few":
            experts = _log(rng, 4, 160)
            case = dict(kind=kind, m=rng.randint(1, 16), d=16 * _log(rng, 8, 256), f=16 * _log(rng, 8, 172), experts=experts,
                        top=rng.randint(1, min(8, experts)), weights=rng.choice(["bf16", "fp8"]), scoring=rng.choice(["softmax", "sigmoid"]), act=act)
        else:
            experts = _log(rng, 4, 96)
            case = dict(kind=kind, m=_log(rng, 17, 4096), d=16 * _log(rng, 8, 160), f=16 * _log(rng, 8, 128), experts=experts,
                        top=rng.randint(1, min(8, experts)), act=act)
        # no more work than the listed cases of the kind, and plain forms (every chosen, or every, expert's matrices at once) that fit
        if kind == "product" and case["m"] * case["n"] * case["k"] > 4096 * 18944 * 3584:
            continue
        if kind == "feedforward" and case["m"] * case["d"] * case["f"] > 2000 * 5120 * 13824:
            continue
        if kind == "few" and (case["m"] * case["top"] * case["d"] * case["f"] > 16 * 8 * 2048 * 768
                              or case["experts"] * case["d"] * case["f"] > 128 * 2048 * 768):
            continue
        if kind == "experts" and case["m"] * case["experts"] * case["d"] * case["f"] > 3001 * 64 * 2048 * 768:
            continue
        return case


def _scale(largest):
    """fl32(largest / 448), at least 2^-126; by a tensor, since a division by a plain number may become a product with its reciprocal"""
    return torch.maximum(largest / torch.full_like(largest, TOP_E4M3), torch.full_like(largest, SMALLEST))


# ---- inputs --------------------------------------------------------------------------------------------------------------
def _rows(m, k, gen):
    """Rows as a norm leaves them: about one in size, a few channels several times as large."""
    x = torch.randn((m, k), generator=gen, device=DEV)
    loud = 1.0 + 7.0 * (torch.rand((k,), generator=gen, device=DEV) < 0.01).float()
    return (x * loud).to(torch.bfloat16)


def _weight(lead, n, k, gen):
    """(e4m3 numbers [*lead, n, k], fp32 scales [*lead, n / 128, k / 128], both counts rounded up) of a random matrix."""
    nb, kb = -(-n // BLOCK), -(-k // BLOCK)
    w = torch.zeros((*lead, nb * BLOCK, kb * BLOCK), device=DEV)
    w[..., :n, :k] = 0.02 * torch.randn((*lead, n, k), generator=gen, device=DEV)
    w = w.view(*lead, nb, BLOCK, kb, BLOCK)
    scales = _scale(w.abs().amax(dim=(-3, -1)))
    values = (w / scales[..., :, None, :, None]).to(torch.float8_e4m3fn)
    values = values.view(torch.uint8).reshape(*lead, nb * BLOCK, kb * BLOCK)[..., :n, :k].contiguous().view(torch.float8_e4m3fn)
    return values, scales.contiguous()


LIMIT = 7.0           # of the clamped activation


def prepare(case, seed):
    gen = torch.Generator(device=DEV)
    gen.manual_seed(seed)
    kind, m = case["kind"], case["m"]
    state = dict(case)
    if kind == "product":
        state["x"] = _rows(m, case["k"], gen)
        state["w"] = _weight((), case["n"], case["k"], gen)
        return state
    d, f = case["d"], case["f"]
    state["x"] = _rows(m, d, gen)
    if kind == "feedforward":
        state["w_in"] = _weight((2,), f, d, gen)           # the gate's matrix, then the up projection's
        state["w_out"] = _weight((), d, f, gen)
        return state
    experts = case["experts"]
    if kind == "few":
        state["router"] = torch.randn((experts, d), generator=gen, device=DEV) * (1.5 / math.sqrt(d))
        if case["weights"] == "bf16":
            state["w_in"] = (0.02 * torch.randn((experts, 2 * f, d), generator=gen, device=DEV)).to(torch.bfloat16)
            state["w_out"] = (0.02 * torch.randn((experts, d, f), generator=gen, device=DEV)).to(torch.bfloat16)
            return state
    else:
        # some experts are chosen far more often than others, as in a trained layer
        liking = torch.randn((m, experts), generator=gen, device=DEV) + 0.7 * torch.randn((1, experts), generator=gen, device=DEV)
        best = torch.topk(liking, case["top"], dim=1)
        state["idx"] = best.indices.to(torch.int32).contiguous()
        state["wts"] = torch.softmax(best.values, dim=1).contiguous()
    state["w_in"] = _weight((experts, 2), f, d, gen)
    state["w_out"] = _weight((experts,), d, f, gen)
    return state


# ---- the plain forms -----------------------------------------------------------------------------------------------------
def _quantised(x):
    """The rows ``x`` (32 bits) as the numbers that their quantised form stands for."""
    m, k = x.shape
    kb = -(-k // BLOCK)
    pad = torch.nn.functional.pad(x, (0, kb * BLOCK - k)).view(m, kb, BLOCK)
    s = _scale(pad.abs().amax(dim=2, keepdim=True))
    return ((pad / s).to(torch.float8_e4m3fn).float() * s).view(m, kb * BLOCK)[:, :k]


def _wide(w):
    """A weight in blocks as 32-bit numbers."""
    values, scales = w
    n, k = values.shape[-2:]
    s = scales.repeat_interleave(BLOCK, dim=-2)[..., :n, :].repeat_interleave(BLOCK, dim=-1)[..., :k]
    return values.float() * s


def _act(g, u, act):
    if act == "clamped":
        g, u = g.clamp(max=LIMIT), u.clamp(-LIMIT, LIMIT)
        return g * torch.sigmoid(1.702 * g) * (u + 1.0)
    if act == "gelu_tanh":
        return 0.5 * g * (1.0 + torch.tanh(math.sqrt(2.0 / math.pi) * (g + 0.044715 * g * g * g))) * u
    return g * torch.sigmoid(g) * u


def _plain_few(state):
    x, m, d, f, top = state["x"].float(), state["m"], state["d"], state["f"], state["top"]
    z = x.double() @ state["router"].double().t()          # in 64 bits: two experts' scores may be near one another
    s = torch.softmax(z, dim=1) if state["scoring"] == "softmax" else torch.sigmoid(z)
    order = torch.sort(s, dim=1, descending=True, stable=True)
    idx, wts = order.indices[:, :top], order.values[:, :top]
    wts = (wts / (wts.sum(dim=1, keepdim=True) + 1e-20)).float()
    chosen = idx.reshape(-1)
    if state["weights"] == "bf16":
        w_in, w_out = state["w_in"][chosen].float().view(m * top, 2, f, d), state["w_out"][chosen].float()
    else:
        w_in, w_out = (_wide((v.view(torch.uint8)[chosen].view(torch.float8_e4m3fn), s[chosen])) for v, s in (state["w_in"], state["w_out"]))
    rows = x.repeat_interleave(top, dim=0).unsqueeze(2)
    hidden = _act(torch.bmm(w_in[:, 0], rows), torch.bmm(w_in[:, 1], rows), state["act"])
    y = torch.bmm(w_out, hidden).view(m, top, d)
    return (y * wts.unsqueeze(2)).sum(dim=1).to(torch.bfloat16)


def _plain_experts(state):
    """Every expert over every row, weighted by nought where it was not chosen."""
    x = _quantised(state["x"].float())
    m, d, f, experts = state["m"], state["d"], state["f"], state["experts"]
    share = torch.zeros((m, experts), device=DEV).scatter_(1, state["idx"].long(), state["wts"])
    w_in = _wide(state["w_in"])
    g = torch.matmul(x, w_in[:, 0].transpose(1, 2))
    u = torch.matmul(x, w_in[:, 1].transpose(1, 2))
    hidden = _quantised(_act(g, u, state["act"]).view(experts * m, f)).view(experts, m, f)
    y = torch.bmm(hidden, _wide(state["w_out"]).transpose(1, 2))
    return (y * share.t().unsqueeze(2)).sum(dim=0).to(torch.bfloat16)


def run(state):
    kind = state["kind"]
    if own:
        from mimirmind_b200.kernels import ops
        x = state["x"]
        if kind == "product":
            return ops.gemm_fp8(x, ops.Fp8Weight(*state["w"]))
        limit = LIMIT if state["act"] == "clamped" else 0.0
        if kind == "feedforward":
            return ops.glu_mlp_fp8(x, ops.Fp8Weight(*state["w_in"]), ops.Fp8Weight(*state["w_out"]), state["act"], limit)
        if kind == "few":
            w_in, w_out = state["w_in"], state["w_out"]
            if state["weights"] == "fp8":
                w_in, w_out = ops.Fp8Weight(*w_in), ops.Fp8Weight(*w_out)
            return ops.moe_few(x, state["router"], w_in, w_out, state["top"], scoring=state["scoring"], renorm=True, activation=state["act"], limit=limit)
        return ops.moe_experts_fp8(x, state["idx"], state["wts"], ops.Fp8Weight(*state["w_in"]), ops.Fp8Weight(*state["w_out"]), state["act"], limit)
    if kind == "product":
        return (_quantised(state["x"].float()) @ _wide(state["w"]).t()).to(torch.bfloat16)
    if kind == "feedforward":
        x, w_in = _quantised(state["x"].float()), _wide(state["w_in"])
        hidden = _act(x @ w_in[0].t(), x @ w_in[1].t(), state["act"])
        return (_quantised(hidden) @ _wide(state["w_out"]).t()).to(torch.bfloat16)
    return _plain_few(state) if kind == "few" else _plain_experts(state)


# ---- what a pass cannot do without -----------------------------------------------------------------------------------------
def work(case):
    kind, m = case["kind"], case["m"]
    if kind == "product":
        n, k = case["n"], case["k"]
        return {"bytes": n * k + 4 * -(-n // BLOCK) * -(-k // BLOCK) + 2 * m * k + 2 * m * n, "flops": 2 * m * n * k}
    d, f = case["d"], case["f"]
    matrix = d * f + 4 * -(-d // BLOCK) * -(-f // BLOCK)
    if kind == "feedforward":
        return {"bytes": 3 * matrix + 4 * m * d, "flops": 6 * m * d * f}
    experts, top = case["experts"], case["top"]
    active = experts * (1.0 - (1.0 - top / experts) ** m)        # the experts that someone chooses, if all are liked alike
    if kind == "few":
        matrix = 2 * d * f if case["weights"] == "bf16" else matrix
        return {"bytes": int(active * 3 * matrix) + 4 * experts * d + 4 * m * d, "flops": 6 * m * top * d * f + 2 * m * experts * d}
    return {"bytes": int(active * 3 * matrix) + 4 * m * d + 8 * m * top, "flops": 6 * m * top * d * f}


# ---- the same in 64 bits ---------------------------------------------------------------------------------------------------
def _e4m3_64(v):
    """Numbers of at most 448 in size rounded to e4m3 (three bits after the first, the least exponent -6), ties to even."""
    size = v.abs()
    exponent = torch.frexp(size)[1].double() - 1.0
    step = torch.exp2(torch.clamp(exponent, min=-6.0) - 3.0)
    return torch.sign(v) * torch.clamp(torch.round(size / step) * step, max=TOP_E4M3)


def _rows_64(x):
    """The quantised rows' numbers, from 64-bit rows; the scale and the quotient are 32-bit numbers by definition."""
    out = torch.empty_like(x)
    for at in range(0, x.shape[1], BLOCK):
        part = x[:, at:at + BLOCK]
        largest = part.abs().max(dim=1, keepdim=True).values.float().double()
        s = torch.clamp((largest / TOP_E4M3).float(), min=SMALLEST)
        out[:, at:at + BLOCK] = _e4m3_64((part.float() / s).double()) * s.double()
    return out


def _matrix_64(values, scales):
    out = values.float().double()
    for i in range(scales.shape[0]):
        for j in range(scales.shape[1]):
            out[i * BLOCK:(i + 1) * BLOCK, j * BLOCK:(j + 1) * BLOCK] *= scales[i, j].double()
    return out


def _act_64(g, u, act):
    if act == "clamped":
        g, u = torch.minimum(g, torch.full_like(g, LIMIT)), torch.maximum(torch.minimum(u, torch.full_like(u, LIMIT)), torch.full_like(u, -LIMIT))
        return g / (1.0 + torch.exp(-1.702 * g)) * (u + 1.0)
    if act == "gelu_tanh":
        z = (2.0 / math.pi) ** 0.5 * (g + 0.044715 * g ** 3)
        return u * g / (1.0 + torch.exp(-2.0 * z))
    return u * g / (1.0 + torch.exp(-g))


def exact(case, seed):
    state = prepare(case, seed)
    kind, x = case["kind"], state["x"].double()
    if kind == "product":
        return _rows_64(x) @ _matrix_64(*state["w"]).t()
    act = case["act"]
    if kind == "feedforward":
        (values, scales), rows = state["w_in"], _rows_64(x)
        hidden = _act_64(rows @ _matrix_64(values[0], scales[0]).t(), rows @ _matrix_64(values[1], scales[1]).t(), act)
        return _rows_64(hidden) @ _matrix_64(*state["w_out"]).t()
    m, f, top = case["m"], case["f"], case["top"]
    y = torch.zeros_like(x)
    if kind == "few":
        z = x @ state["router"].double().t()
        s = 1.0 / (1.0 + torch.exp(-z)) if case["scoring"] == "sigmoid" else torch.exp(z - torch.logsumexp(z, dim=1, keepdim=True))
        idx = torch.argsort(s, dim=1, descending=True, stable=True)[:, :top]
        wts = torch.gather(s, 1, idx)
        wts = wts / (wts.sum(dim=1, keepdim=True) + 1e-20)
        rows = x
    else:
        idx, wts, rows = state["idx"].long(), state["wts"].double(), _rows_64(x)
    for e in torch.unique(idx).tolist():
        token, choice = torch.nonzero(idx == e, as_tuple=True)
        if kind == "few" and case["weights"] == "bf16":
            gate, up, down = state["w_in"][e, :f].double(), state["w_in"][e, f:].double(), state["w_out"][e].double()
        else:
            (vi, si), (vo, so) = state["w_in"], state["w_out"]
            gate, up, down = _matrix_64(vi[e, 0], si[e, 0]), _matrix_64(vi[e, 1], si[e, 1]), _matrix_64(vo[e], so[e])
        hidden = _act_64(rows[token] @ gate.t(), rows[token] @ up.t(), act)
        if kind == "experts":
            hidden = _rows_64(hidden)
        y.index_add_(0, token, (hidden @ down.t()) * wts[token, choice].unsqueeze(1))
    return y
