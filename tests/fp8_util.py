"""Layer weights in 8 bits in plain torch, in 64 bits, with what a result may be off by.

Half a step of a rounding is 2^-4 of the value in e4m3 and 2^-8 in bf16.  A hidden row that is quantised from sums in fp32 may
round the other way than the same from sums in 64 bits where the quotient stands within the sums' error of the middle of two
e4m3 numbers: ``quantised`` says for every number how far off that can put it.
"""
import torch

BLOCK = 128


def scale(largest):
    """by a tensor: torch turns a division by a plain number into a product with its reciprocal"""
    return (largest / torch.full_like(largest, 448.0)).clamp_min(2.0 ** -126)


def _e4m3(v):
    """(v rounded to e4m3, the step there), |v| <= 448, ties to even"""
    size = v.abs().clamp_min(2.0 ** -30)
    step = torch.exp2((torch.floor(torch.log2(size))).clamp_min(-6.0) - 3.0)
    return (torch.round(v / step) * step).clamp(-448.0, 448.0), step


def quantised(x, err=None):
    """Rows in 64 bits -> (the numbers their quantised form stands for, what those may be off by if the rows are off by ``err``).
    The scale is off by the relative error ``d`` of the block's largest number, a quotient by err / s and d of itself; one that can
    reach a middle that way may be a whole step off."""
    m, k = x.shape
    kb = -(-k // BLOCK)

    def blocks(t):
        return torch.nn.functional.pad(t.double(), (0, kb * BLOCK - k)).view(m, kb, BLOCK)

    pad = blocks(x)
    s = scale(pad.abs().amax(dim=2, keepdim=True).float())
    v = (pad.float() / s).double()
    q, step = _e4m3(v)
    s = s.double()
    if err is None:
        return (q * s).view(m, -1)[:, :k], None
    d = blocks(err).amax(dim=2, keepdim=True) / pad.abs().amax(dim=2, keepdim=True).clamp_min(2.0 ** -126) + 2.0 ** -22
    at = (v / step).abs()
    from_middle = ((at - torch.floor(at)) - 0.5).abs() * step
    off = torch.where(from_middle <= blocks(err) / s + v.abs() * d, step, torch.zeros_like(step)) + q.abs() * d
    return (q * s).view(m, -1)[:, :k], (off * s).view(m, -1)[:, :k]


def sum_error(k):
    """A bound on the relative error of a sum over k numbers by blocks of 128, relative to the sum of sizes: an addition is off by a step of
    2^-23 at most (the tensor cores may cut instead of rounding), 128 in a block, one per block, three roundings of the scales."""
    return (BLOCK + -(-k // BLOCK) + 3) * 2.0 ** -23


def product(x, w, bias=None, off=None):
    """(x w^T + bias, what it may be off by in fp32) from 64-bit numbers; ``off``: what x's numbers may be off by"""
    y = x @ w.t()
    err = (x.abs() @ w.abs().t()) * sum_error(x.shape[1])
    if off is not None:
        err = err + off @ w.abs().t()
    if bias is not None:
        y = y + bias.double()
        err = err + y.abs() * 2.0 ** -24
    return y, err


def rounded(y, err, dtype):
    return err * 1.01 + (y.abs() + err) * (2.0 ** -8 if dtype == torch.bfloat16 else 2.0 ** -24)


def act64(g, u, name, limit):
    if name == "clamped":
        g, u = g.clamp(max=limit), u.clamp(-limit, limit)
        return g * torch.sigmoid(1.702 * g) * (u + 1.0)
    if name == "gelu_tanh":
        return 0.5 * g * (1.0 + torch.tanh((2.0 / torch.pi) ** 0.5 * (g + 0.044715 * g ** 3))) * u
    return g * torch.sigmoid(g) * u


def hidden64(x, gate, up, name, limit, scale=None, off=None):
    """act(x gate^T, x up^T) in 64 bits and what fp32 sums and an fp32 activation may put it off by: the sums' errors through slopes of
    at most 1.2 |u| + 0.2 (g) and 1.2 |g| + 1.2 (u), and 2^-18 of its size for the activation's own arithmetic.  ``off``: as for ``product``."""
    (g, ge), (u, ue) = product(x, gate, off=off), product(x, up, off=off)
    if scale is not None:
        g, ge, u, ue = g * scale, ge * scale.abs(), u * scale, ue * scale.abs()
    h = act64(g, u, name, limit)
    return h, ge * 1.7 * (u.abs() + 1.0) + ue * 1.2 * (g.abs() + 1.0) + h.abs() * 2.0 ** -18
