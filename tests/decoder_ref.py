"""64-bit references of the operators around attention (rotary positions, the
paged cache, the gated linear), each with a bound of how far a correct 32-bit
computation of it may be off, counted as in transformer_ref."""

import math

import torch

import transformer_ref as ref
from transformer_ref import SLACK, U, half, tiny


def rotary(x, positions, frequencies, interleaved=False, amplitude=1.0, inverse=False):
    """(value, bound) of x [tokens, heads, dim] turned."""
    n = frequencies.numel()
    angle = positions.double()[:, None] * frequencies.double()
    c, s = (amplitude * f(angle)[:, None] for f in (torch.cos, torch.sin))
    s = -s if inverse else s
    i = torch.arange(n, device=x.device)
    first, second = (2 * i, 2 * i + 1) if interleaved else (i, i + n)
    value, bound = x.double().clone(), torch.zeros(x.shape, dtype=torch.float64, device=x.device)
    a, b = value[..., first].clone(), value[..., second].clone()
    value[..., first], value[..., second] = a * c - b * s, a * s + b * c
    # The angle, counted in turns, is rounded to fp32 once it lies within half a
    # turn (pi u), and was off by 2^-51 of itself before (three roundings in 64
    # bits, one of the oracle's); cosine and sine are good to 2 u of 1, and are
    # multiplied by the amplitude; then two products and their sum.
    off = (math.pi + 6) * U + 2.0 ** -51 * angle.abs()[:, None]
    size = abs(amplitude) * (a.abs() + b.abs())
    for at in (first, second):
        y = value[..., at]
        bound[..., at] = SLACK * off * size + half(x.dtype) * y.abs() + tiny(x.dtype) + 1e-30
    return value, bound


def gathered(pages, table, lengths):
    """Rows of all sequences, one after the other, and their starts."""
    size, rows = pages.shape[1], []
    for b, n in enumerate(lengths.tolist()):
        at = torch.arange(n, device=pages.device)
        rows.append(pages[table[b].long()[at // size], at % size])
    starts = torch.nn.functional.pad(lengths, (1, 0)).cumsum(0).int()
    return torch.cat(rows) if rows else pages.new_zeros((0, *pages.shape[2:])), starts


def paged_attention(q, k_pages, v_pages, table, starts, lengths, scale, bias=None, left=False):
    """Dict of (value, bound) for out and lse.  left: probabilities are multiplied
    with twice the type's precision."""
    k, k_starts = gathered(k_pages, table, lengths)
    v, _ = gathered(v_pages, table, lengths)
    both = ref.attention(q, k, v, starts, k_starts, True, scale, bias, left=left)
    return {n: both[n] for n in ("out", "lse")}


def _activation(kind, g, dtype):
    """(act(g), act'(g), their errors in units of U): the exponential's and erfc's
    arguments are rounded, which counts |g| and g^2 times.  For 16-bit types erfc
    is a fit, off by 3e-6 (50 U) of itself: a fiftieth of half a step of fp16."""
    if kind == "silu":
        s = torch.sigmoid(g)
        rest = g * torch.sigmoid(-g)
        off = 16 + 2 * g.abs()
        return g * s, s * (1 + rest), off * (g * s).abs(), off * s * (1 + rest.abs())
    if kind == "gelu":
        cdf, pdf = 0.5 * torch.special.erfc(-g / math.sqrt(2)), torch.exp(-g * g / 2) / math.sqrt(2 * math.pi)
        off = 16 + 2 * g * g + (0 if dtype == torch.float32 else 50)
        return g * cdf, cdf + g * pdf, off * (g * cdf).abs(), off * (cdf + (g * pdf).abs())
    return g.clamp_min(0), (g > 0).double(), 0 * g, 0 * g


def gated_linear(x, w_gate, w_up, activation):
    """Dict of (value, bound) for h, gate and up."""
    h, t, n, dtype = half(x.dtype), tiny(x.dtype), x.shape[1], x.dtype
    x, wg, wu = x.double(), w_gate.double().T.contiguous(), w_up.double().T.contiguous()
    g, u = x @ wg, x @ wu
    e_g, e_u = (n + 8) * U * (x.abs() @ wg.abs()), (n + 8) * U * (x.abs() @ wu.abs())
    a, _, e_a, _ = _activation(activation, g, dtype)
    e_a = U * e_a + 1.13 * e_g  # (no slope is larger)
    y = a * u
    out = a.abs() * e_u + (u.abs() + e_u) * e_a + 2 * U * y.abs()
    return dict(h=(y, SLACK * out + h * y.abs() + t + 1e-30), gate=(g, SLACK * e_g + U * g.abs() + 1e-30),
                up=(u, SLACK * e_u + U * u.abs() + 1e-30))


def gated_linear_backward(dh, x, w_gate, w_up, gate, up, activation, left=False):
    """Dict of (value, bound) for dx, dw_gate and dw_up.  left: what the slopes'
    rounding left is taken too (few slopes), which leaves a rounding of that, and
    twice as many terms."""
    h, t, (rows, hidden) = half(x.dtype), tiny(x.dtype), gate.shape
    dtype = x.dtype
    hp = 0.0 if dtype == torch.float32 else h  # rounding on the way into the matrix cores
    hp, terms = (hp * hp, 2) if left else (hp, 1)
    dh, x, wg, wu, g, u = (v.double() for v in (dh, x, w_gate, w_up, gate, up))
    a, d, e_a, e_d = _activation(activation, g, dtype)
    dg, du = dh * u * d, dh * a
    e_g = (dh * u).abs() * U * e_d + 4 * U * dg.abs()
    e_u = dh.abs() * U * e_a + 4 * U * du.abs()
    e_g, e_u = e_g + hp * (dg.abs() + e_g), e_u + hp * (du.abs() + e_u)
    if dtype == torch.float16 and dg.numel():
        # half of fp16's smallest step below the largest, which is at least 2^14
        most = max(dg.abs().max(), du.abs().max()) * 2.0 ** (-25 - 14)
        e_g, e_u = e_g + most, e_u + most
    res = {}
    k = terms * 2 * hidden + 16
    res["dx"] = dg @ wg + du @ wu, (e_g + k * U * dg.abs()) @ wg.abs() + (e_u + k * U * du.abs()) @ wu.abs()
    xa, k = x.abs().contiguous(), terms * rows + 16
    for name, v, e in (("dw_gate", dg, e_g), ("dw_up", du, e_u)):
        res[name] = v.T.contiguous() @ x, (e + k * U * v.abs()).T.contiguous() @ xa
    return {n: (v, SLACK * b + h * v.abs() + t + 1e-30) for n, (v, b) in res.items()}
