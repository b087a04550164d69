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


def paged_attention(q, k_pages, v_pages, table, starts, lengths, scale, bias=None):
    """Dict of (value, bound) for out and lse."""
    k, k_starts = gathered(k_pages, table, lengths)
    v, _ = gathered(v_pages, table, lengths)
    both = ref.attention(q, k, v, starts, k_starts, True, scale, bias)
    return {n: both[n] for n in ("out", "lse")}
