"""64-bit references of the transformer operators, each with a bound of how far
a correct 32-bit computation of it may be off, element by element.

Bounds count roundings: u = 2^-24 per fp32 operation, h = half a step of the
operands' type where a value is rounded to it (results, and probabilities and
score gradients on their way into the matrix cores; 0 for fp32, which is not
rounded there).  Below fp16's smallest normal number, 2^-14, the step is 2^-24
whatever the value, so a rounding to fp16 adds half of that, t = 2^-25, to what
h times the value covers (bf16 and fp32 have fp32's range: t = 0).  A sum of n terms in any order is off by at most n u times the
sum of their absolute values.  Second-order terms are covered by a factor of
1.05 and by whole counts where fractions would do.
"""

import math

import torch

U = 2.0 ** -24
SLACK = 1.05


def half(dtype):
    return torch.finfo(dtype).eps / 2


def tiny(dtype):
    return 2.0 ** -25 if dtype == torch.float16 else 0.0


def check(name, got, want, bound):
    """|got - want| <= bound everywhere; prints the largest share of it."""
    diff = (got.double() - want).abs()
    assert torch.isfinite(got).all(), f"{name}: not finite"
    share = (diff / bound.clamp_min(1e-300)).max().item() if diff.numel() else 0.0
    print(f"[bound] {name}: {share:.3f}", flush=True)
    assert share <= 1.0, f"{name}: {share:.3f} of the bound, largest error {diff.max():.3e}"


def layer_norm(x, gamma, beta, eps, dy=None):
    """Dict of (value, bound) for y, mean, rstd and, with dy, dx, dgamma,
    dbeta."""
    h, t, n, rows = half(x.dtype), tiny(x.dtype), x.shape[1], x.shape[0]
    ones = torch.ones(n, dtype=torch.float64, device=x.device)
    x = x.double()
    g = ones if gamma is None else gamma.double()
    b = 0 * ones if beta is None else beta.double()
    m = x.mean(1, keepdim=True)
    c = x - m
    r = (c.square().mean(1, keepdim=True) + eps).rsqrt()
    unit = c * r
    chain = n / 64 + 16  # a row's sums: a lane's share, then a tree
    e_m = (chain + 1) * U * x.abs().mean(1, keepdim=True) + U * m.abs()
    # The squares' mean sees the mean's error squared, and each centred value's.
    e_r = (chain + 8) * U + 2 * (e_m * r).square() + 2 * U * x.abs().amax(1, keepdim=True) * r
    e_unit = (e_m + U * x.abs()) * r + unit.abs() * (e_r + 2 * U)
    y = unit * g + b
    out = dict(y=(y, h * y.abs() + t + SLACK * (g.abs() * e_unit + 3 * U * ((unit * g).abs() + b.abs()))),
               mean=(m[:, 0], SLACK * e_m[:, 0]), rstd=(r[:, 0], SLACK * (e_r * r)[:, 0]))
    if dy is None:
        return out
    dy = dy.double()
    gy = dy * g
    s1, s2 = gy.mean(1, keepdim=True), (gy * unit).mean(1, keepdim=True)
    e_1 = (chain + 2) * U * gy.abs().mean(1, keepdim=True)
    e_2 = (chain + 3) * U * (gy * unit).abs().mean(1, keepdim=True) + (gy.abs() * e_unit).mean(1, keepdim=True)
    inner = gy - s1 - unit * s2
    e_in = e_1 + unit.abs() * e_2 + e_unit * s2.abs() + 4 * U * (gy.abs() + s1.abs() + (unit * s2).abs())
    dx = r * inner
    out["dx"] = dx, h * dx.abs() + t + SLACK * (r * e_in + dx.abs() * (e_r + 2 * U))
    chain = rows / 64 + 128  # rows: at least 64 partial sums, then theirs
    out["dgamma"] = (dy * unit).sum(0), SLACK * ((dy.abs() * e_unit).sum(0) + chain * U * (dy * unit).abs().sum(0))
    out["dbeta"] = dy.sum(0), SLACK * chain * U * dy.abs().sum(0)
    return out


def position_bias(table, buckets):
    known = (buckets >= 0) & (buckets < table.shape[0])
    return torch.where(known, table.T[:, buckets.long().clamp(0, table.shape[0] - 1)], 0.0)


def position_bias_backward(dbias, buckets, count):
    """(value, bound): a bucket's sum has as many terms as the bucket pairs."""
    d, at = dbias.double().flatten(1), buckets.flatten().long()
    known = (at >= 0) & (at < count)
    sums = torch.zeros((count, dbias.shape[0]), dtype=torch.float64, device=dbias.device)
    total = sums.index_add(0, at[known], d[:, known].T)
    size = sums.index_add(0, at[known], d[:, known].abs().T)
    n = torch.bincount(at[known], minlength=count)[:, None]
    return total, n * U * size


def attention(q, k, v, q_starts, k_starts, causal, scale, bias=None, dout=None, left=False):
    """Dict of (value, bound) for out, lse (-inf where no key is seen) and, with
    dout, dq, dk, dv and dbias.  Rows outside every sequence: zero, bound 0.
    left: what the probabilities' rounding left is taken too (not with dout)."""
    assert not left or dout is None
    h = half(q.dtype)
    t = tiny(q.dtype)
    hp = 0.0 if q.dtype == torch.float32 else h  # rounding on the way into the matrix cores
    hp = hp * hp if left else hp
    heads, kv_heads, dim, dev = q.shape[1], k.shape[1], q.shape[2], q.device
    zeros = lambda *shape: torch.zeros(shape, dtype=torch.float64, device=dev)
    res = {n: (zeros(*x.shape), zeros(*x.shape)) for n, x in
           (("out", q), ("dq", q), ("dk", k), ("dv", v))}
    res["lse"] = zeros(heads, q.shape[0]), zeros(heads, q.shape[0])
    reach = 0 if bias is None else bias.shape[1] // 2
    res["dbias"] = zeros(heads, 2 * reach + 1), zeros(heads, 2 * reach + 1)
    qs, ks = q_starts.tolist(), k_starts.tolist()
    most = {}
    for b in range(len(qs) - 1):
        nq, nk = qs[b + 1] - qs[b], ks[b + 1] - ks[b]
        rows, keys = slice(qs[b], qs[b + 1]), slice(ks[b], ks[b + 1])
        pos = torch.arange(nq, device=dev)[:, None] + nk - nq
        far = torch.arange(nk, device=dev)[None, :] - pos
        seen = far <= 0 if causal else torch.ones_like(far, dtype=torch.bool)
        for hd in range(heads):
            kv = hd // (heads // kv_heads)
            Q, K, V = q[rows, hd].double(), k[keys, kv].double(), v[keys, kv].double()
            K = torch.where(seen.any(0)[:, None], K, 0.0)
            s = scale * (Q @ K.T)
            size = abs(scale) * (Q.abs() @ K.abs().T)
            if bias is not None:
                add = bias[hd].double()[far.clamp(-reach, reach) + reach]
                s, size = s + add, size + torch.where(torch.isfinite(add), add.abs(), 0.0)
            s = torch.where(seen, s, -math.inf)
            alive = (s > -math.inf).any(1, keepdim=True) if nk else torch.zeros((nq, 1), dtype=torch.bool, device=dev)
            top = torch.where(alive, s.amax(1, keepdim=True) if nk else zeros(nq, 1), 0.0)
            ex = torch.exp(s - top)
            l = ex.sum(1, keepdim=True)
            p = ex / torch.where(alive, l, 1.0)
            lse = torch.where(alive, top + torch.log(torch.where(alive, l, 1.0)), -math.inf)
            # What a score may be off: its sum's roundings, the base's change
            # and the subtraction of the maximum; p is off by as much, relative.
            size = torch.where(seen & (s > -math.inf), size, 0.0)
            d = (dim + 8) * U * (size.amax(1, keepdim=True) if nk else zeros(nq, 1)) + 8 * U * (1 + top.abs())
            V = torch.where(seen.any(0)[:, None], V, 0.0)
            A = p @ V.abs()
            o = p @ V
            # Probabilities enter as 2^(s - top), at most 1, over their sum, at least 1.
            e_o = (2 * d + hp + (nk + 8) * U) * A + t * (seen.double() @ V.abs())
            res["out"][0][rows, hd], res["out"][1][rows, hd] = o, SLACK * (e_o + h * o.abs() + t)
            res["lse"][0][hd, rows] = lse[:, 0]
            res["lse"][1][hd, rows] = SLACK * (2 * d + (nk + 8) * U + 4 * U * torch.where(alive, lse, 0.0).abs())[:, 0]
            if dout is None:
                continue
            # p again from the stored lse.
            d = 3 * d + (nk + 16) * U + 8 * U * torch.where(alive, lse, 0.0).abs()
            G = dout[rows, hd].double()
            dp = G @ V.T
            delta = (p * dp).sum(1, keepdim=True)
            e_dp = (dim + 2) * U * (G.abs() @ V.abs().T)
            e_delta = (G.abs() * (SLACK * (e_o + h * o.abs() + t) + dim * U * o.abs())).sum(1, keepdim=True)
            ds = p * (dp - delta)
            e_ds = p * (d * (dp - delta).abs() + e_dp + e_delta + 4 * U * (dp.abs() + delta.abs()))
            once = t * seen.double()
            E = e_ds + hp * (ds.abs() + e_ds) + once
            n = heads // kv_heads * nq + 8
            parts = dict(
                dq=(rows, hd, scale * (ds @ K), abs(scale) * (E @ K.abs() + (nk + 8) * U * (ds.abs() @ K.abs()))),
                dk=(keys, kv, scale * (ds.T @ Q), abs(scale) * (E.T @ Q.abs() + n * U * (ds.abs().T @ Q.abs()))),
                dv=(keys, kv, p.T @ G, ((p * (d + hp) + once).T @ G.abs() + n * U * (p.T @ G.abs()))))
            for name, (at, hh, value, bound) in parts.items():
                res[name][0][at, hh] += value
                res[name][1][at, hh] += bound
            if bias is not None:
                e = (far.clamp(-reach, reach) + reach).flatten()
                res["dbias"][0][hd].index_add_(0, e, ds.flatten())
                # Sums of nq x nk terms at most.
                res["dbias"][1][hd].index_add_(0, e, (e_ds + (nq + nk) * len(qs) * U * ds.abs()).flatten())
    for name in ("dq", "dk", "dv"):
        value, bound = res[name]
        res[name] = value, SLACK * bound + h * value.abs() + t + 1e-30
    res["dbias"] = res["dbias"][0], SLACK * res["dbias"][1] + 1e-30
    return res
