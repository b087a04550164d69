"""The calls that the speed of the operators around attention is measured on:
rotary positions, the paged cache of keys and values with the attention that
reads it, and the gated linear of a feed-forward block.

``listed()`` names the cases, ``draw(rng)`` gives further ones of the same
ranges, ``prepare`` builds what a program has in hand before the call, ``run``
makes one pass, ``work`` says what a pass cannot do without, and ``exact``
computes the outputs in 64 bits.  With ``own`` false, ``run`` computes the
operators in their plain form, out of elementary torch operations in 32 bits
(angles in 64); with ``own`` true it calls ``bfhip``.
"""

import math
import os
import sys

import torch

own = False

DEV = "cuda:0"
TYPES = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}
BYTES = {"f32": 4, "f16": 2, "bf16": 2}


def _bfhip():
    root = os.path.join(os.getcwd(), "bevfusion.c_amd")
    if root not in sys.path:
        sys.path.insert(0, root)
    import bfhip
    return bfhip


# ------------------------------------------------------------------ the cases
def listed():
    return [
        # One new token for each of 48 sequences, far into them: the smallest
        # call, where latency counts.
        dict(name="rotary_48_h32_d128_bf16", kind="rotary", type="bf16", tokens=48, heads=32,
             kv_heads=8, dim=128, part=128, interleaved=False, far=131072, factor=8.0,
             train=False),
        # A training step over a packed batch of 16 K tokens: queries and keys
        # out of one projection, and their gradients.
        dict(name="rotary_train_16384_h32_d128_bf16", kind="rotary", type="bf16", tokens=16384,
             heads=32, kv_heads=8, dim=128, part=128, interleaved=False, far=8192, factor=1.0,
             train=True),
        # Half of heads of 80 in neighbouring pairs, an odd number of tokens.
        dict(name="rotary_train_9999_h12_d80_f32", kind="rotary", type="f32", tokens=9999,
             heads=12, kv_heads=12, dim=80, part=40, interleaved=True, far=4096, factor=4.0,
             train=True),
        # The new tokens' keys and values of 48 sequences go into their pages.
        dict(name="append_48_h8_d128_bf16", kind="append", type="bf16", kv_heads=8, dim=128,
             page=16, q_lens="1*48", k_lens="1024,1,819,1200,500,409*8,204*16,102*16,33*3"),
        # Prompts and parts of prompts go in, behind what is there.
        dict(name="append_12319_h8_d128_f16", kind="append", type="f16", kv_heads=8, dim=128,
             page=64, q_lens="8192,2049,2000,1,77", k_lens="8192,4096,2000,313,4077"),
        # One new token of one long sequence: all the work is along its cache.
        dict(name="paged_1_on_131071_h32_d128_bf16", kind="paged", type="bf16", heads=32,
             kv_heads=8, dim=128, page=64, q_lens="1", k_lens="131071"),
        # One new token for each of 48 sequences, from one token to long ones.
        dict(name="paged_48_h32_d128_bf16", kind="paged", type="bf16", heads=32, kv_heads=8,
             dim=128, page=16, q_lens="1*48",
             k_lens="16384,1,8191,12000,500,4099*8,2048*16,1025*16,33*3"),
        # Three tokens at once for each of 100 sequences, every head with keys
        # of its own, pages of an odd size.
        dict(name="paged_100x3_h12_d64_f16", kind="paged", type="f16", heads=12, kv_heads=12,
             dim=64, page=7, q_lens="3*100", k_lens="1500*10,700*40,333*30,3*20"),
        # One token through a feed-forward block: both weights are read once.
        dict(name="gated_1x4096x11008_bf16", kind="gated", type="bf16", rows=1, features=4096,
             hidden=11008, activation="silu", train=False),
        # A long prompt through it.
        dict(name="gated_8192x4096x11008_bf16", kind="gated", type="bf16", rows=8192,
             features=4096, hidden=11008, activation="silu", train=False),
        # A training step of a packed batch of 8 K tokens.
        dict(name="gated_train_8192x2048x5632_bf16", kind="gated", type="bf16", rows=8192,
             features=2048, hidden=5632, activation="silu", train=True),
        # A training step with odd sizes, so that no row but the first is aligned.
        dict(name="gated_train_999x771x2055_f16", kind="gated", type="f16", rows=999,
             features=771, hidden=2055, activation="gelu", train=True),
    ]


def _log(rng, low, high):
    """A whole number, spread over its logarithm."""
    return min(high, max(low, int(round(math.exp(rng.uniform(math.log(low), math.log(high)))))))


def draw(rng):
    kind = rng.choice(("rotary", "append", "paged", "paged", "gated", "gated", "gated"))
    base = dict(kind=kind, type=rng.choice(("f32", "f16", "bf16", "bf16")))
    if kind == "gated":
        train = rng.random() < 0.5
        features, hidden = _log(rng, 64, 4096), _log(rng, 64, 11008)
        if rng.random() < 0.7:
            features, hidden = -(-features // 64) * 64, -(-hidden // 64) * 64
        most = (1 << 37) if base["type"] == "f32" else (1 << 38) if train else (1 << 39)
        rows = _log(rng, 1, 8192)
        if rng.random() < 0.3:
            rows = _log(rng, 1, 64)
        return dict(base, rows=max(1, min(rows, most // (features * hidden))), features=features,
                    hidden=hidden, activation=rng.choice(("silu", "silu", "gelu", "relu")),
                    train=train)
    kv_heads = rng.choice((1, 2, 3, 4, 8, 12))
    base.update(kv_heads=kv_heads, dim=rng.choice((16, 32, 40, 64, 64, 80, 96, 128, 128)))
    if kind != "append":
        base["heads"] = kv_heads * rng.choice((1, 1, 2, 4, 8) if kv_heads < 4 else (1, 2, 4))
    if kind == "rotary":
        heads = base["heads"] + kv_heads
        part = base["dim"] if rng.random() < 0.6 else 2 * rng.randint(1, base["dim"] // 2)
        return dict(base, tokens=_log(rng, 1, min(32768, (1 << 26) // (heads * base["dim"]))),
                    part=part, interleaved=rng.random() < 0.5, far=_log(rng, 1024, 1 << 20),
                    factor=rng.choice((1.0, 1.0, 4.0, 8.0, 32.0)), train=rng.random() < 0.5)
    base["page"] = rng.choice((1, 7, 16, 16, 32, 64, 100, 128, 256))
    n = _log(rng, 1, 128)
    if kind == "append":
        q = [_log(rng, 1, 1024 if n > 8 else 4096) if rng.random() < 0.5 else 1 for _ in range(n)]
        while sum(q) > 12288:
            q[q.index(max(q))] //= 2
        return dict(base, q_lens=_text(q), k_lens=_text([m + _log(rng, 1, 600) - 1 for m in q]))
    k = [_log(rng, 8, 65536 if n < 4 else 16384 if n < 32 else 4096) for _ in range(n)]
    most = 100_000_000 // (kv_heads * base["dim"] * BYTES[base["type"]])
    while sum(k) > min(most, 120000):
        k[k.index(max(k))] //= 2
    q = [1 if rng.random() < 0.8 else rng.randint(1, 8) for _ in range(n)]
    return dict(base, q_lens=_text(q), k_lens=_text([max(a, b) for a, b in zip(q, k)]))


def _text(lens):
    return ",".join(str(n) for n in lens)


def _lens(case):
    """Lengths of the sequences' new tokens and of their caches: "8,5*3" is
    8, 5, 5, 5."""
    def read(text):
        out = []
        for part in text.split(","):
            n, _, times = part.partition("*")
            out += [int(n)] * int(times or 1)
        return out
    return read(case["q_lens"]), read(case["k_lens"])


# ----------------------------------------------------------------- the inputs
def _randn(gen, shape, scale, dtype=torch.float32):
    return torch.randn(shape, generator=gen, device=DEV).mul_(scale).to(dtype)


def _frequencies(part, factor):
    """Angles per position of each pair: 10000^(-2 i / part); those that turn
    less than once over 8192 positions divided by the factor, those that turn
    more than four times kept, the ones between mixed."""
    f = 10000.0 ** (-torch.arange(0, part, 2, device=DEV, dtype=torch.float64) / part)
    keep = ((8192 * f / (2 * math.pi) - 1.0) / 3.0).clamp(0.0, 1.0)
    return f * (keep + (1.0 - keep) / factor)


def prepare(case, seed):
    gen = torch.Generator(DEV).manual_seed(seed)
    s, t = dict(case=case), TYPES[case["type"]]
    if case["kind"] == "rotary":
        n, h, hk, d = case["tokens"], case["heads"], case["kv_heads"], case["dim"]

        def rows():  # of one projection
            both = _randn(gen, (n, (h + hk) * d), 1.0, t)
            q, k = both.split([h * d, hk * d], 1)
            return q.unflatten(1, (h, d)), k.unflatten(1, (hk, d))
        s["q"], s["k"] = rows()
        if case["train"]:
            s["dq"], s["dk"] = rows()
        s["positions"] = torch.randint(0, case["far"], (n,), generator=gen, device=DEV,
                                       dtype=torch.int32)
        s["frequencies"] = _frequencies(case["part"], case["factor"])
        s["amplitude"] = 0.1 * math.log(case["factor"]) + 1.0
    elif case["kind"] == "gated":
        m, n, f = case["rows"], case["features"], case["hidden"]
        s.update(x=_randn(gen, (m, n), 1.0, t), w_gate=_randn(gen, (f, n), n ** -0.5, t),
                 w_up=_randn(gen, (f, n), n ** -0.5, t))
        if case["train"]:
            s["dh"] = _randn(gen, (m, f), 1.0, t)
    else:
        hk, d, page = case["kv_heads"], case["dim"], case["page"]
        ql, kl = _lens(case)
        used = [-(-n // page) for n in kl]
        total = sum(used) + 3  # a few pages are free
        s["k_pages"] = _randn(gen, (total, page, hk, d), 1.0, t)
        s["v_pages"] = _randn(gen, (total, page, hk, d), 1.0, t)
        order = torch.randperm(total, generator=gen, device=DEV).int()
        s["page_table"] = torch.zeros((len(kl), max(used)), device=DEV, dtype=torch.int32)
        at = 0
        for b, n in enumerate(used):
            s["page_table"][b, :n] = order[at:at + n]
            at += n
        s["starts"] = torch.tensor([0] + ql).cumsum(0).int().to(DEV)
        s["lengths"] = torch.tensor(kl, dtype=torch.int32).to(DEV)
        s["q_lens"], s["k_lens"] = ql, kl
        if case["kind"] == "append":
            rows = _randn(gen, (sum(ql), 2 * hk * d), 1.0, t).split([hk * d, hk * d], 1)
            s["k"], s["v"] = (r.unflatten(1, (hk, d)) for r in rows)
        else:
            s["q"] = _randn(gen, (sum(ql), case["heads"], d), 1.0, t)
            s["scale"] = d ** -0.5
    torch.cuda.synchronize()
    return s


# ------------------------------------------------------------------- one pass
def run(s):
    kind = s["case"]["kind"]
    if kind == "rotary":
        return (_rotary_own if own else _rotary_plain)(s, s["case"])
    if kind == "gated":
        return (_gated_own if own else _gated_plain)(s, s["case"])
    if kind == "append":
        return (_append_own if own else _append_plain)(s, s["case"])
    return (_paged_own if own else _paged_plain)(s, s["case"])


def _rotary_own(s, case):
    bfhip = _bfhip()
    call = dict(interleaved=case["interleaved"], amplitude=s["amplitude"])
    out = bfhip.rotary(s["q"], s["k"], s["positions"], s["frequencies"], **call)
    if not case["train"]:
        return list(out)
    return [*out, *bfhip.rotary_backward(s["dq"], s["dk"], s["positions"], s["frequencies"],
                                         **call)]


def _rotary_plain(s, case):
    angle = s["positions"].double()[:, None] * s["frequencies"]
    cos = (angle.cos() * s["amplitude"]).float()[:, None]
    sin = (angle.sin() * s["amplitude"]).float()[:, None]
    part = case["part"]

    def turn(x, sin):
        y = x.clone()
        if case["interleaved"]:
            a, b = slice(0, part, 2), slice(1, part, 2)
        else:
            a, b = slice(0, part // 2), slice(part // 2, part)
        xa, xb = x[..., a].float(), x[..., b].float()
        y[..., a] = (xa * cos - xb * sin).to(x.dtype)
        y[..., b] = (xa * sin + xb * cos).to(x.dtype)
        return y
    out = [turn(s["q"], sin), turn(s["k"], sin)]
    if case["train"]:
        out += [turn(s["dq"], -sin), turn(s["dk"], -sin)]
    return out


def _append_own(s, case):
    _bfhip().cache_append(s["k"], s["v"], s["k_pages"], s["v_pages"], s["page_table"], s["starts"],
                          s["lengths"])
    return [s["k_pages"], s["v_pages"]]


def _append_plain(s, case):
    page = case["page"]
    tokens = torch.arange(s["k"].shape[0], device=DEV)
    b = torch.bucketize(tokens, s["starts"][1:], right=True)
    at = tokens - s["starts"][1:][b] + s["lengths"][b]
    rows = s["page_table"][b, at // page].long() * page + at % page
    for new, pages in ((s["k"], s["k_pages"]), (s["v"], s["v_pages"])):
        pages.view(-1, *pages.shape[2:])[rows] = new
    return [s["k_pages"], s["v_pages"]]


def _paged_own(s, case):
    return [_bfhip().paged_attention(s["q"], s["k_pages"], s["v_pages"], s["page_table"],
                                     s["starts"], s["lengths"], scale=s["scale"])]


def _paged_plain(s, case):
    page, g = case["page"], case["heads"] // case["kv_heads"]
    out = torch.zeros_like(s["q"])
    i0 = 0
    for b, (nq, nk) in enumerate(zip(s["q_lens"], s["k_lens"])):
        table = s["page_table"][b, :-(-nk // page)].long()
        k, v = (s[n][table].flatten(0, 1)[:nk].float().movedim(1, 0) for n in ("k_pages", "v_pages"))
        # [kv_heads, group * queries, dim]: a head's group shares its keys
        q = s["q"][i0:i0 + nq].float().unflatten(1, (-1, g)).movedim(0, 2).flatten(1, 2)
        p = torch.matmul(q, k.transpose(1, 2).contiguous()).mul_(s["scale"]).unflatten(1, (g, nq))
        seen = torch.arange(nk, device=DEV) <= torch.arange(nk - nq, nk, device=DEV)[:, None]
        p = p.masked_fill_(~seen, -math.inf)
        p = p.sub_(p.amax(3, keepdim=True)).exp_()
        p /= p.sum(3, keepdim=True)
        o = torch.matmul(p.flatten(1, 2), v.contiguous()).unflatten(1, (g, nq))
        out[i0:i0 + nq] = o.movedim(2, 0).flatten(1, 2).to(out.dtype)
        i0 += nq
    return [out]


def _gated_own(s, case):
    bfhip = _bfhip()
    x, weights, act = s["x"], (s["w_gate"], s["w_up"]), case["activation"]
    if not case["train"]:
        return [bfhip.gated_linear(x, *weights, activation=act)]
    h, gate, up = bfhip.gated_linear(x, *weights, activation=act, save=True)
    return [h, *bfhip.gated_linear_backward(s["dh"], x, *weights, gate, up, activation=act)]


def _activation(name, g):
    """The activation and its derivative."""
    if name == "silu":
        sig = 1.0 / (1.0 + (-g).exp())
        return g * sig, sig * (1.0 + g * (1.0 - sig))
    if name == "gelu":
        cdf = 0.5 * (1.0 + (g * 0.5 ** 0.5).erf())
        return g * cdf, cdf + g * (-0.5 * g * g).exp() * (2.0 * math.pi) ** -0.5
    return g.clamp_min(0.0), (g > 0).to(g.dtype)


def _gated_plain(s, case):
    t = s["x"].dtype
    x, wg, wu = s["x"].float(), s["w_gate"].float(), s["w_up"].float()
    g, u = torch.mm(x, wg.T), torch.mm(x, wu.T)
    a, da = _activation(case["activation"], g)
    h = (a * u).to(t)
    if not case["train"]:
        return [h]
    dh = s["dh"].float()
    dg, du = dh * u * da, dh * a
    dx = torch.mm(dg, wg).add_(torch.mm(du, wu))
    return [h, dx.to(t), torch.mm(dg.T, x).to(t), torch.mm(du.T, x).to(t)]


# ------------------------------------------------------------------- the work
def work(case):
    """Inputs read once, outputs written once; sums and products of the
    formulas."""
    size = BYTES[case["type"]]
    if case["kind"] == "rotary":
        n = case["tokens"] * (case["heads"] + case["kv_heads"])
        passes = 2 if case["train"] else 1
        return {"bytes": passes * (2 * n * case["dim"] * size + 4 * case["tokens"]
                                   + 4 * case["part"]),
                "flops": passes * 3 * n * case["part"]}
    if case["kind"] == "gated":
        m, n, f = case["rows"], case["features"], case["hidden"]
        if case["train"]:  # x, both weights and their gradients; h and its
            return {"bytes": size * (2 * m * n + 4 * f * n + 2 * m * f), "flops": 12 * m * n * f}
        return {"bytes": size * (m * n + 2 * f * n + m * f), "flops": 4 * m * n * f}
    ql, kl = _lens(case)
    row = case["kv_heads"] * case["dim"] * size
    if case["kind"] == "append":
        return {"bytes": 4 * sum(ql) * row, "flops": 0}
    pairs = sum(nq * nk - nq * (nq - 1) // 2 for nq, nk in zip(ql, kl))
    return {"bytes": 2 * sum(kl) * row + 2 * sum(ql) * case["heads"] * case["dim"] * size,
            "flops": 4 * case["dim"] * case["heads"] * pairs}


# ------------------------------------------------------- the outputs in 64 bits
def exact(case, seed):
    """What ``run`` returns, from the definitions in 64 bits: rotations as
    products of complex numbers, cache rows and heads one by one, gradients in
    pieces of rows."""
    s = prepare(case, seed)
    return dict(rotary=_rotary_exact, append=_append_exact, paged=_paged_exact,
                gated=_gated_exact)[case["kind"]](s, case)


def _rotary_exact(s, case):
    half = case["part"] // 2
    i = torch.arange(half, device=DEV)
    first, second = (2 * i, 2 * i + 1) if case["interleaved"] else (i, i + half)
    phase = torch.outer(s["positions"].double(), s["frequencies"])
    turn = torch.polar(torch.full_like(phase, s["amplitude"]), phase)[:, None]

    def turned(x, by):
        x = x.double()
        z = torch.complex(x[..., first], x[..., second]) * by
        x[..., first], x[..., second] = z.real, z.imag
        return x
    out = [turned(s["q"], turn), turned(s["k"], turn)]
    if case["train"]:
        out += [turned(s["dq"], turn.conj()), turned(s["dk"], turn.conj())]
    return out


def _append_exact(s, case):
    k, v = s["k_pages"].double(), s["v_pages"].double()
    table, page, t = s["page_table"].tolist(), case["page"], 0
    for b, (nq, nk) in enumerate(zip(s["q_lens"], s["k_lens"])):
        at = nk - nq
        while at < nk:  # what is left of a page, page by page
            n = min(nk - at, page - at % page)
            rows = slice(at % page, at % page + n)
            k[table[b][at // page], rows] = s["k"][t:t + n].double()
            v[table[b][at // page], rows] = s["v"][t:t + n].double()
            at, t = at + n, t + n
    return [k, v]


def _paged_exact(s, case):
    out = torch.zeros(s["q"].shape, dtype=torch.float64, device=DEV)
    page, i0 = case["page"], 0
    for b, (nq, nk) in enumerate(zip(s["q_lens"], s["k_lens"])):
        at = torch.arange(nk, device=DEV)
        pages = s["page_table"][b].long()[at // page]
        k, v = s["k_pages"][pages, at % page].double(), s["v_pages"][pages, at % page].double()
        q = s["q"][i0:i0 + nq].double()
        hidden = at > (torch.arange(nq, device=DEV) + nk - nq)[:, None]
        for kv in range(case["kv_heads"]):
            kt, vt = k[:, kv].T.contiguous(), v[:, kv].contiguous()
            for head in range(kv * case["heads"] // case["kv_heads"],
                              (kv + 1) * case["heads"] // case["kv_heads"]):
                score = (q[:, head] @ kt * s["scale"]).masked_fill(hidden, -math.inf)
                out[i0:i0 + nq, head] = torch.softmax(score, 1) @ vt
        i0 += nq
    return [out]


def _gated_exact(s, case):
    wg, wu = s["w_gate"].double(), s["w_up"].double()
    wgt, wut = wg.T.contiguous(), wu.T.contiguous()
    hs, dxs, dwg, dwu = [], [], torch.zeros_like(wg), torch.zeros_like(wu)
    for at in range(0, case["rows"], 2048):
        x = s["x"][at:at + 2048].double()
        g, u = x @ wgt, x @ wut
        if case["activation"] == "silu":
            slope = torch.sigmoid(g)
            a, slope = g * slope, slope + g * slope * torch.sigmoid(-g)
        elif case["activation"] == "gelu":
            slope = 0.5 * torch.special.erfc(-g / math.sqrt(2.0))
            a = g * slope
            slope = slope + g * torch.exp(-g * g / 2.0) / math.sqrt(2.0 * math.pi)
        else:
            slope = torch.where(g > 0, 1.0, 0.0).double()
            a = g * slope
        hs.append(u * a)
        if case["train"]:
            dh = s["dh"][at:at + 2048].double()
            dg, du = u * slope * dh, a * dh
            dxs.append(dg @ wg + du @ wu)
            dwg += dg.T.contiguous() @ x
            dwu += du.T.contiguous() @ x
    return [torch.cat(hs)] + ([torch.cat(dxs), dwg, dwu] if case["train"] else [])
