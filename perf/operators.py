"""The calls that the speed of the transformer operators is measured on: layer
norm, position bias by buckets, and attention over packed sequences.

``listed()`` names the cases, ``draw(rng)`` gives further ones of the same
ranges, ``prepare`` builds what a program has in hand before the call, ``run``
makes one pass, ``work`` says what a pass cannot do without, and ``exact``
computes the outputs in 64 bits.  With ``own`` false, ``run`` computes the
operators in their plain form, out of elementary torch operations in 32 bits;
with ``own`` true it calls ``bfhip``.
"""

import math
import os
import sys

import torch

own = False

DEV = "cuda:0"
TYPES = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}
BYTES = {"f32": 4, "f16": 2, "bf16": 2}
EPS = 1e-5


def _bfhip():
    root = os.path.join(os.getcwd(), "bevfusion.c_amd")
    if root not in sys.path:
        sys.path.insert(0, root)
    import bfhip
    return bfhip


# ------------------------------------------------------------------ the cases
def listed():
    return [
        # The norm after one decoder layer over 200 proposals of 128 channels:
        # the smallest call, where latency counts.
        dict(name="norm_200x128_f32", kind="norm", rows=200, cols=128, type="f32", train=False),
        # The norm before stage 0's blocks over six cameras of 64 x 176 tokens.
        dict(name="norm_67584x96_f32", kind="norm", rows=67584, cols=96, type="f32", train=False),
        # A training step through a norm whose rows are odd in number and in
        # length, so that no row but the first is aligned.
        dict(name="norm_train_9999x257_f16", kind="norm", rows=9999, cols=257, type="f16",
             train=True),
        # A training step of a long packed batch: 64 K tokens of 768 channels.
        dict(name="norm_train_65536x768_bf16", kind="norm", rows=65536, cols=768, type="bf16",
             train=True),
        # The table of a 7 x 7 window (169 buckets) spread over its 49 x 49
        # pairs for 12 heads, and the table's gradient from the pairs'.
        dict(name="bias_169x12_49x49", kind="bias", buckets=169, heads=12, rows=49, cols=49,
             rule="window"),
        # The same for all pairs of 1024 positions, buckets by distance.
        dict(name="bias_32x16_1024x1024", kind="bias", buckets=32, heads=16, rows=1024, cols=1024,
             rule="distance"),
        # Cross attention of 200 proposals over a 180 x 180 map, eight heads of
        # 16 channels: few rows on a long key axis.
        dict(name="cross_200x32400_h8_d16_f16", kind="attention", type="f16", heads=8, kv_heads=8,
             dim=16, q_lens="200", k_lens="32400", causal=False, reach=0, train=False),
        # A packed batch of prompts, causal, four query heads on a key head.
        dict(name="prompt_16384_h32_d128_bf16", kind="attention", type="bf16", heads=32, kv_heads=8,
             dim=128, q_lens="8192,4097,2000,1,1033,517,300,244", k_lens="", causal=True, reach=0,
             train=False),
        # One new token for each of 48 sequences whose keys are kept: lengths
        # from one token to long ones.
        dict(name="token_48_h32_d128_bf16", kind="attention", type="bf16", heads=32, kv_heads=8,
             dim=128, q_lens="1*48", k_lens="16384,1,8191,12000,500,4099*8,2048*16,1025*16,33*3",
             causal=True, reach=0, train=False),
        # A training step through causal attention on a packed batch.
        dict(name="train_8192_h16_d128_bf16", kind="attention", type="bf16", heads=16, kv_heads=4,
             dim=128, q_lens="4096,2049,1000,777,270", k_lens="", causal=True, reach=0, train=True),
        # A training step of an encoder whose position bias is learned by
        # buckets of the distance (saturating at 128): table to gradient.
        dict(name="train_bias_7709_h12_d64_f16", kind="attention", type="f16", heads=12,
             kv_heads=12, dim=64, q_lens="512*14,411,130", k_lens="", causal=False, reach=128,
             train=True),
        # A training step in fp32 with more queries than keys in one sequence
        # (rows that see no key), an empty sequence and short ragged ones.
        dict(name="train_ragged_h6_d32_f32", kind="attention", type="f32", heads=6, kv_heads=3,
             dim=32, q_lens="65,1,200,0,49*8,333,31", k_lens="60,130,200,17,49*8,500,31",
             causal=True, reach=0, train=True),
    ]


def _log(rng, low, high):
    """A whole number, spread over its logarithm."""
    return min(high, max(low, int(round(math.exp(rng.uniform(math.log(low), math.log(high)))))))


def draw(rng):
    kind = rng.choice(("norm", "norm", "bias", "attention", "attention", "attention"))
    if kind == "norm":
        cols = _log(rng, 8, 4096)
        rows = _log(rng, 1, 65536 * 768 // cols)
        return dict(kind=kind, rows=rows, cols=cols, type=rng.choice(("f32", "f16", "bf16")),
                    train=rng.random() < 0.6)
    if kind == "bias":
        rows, cols = _log(rng, 7, 1024), _log(rng, 7, 1024)
        return dict(kind=kind, buckets=_log(rng, 8, 512), heads=rng.randint(1, 16), rows=rows,
                    cols=cols, rule="distance")
    kv_heads = rng.choice((1, 2, 3, 4, 8))
    heads = kv_heads * rng.choice((1, 1, 2, 4, 8) if kv_heads < 4 else (1, 2, 4))
    base = dict(kind=kind, type=rng.choice(("f32", "f16", "bf16", "bf16")), heads=heads,
                kv_heads=kv_heads, dim=rng.choice((16, 32, 40, 64, 64, 80, 96, 128, 128)))
    form = rng.choice(("prompt", "token", "train", "train"))
    if form == "token":
        n = _log(rng, 1, 64)
        k = [_log(rng, 1, 16384 if n < 32 else 4096) for _ in range(n)]
        while sum(k) > (50000 if base["type"] == "f32" else 100000):
            k[k.index(max(k))] //= 2
        q = [1 if rng.random() < 0.8 else rng.randint(1, 8) for _ in range(n)]
        return dict(base, q_lens=_text(q), k_lens=_text(k), causal=True, reach=0, train=False)
    longest = _log(rng, 16, 4096)
    left, q = _log(rng, longest, 8192), []
    while left > 0 and len(q) < 64:
        q.append(min(left, max(1, int(longest * rng.random() ** 2) if q else longest)))
        left -= q[-1]
    train = form == "train"
    causal = rng.random() < 0.6
    k = [n if rng.random() < 0.8 else max(1, n + rng.randint(-9, 9)) for n in q]
    if base["type"] == "f32":  # at the rate of fp32 products
        q, k = [max(1, n // 2) for n in q], [max(1, n // 2) for n in k]
    return dict(base, q_lens=_text(q), k_lens=_text(k), causal=causal,
                reach=rng.choice((0, 0, rng.randint(4, 200))), train=train)


def _text(lens):
    return ",".join(str(n) for n in lens)


def _lens(case):
    """Lengths of the sequences' queries and keys: "8,5*3" is 8, 5, 5, 5."""
    def read(text):
        out = []
        for part in text.split(","):
            n, _, times = part.partition("*")
            out += [int(n)] * int(times or 1)
        return out
    q = read(case["q_lens"])
    return q, (read(case["k_lens"]) if case["k_lens"] else list(q))


# ----------------------------------------------------------------- the inputs
def _randn(gen, shape, scale, dtype=torch.float32):
    return (torch.randn(shape, generator=gen, device=DEV) * scale).to(dtype)


def _distance_map(distance, buckets):
    """Buckets of signed distances: half of them for each sign; of a half, the
    first half one distance each, the others spread over the logarithm up to
    128, beyond which the last one holds."""
    half = max(1, buckets // 2)
    near = max(1, half // 2)
    d = distance.abs().double()
    far = near + torch.floor(torch.log((d / near).clamp_min(1.0)) / math.log(max(2.0, 128 / near))
                             * (half - near)).long()
    n = torch.where(d < near, d.long(), far.clamp_max(half - 1))
    return (n + half * (distance > 0)).clamp_max(buckets - 1).int()


def _window_map(rows):
    """Pairs of a square window of `rows` tokens: one bucket per offset."""
    side = math.isqrt(rows)
    at = torch.arange(rows, device=DEV)
    y, x = at // side, at % side
    dy, dx = y[:, None] - y[None, :] + side - 1, x[:, None] - x[None, :] + side - 1
    return (dy * (2 * side - 1) + dx).int()


def prepare(case, seed):
    gen = torch.Generator(DEV).manual_seed(seed)
    s = dict(case=case)
    if case["kind"] == "norm":
        r, c, t = case["rows"], case["cols"], TYPES[case["type"]]
        # Tokens of a residual stream: channels with offsets and spreads of
        # their own, rows that differ in size.
        x = _randn(gen, (r, c), 1.0) * (0.3 + torch.rand(c, generator=gen, device=DEV))
        x = (x + _randn(gen, (c,), 0.5)) * (0.5 + torch.rand((r, 1), generator=gen, device=DEV))
        s.update(x=x.to(t), gamma=1 + _randn(gen, (c,), 0.2), beta=_randn(gen, (c,), 0.2))
        if case["train"]:
            s["dy"] = _randn(gen, (r, c), 1.0, t)
    elif case["kind"] == "bias":
        r, c = case["rows"], case["cols"]
        if case["rule"] == "window":
            s["map"] = _window_map(r)
        else:
            s["map"] = _distance_map(torch.arange(c, device=DEV)[None, :]
                                     - torch.arange(r, device=DEV)[:, None], case["buckets"])
        s["table"] = _randn(gen, (case["buckets"], case["heads"]), 0.5)
        s["dbias"] = _randn(gen, (case["heads"], r, c), 1.0)
    else:
        h, hk, d, t = case["heads"], case["kv_heads"], case["dim"], TYPES[case["type"]]
        ql, kl = _lens(case)
        tq, tk = sum(ql), sum(kl)
        if ql == kl:  # self attention: the three come out of one linear
            rows = _randn(gen, (tq, (h + 2 * hk) * d), 1.0, t)
            q, k, v = rows.split([h * d, hk * d, hk * d], 1)
        else:
            q = _randn(gen, (tq, h * d), 1.0, t)
            k, v = _randn(gen, (tk, 2 * hk * d), 1.0, t).split([hk * d, hk * d], 1)
        s.update(q=q.unflatten(1, (h, d)), k=k.unflatten(1, (hk, d)), v=v.unflatten(1, (hk, d)),
                 scale=d ** -0.5)
        for name, lens in (("q_starts", ql), ("k_starts", kl)):
            s[name] = torch.tensor([0] + lens).cumsum(0).int().to(DEV)
        s["q_lens"], s["k_lens"] = ql, kl
        if case["reach"]:
            n = case["reach"]
            s["map"] = _distance_map(torch.arange(-n, n + 1, device=DEV), 32)
            s["table"] = _randn(gen, (32, h), 1.0)
        if case["train"]:
            s["dout"] = _randn(gen, (tq, h, d), 1.0, t)
    torch.cuda.synchronize()
    return s


# ------------------------------------------------------------------- one pass
def run(s):
    case = s["case"]
    if case["kind"] == "norm":
        return (_norm_own if own else _norm_plain)(s, case["train"])
    if case["kind"] == "bias":
        return (_bias_own if own else _bias_plain)(s)
    return (_attention_own if own else _attention_plain)(s, case)


def _norm_own(s, train):
    bfhip = _bfhip()
    if not train:
        return [bfhip.layer_norm(s["x"], s["gamma"], s["beta"], EPS)]
    y, mean, rstd = bfhip.layer_norm(s["x"], s["gamma"], s["beta"], EPS, stats=True)
    return [y, *bfhip.layer_norm_backward(s["dy"], s["x"], mean, rstd, s["gamma"])]


def _norm_plain(s, train):
    x = s["x"].float()
    mean = x.mean(1, keepdim=True)
    rstd = ((x - mean).square().mean(1, keepdim=True) + EPS).rsqrt()
    xh = (x - mean) * rstd
    y = (xh * s["gamma"] + s["beta"]).to(s["x"].dtype)
    if not train:
        return [y]
    dy = s["dy"].float()
    g = dy * s["gamma"]
    dx = rstd * (g - g.mean(1, keepdim=True) - xh * (g * xh).mean(1, keepdim=True))
    return [y, dx.to(s["x"].dtype), (dy * xh).sum(0), dy.sum(0)]


def _bias_own(s):
    bfhip = _bfhip()
    return [bfhip.position_bias(s["table"], s["map"]),
            bfhip.position_bias_backward(s["dbias"], s["map"], s["table"].shape[0])]


def _spread(table, buckets):
    return table[buckets.long()].movedim(-1, 0).contiguous()


def _gather_grad(dbias, buckets, count):
    """Sums by bucket, in 64 bits (a bucket may hold very many pairs): products
    of pieces of 1024 pairs with ones where the bucket is the pair's."""
    short = -buckets.numel() % 1024
    rows = torch.nn.functional.pad(dbias.flatten(1).double(), (0, short)).unflatten(1, (-1, 1024))
    at = torch.nn.functional.pad(buckets.flatten(), (0, short), value=-1).view(-1, 1024, 1)
    ones = (at == torch.arange(count, device=DEV)).double()
    return torch.matmul(rows.movedim(1, 0).contiguous(), ones).sum(0).T.float()


def _bias_plain(s):
    return [_spread(s["table"], s["map"]), _gather_grad(s["dbias"], s["map"], s["table"].shape[0])]


def _attention_own(s, case):
    bfhip = _bfhip()
    bias = bfhip.position_bias(s["table"], s["map"]) if case["reach"] else None
    call = dict(causal=case["causal"], scale=s["scale"], bias=bias)
    q, k, v, starts = s["q"], s["k"], s["v"], (s["q_starts"], s["k_starts"])
    if not case["train"]:
        return [bfhip.attention(q, k, v, *starts, **call)]
    out, lse = bfhip.attention(q, k, v, *starts, lse=True, **call)
    grads = bfhip.attention_backward(s["dout"], q, k, v, out, lse, *starts, **call)
    if bias is None:
        return [out, *grads]
    return [out, *grads[:3], bfhip.position_bias_backward(grads[3], s["map"], s["table"].shape[0])]


def _heads_first(t, repeat):
    return t.float().movedim(1, 0).repeat_interleave(repeat, 0).contiguous()


def _diagonals(x):
    """Sums of x [heads, rows, cols] along its diagonals, from the one in the
    lower left corner: the rows from the last one on, each moved one to the
    right of the one before."""
    rows, cols = x.shape[1:]
    skewed = torch.nn.functional.pad(x.flip(1), (0, rows)).flatten(1)[:, :-rows]
    return skewed.view(-1, rows, rows + cols - 1).sum(1, dtype=torch.float64)


def _ends(nq, nk, reach):
    """Where each diagonal's distance, from 1 - nk to nq - 1, stands in
    the bias."""
    return torch.arange(1 - nk, nq, device=DEV).clamp(-reach, reach) + reach


def _attention_plain(s, case):
    h, hk, reach, train = case["heads"], case["kv_heads"], case["reach"], case["train"]
    g, t, scale = h // hk, s["q"].dtype, s["scale"]
    out = torch.zeros(s["q"].shape, dtype=t, device=DEV)
    bias = _spread(s["table"], s["map"]) if reach else None
    if train:
        dq, dk, dv = (torch.zeros(s[n].shape, dtype=t, device=DEV) for n in "qkv")
        dbias = torch.zeros((h, 2 * reach + 1), dtype=torch.float64, device=DEV)
    i0 = j0 = 0
    for nq, nk in zip(s["q_lens"], s["k_lens"]):
        rows, keys = slice(i0, i0 + nq), slice(j0, j0 + nk)
        i0, j0 = i0 + nq, j0 + nk
        if not nq or not nk:
            continue
        q = _heads_first(s["q"][rows], 1)
        k, v = _heads_first(s["k"][keys], g), _heads_first(s["v"][keys], g)
        p = torch.matmul(q, k.transpose(1, 2).contiguous()).mul_(scale)
        far = (torch.arange(nk, device=DEV)[None, :]
               - (torch.arange(nq, device=DEV)[:, None] + nk - nq))
        if reach:
            at = far.clamp(-reach, reach) + reach
            p += bias[:, at]
        if case["causal"]:
            p.masked_fill_(far > 0, -math.inf)
        top = p.amax(2, keepdim=True)
        p = p.sub_(top.masked_fill(top == -math.inf, 0.0)).exp_()
        total = p.sum(2, keepdim=True)
        p /= total.masked_fill(total == 0, 1.0)
        o = torch.matmul(p, v)
        out[rows] = o.movedim(0, 1).to(t)
        if not train:
            continue
        do = _heads_first(s["dout"][rows], 1)
        dv[keys] = (torch.matmul(p.transpose(1, 2).contiguous(), do).unflatten(0, (hk, g)).sum(1)
                    .movedim(0, 1).to(t))
        ds = torch.matmul(do, v.transpose(1, 2).contiguous())
        ds = ds.sub_((do * o).sum(2, keepdim=True)).mul_(p)
        if reach:
            dbias.index_add_(1, _ends(nq, nk, reach), _diagonals(ds))
        dq[rows] = (torch.matmul(ds, k) * scale).movedim(0, 1).to(t)
        dk[keys] = ((torch.matmul(ds.transpose(1, 2).contiguous(), q) * scale)
                    .unflatten(0, (hk, g)).sum(1).movedim(0, 1).to(t))
    if not train:
        return [out]
    if not reach:
        return [out, dq, dk, dv]
    return [out, dq, dk, dv, _gather_grad(dbias, s["map"], s["table"].shape[0])]


# ------------------------------------------------------------------- the work
def _pairs(case):
    total = 0
    for nq, nk in zip(*_lens(case)):
        if not case["causal"]:
            total += nq * nk
        else:  # the last query sees every key, each one before it a key less
            n = min(nq, nk)
            total += n * nk - n * (n - 1) // 2
    return total


def work(case):
    """Inputs read once, outputs written once; sums and products of the
    formulas."""
    if case["kind"] == "norm":
        n, c, b = case["rows"] * case["cols"], case["cols"], BYTES[case["type"]]
        if case["train"]:
            return {"bytes": 4 * n * b + 16 * c, "flops": 18 * n}
        return {"bytes": 2 * n * b + 8 * c, "flops": 7 * n}
    if case["kind"] == "bias":
        n, t = case["rows"] * case["cols"], case["buckets"] * case["heads"]
        return {"bytes": 4 * (2 * n * case["heads"] + n + 2 * t), "flops": n * case["heads"]}
    ql, kl = _lens(case)
    q = sum(ql) * case["heads"] * case["dim"]
    kv = 2 * sum(kl) * case["kv_heads"] * case["dim"]
    products = 4 * case["dim"] * case["heads"] * _pairs(case)
    bias = 4 * 64 * case["heads"] if case["reach"] else 0
    if case["train"]:
        return {"bytes": BYTES[case["type"]] * (4 * q + 2 * kv) + bias, "flops": 7 * products // 2}
    return {"bytes": BYTES[case["type"]] * (2 * q + kv) + bias // 2, "flops": products}


# ------------------------------------------------------- the outputs in 64 bits
def exact(case, seed):
    """What ``run`` returns, from the definitions, row by row or head by head
    in 64 bits."""
    s = prepare(case, seed)
    if case["kind"] == "norm":
        return _norm_exact(s, case)
    if case["kind"] == "bias":
        flat = s["map"].flatten().long()
        bias = torch.stack([s["table"].double()[:, h].take(flat)
                            for h in range(case["heads"])]).view(s["dbias"].shape)
        return [bias, _bucket_sums(s["dbias"].double().flatten(1), flat, case["buckets"])]
    return _attention_exact(s, case)


def _norm_exact(s, case):
    n = case["cols"]
    gamma, beta = s["gamma"].double(), s["beta"].double()
    y, dx = [], []
    dgamma, dbeta = torch.zeros_like(gamma), torch.zeros_like(gamma)
    for at in range(0, case["rows"], 8192):
        x = s["x"][at:at + 8192].double()
        centred = x - (x.sum(1) / n)[:, None]
        dev = torch.sqrt((centred * centred).sum(1) / n + EPS)[:, None]
        unit = centred / dev
        y.append(beta + gamma * unit)
        if case["train"]:
            dy = s["dy"][at:at + 8192].double()
            dgamma += (dy * unit).sum(0)
            dbeta += dy.sum(0)
            # d unit_i / d x_j = (delta_ij - 1/n - unit_i unit_j / n) / dev
            g = dy * gamma
            along = (g * unit).sum(1)[:, None] / n
            dx.append((g - g.sum(1)[:, None] / n - along * unit) / dev)
    return [torch.cat(y)] + ([torch.cat(dx), dgamma, dbeta] if case["train"] else [])


def _bucket_sums(rows, flat, count):
    """rows [heads, n] summed over the n that share a bucket: running sums of
    the values in the order of their buckets, and their differences."""
    order = torch.argsort(flat, stable=True)
    ends = torch.bincount(flat, minlength=count).cumsum(0)
    sums = torch.nn.functional.pad(rows[:, order].cumsum(1), (1, 0))
    ends = torch.nn.functional.pad(ends, (1, 0))
    return (sums[:, ends[1:]] - sums[:, ends[:-1]]).T.contiguous()


def _attention_exact(s, case):
    h, hk, reach, train = case["heads"], case["kv_heads"], case["reach"], case["train"]
    names = ["q", "k", "v"]
    grads = {n: torch.zeros(s[n].shape, dtype=torch.float64, device=DEV) for n in names if train}
    out = torch.zeros(s["q"].shape, dtype=torch.float64, device=DEV)
    dtable = torch.zeros((32, h), dtype=torch.float64, device=DEV)
    i0 = j0 = 0
    for nq, nk in zip(s["q_lens"], s["k_lens"]):
        for head in range(h) if nq and nk else ():
            kv = head * hk // h
            k, v = s["k"][j0:j0 + nk, kv].double(), s["v"][j0:j0 + nk, kv].double()
            kt, vt = k.T.contiguous(), v.T.contiguous()
            for at in range(0, nq, 2048):
                rows = slice(i0 + at, i0 + min(at + 2048, nq))
                q = s["q"][rows, head].double()
                pos = torch.arange(at, min(at + 2048, nq), device=DEV) + (nk - nq)
                far = torch.arange(nk, device=DEV) - pos[:, None]
                score = (q @ kt) * s["scale"]
                if reach:
                    bucket = s["map"].long()[far.clamp(-reach, reach) + reach]
                    score += s["table"].double()[:, head][bucket]
                seen = far <= 0 if case["causal"] else torch.ones_like(far, dtype=torch.bool)
                alive = seen.any(1, keepdim=True)
                score = torch.where(seen, score, -math.inf)
                lse = torch.logsumexp(torch.where(alive, score, 0.0), 1, keepdim=True)
                p = torch.where(seen, torch.exp(score - lse), 0.0)
                o = p @ v
                out[rows, head] = o
                if not train:
                    continue
                do = s["dout"][rows, head].double()
                dp = do @ vt
                ds = p * (dp - (p * dp).sum(1, keepdim=True))
                grads["q"][rows, head] = ds @ k * s["scale"]
                grads["k"][j0:j0 + nk, kv] += ds.T.contiguous() @ q * s["scale"]
                grads["v"][j0:j0 + nk, kv] += p.T.contiguous() @ do
                if reach:
                    dtable[:, head] += torch.bincount(bucket.flatten(), ds.flatten(), 32)
        i0, j0 = i0 + nq, j0 + nk
    result = [out] + [grads[n] for n in names if train]
    return result + ([dtable] if train and reach else [])
