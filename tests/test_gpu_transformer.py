"""Layer norm, position bias and packed attention (include/bfhip_transformer.h)
against 64-bit references, within bounds counted from their roundings
(tests/transformer_ref.py)."""

import math

import pytest
import torch

import bfhip
import transformer_ref as ref

pytestmark = pytest.mark.gpu

F32, F16, BF16 = torch.float32, torch.float16, torch.bfloat16


def gen(device, seed):
    return torch.Generator(device).manual_seed(seed)


def randn(g, *shape, scale=1.0, dtype=F32):
    return (torch.randn(shape, generator=g, device=g.device) * scale).to(dtype)


# ----------------------------------------------------------------- layer norm
NORMS = [(F32, 200, 128), (F16, 1, 1), (BF16, 3, 7), (F32, 5, 96), (BF16, 130, 768), (F16, 67, 257),
         (BF16, 33, 1023), (F32, 9, 4100), (F16, 1030, 64), (BF16, 5, 16384), (F32, 2, 65536), (BF16, 4099, 40),
         (F32, 300, 33), (F16, 2, 5000), (F32, 1, 3), (F16, 700, 8), (BF16, 2500, 1600)]


def norm_inputs(device, dtype, rows, n, seed=0):
    g = gen(device, seed)
    x = randn(g, rows, n) * 1.5 + randn(g, rows, 1)
    return x.to(dtype), 1 + randn(g, n, scale=0.2), randn(g, n, scale=0.3), randn(g, rows, n, dtype=dtype)


@pytest.mark.parametrize("dtype,rows,n", NORMS)
def test_layer_norm(device, dtype, rows, n):
    x, gamma, beta, dy = norm_inputs(device, dtype, rows, n)
    want = ref.layer_norm(x, gamma, beta, 1e-5, dy)
    y, mean, rstd = bfhip.layer_norm(x, gamma, beta, 1e-5, stats=True)
    dx, dgamma, dbeta = bfhip.layer_norm_backward(dy, x, mean, rstd, gamma)
    for name, got in dict(y=y, mean=mean, rstd=rstd, dx=dx, dgamma=dgamma, dbeta=dbeta).items():
        ref.check(name, got, *want[name])
    again = bfhip.layer_norm_backward(dy, x, mean, rstd, gamma)
    assert all(torch.equal(a, b) for a, b in zip((dx, dgamma, dbeta), again))


@pytest.mark.parametrize("dtype", [F32, F16, BF16])
@pytest.mark.parametrize("n,stride,shift", [(96, 128, 0), (96, 97, 1), (250, 251, 3), (768, 776, 8), (2050, 2051, 5)])
def test_layer_norm_strided_rows_and_in_place(device, dtype, n, stride, shift):
    """Rows of a wider buffer at any alignment; y over x, dx over dy; what lies
    between the rows stays."""
    rows = 37
    x, gamma, beta, dy = norm_inputs(device, dtype, rows, n, seed=3)
    want = ref.layer_norm(x, gamma, beta, 1e-5, dy)

    def wide(t):
        buf = torch.full((rows * stride + shift,), 7.0, dtype=dtype, device=device)
        view = buf[shift:].view(rows, stride)[:, :n]
        view.copy_(t)
        return buf, view

    xb, xv = wide(x)
    gb, gv = wide(dy)
    keep, kv = wide(x)
    y, mean, rstd = bfhip.layer_norm(xv, gamma, beta, 1e-5, stats=True, out=xv)
    dx, dgamma, dbeta = bfhip.layer_norm_backward(gv, kv, mean, rstd, gamma, out=gv)
    for name, got in dict(y=xv, mean=mean, rstd=rstd, dx=gv, dgamma=dgamma, dbeta=dbeta).items():
        ref.check(name, got, *want[name])
    for buf in (xb, gb):
        rest = torch.ones_like(buf, dtype=torch.bool)
        rest[shift:].view(rows, stride)[:, :n] = False
        assert (buf[rest] == 7).all()
    dx2, _, _ = bfhip.layer_norm_backward(dy, kv, mean, rstd, gamma, out=kv)  # dx over x
    assert torch.equal(kv, gv)


def test_layer_norm_without_weights_and_without_rows(device):
    x, _, _, dy = norm_inputs(device, F32, 50, 200, seed=4)
    want = ref.layer_norm(x, None, None, 1e-5, dy)
    y, mean, rstd = bfhip.layer_norm(x, stats=True)
    got = bfhip.layer_norm_backward(dy, x, mean, rstd)
    for name, t in zip(("y", "dx", "dgamma", "dbeta"), (y, *got)):
        ref.check(name, t, *want[name])
    empty = torch.empty((0, 200), device=device)
    y, mean, rstd = bfhip.layer_norm(empty, stats=True)
    dx, dgamma, dbeta = bfhip.layer_norm_backward(empty, empty, mean, rstd)
    assert y.shape == dx.shape == (0, 200) and not dgamma.any() and not dbeta.any()


def test_layer_norm_constant_rows_and_offsets(device):
    """A row without spread is beta exactly; a spread far below the mean
    survives; a NaN stays in its row."""
    g = gen(device, 5)
    x = randn(g, 6, 384) * 0.01 + 1000.0
    x[2] = 3.0
    beta = randn(g, 384)
    want = ref.layer_norm(x, None, beta, 1e-5)
    y = bfhip.layer_norm(x, None, beta, 1e-5)
    ref.check("y", y, *want["y"])
    assert torch.equal(y[2], beta)
    x[4, 100] = math.nan
    again = bfhip.layer_norm(x, None, beta, 1e-5)
    assert again[4].isnan().all() and torch.equal(again[[0, 1, 2, 3, 5]], y[[0, 1, 2, 3, 5]])


def test_layer_norm_gradient_by_differences(device):
    g = gen(device, 6)
    x, gamma, beta, dy = norm_inputs(device, F32, 4, 65, seed=6)
    y, mean, rstd = bfhip.layer_norm(x, gamma, beta, 1e-5, stats=True)
    dx, dgamma, dbeta = bfhip.layer_norm_backward(dy, x, mean, rstd, gamma)

    def loss(x, gamma, beta):
        m = x.mean(1, keepdim=True)
        h = (x - m) / (x.var(1, unbiased=False, keepdim=True) + 1e-5).sqrt()
        return ((h * gamma + beta) * dy.double()).sum()

    args = [t.double() for t in (x, gamma, beta)]
    for i, grad in enumerate((dx, dgamma, dbeta)):
        way = randn(g, *args[i].shape).double()
        step = 1e-5
        moved = [[a + (sign * step * way if j == i else 0) for j, a in enumerate(args)] for sign in (1, -1)]
        slope = (loss(*moved[0]) - loss(*moved[1])) / (2 * step)
        # Central differences: step^2 times a third derivative, and 2^-52 / step of the loss.
        assert abs((grad.double() * way).sum() - slope) <= 1e-5 * (grad.double() * way).abs().sum()


# -------------------------------------------------------------- position bias
def window_map(side, device):
    at = torch.arange(side * side, device=device)
    y, x = at // side, at % side
    return ((y[:, None] - y[None, :] + side - 1) * (2 * side - 1) + x[:, None] - x[None, :] + side - 1).int()


def random_map(g, shape, count, low=0):
    return torch.randint(low, count, shape, generator=g, device=g.device).int()


@pytest.mark.parametrize("count,heads,shape,rule", [
    (169, 12, (49, 49), "window"), (32, 16, (70, 65), "random"), (1, 1, (1,), "random"), (5, 3, (257,), "outside"),
    (600, 7, (100, 33), "random"), (32, 20, (1031,), "runs"), (2000, 33, (50, 50), "random"), (9, 1, (3, 5, 7), "random"),
    (32, 5, (300, 301), "runs"), (4097, 2, (999,), "outside"), (3, 100, (77,), "random"), (64, 64, (64, 64), "runs")])
def test_position_bias(device, count, heads, shape, rule):
    g = gen(device, count)
    if rule == "window":
        at = window_map(7, device)
    elif rule == "runs":
        n = math.prod(shape)
        at = (torch.arange(n, device=device) * count // n).view(shape).int()
    else:
        at = random_map(g, shape, count + (3 if rule == "outside" else 0), -3 if rule == "outside" else 0)
    table, dbias = randn(g, count, heads), randn(g, heads, *shape)
    bias = bfhip.position_bias(table, at)
    assert torch.equal(bias, ref.position_bias(table, at))
    got = bfhip.position_bias_backward(dbias, at, count)
    ref.check("dtable", got, *ref.position_bias_backward(dbias, at, count))
    assert torch.equal(got, bfhip.position_bias_backward(dbias, at, count))
    # The gradient is the transpose of the spreading, which is linear.
    left, right = (bias.double() * dbias).sum(), (table.double() * got).sum()
    assert abs(left - right) <= 1e-6 * (bias.double() * dbias).abs().sum()


def test_position_bias_of_no_positions(device):
    at = torch.empty((0, 5), dtype=torch.int32, device=device)
    assert bfhip.position_bias(torch.ones((4, 2), device=device), at).shape == (2, 0, 5)
    assert not bfhip.position_bias_backward(torch.empty((2, 0, 5), device=device), at, 4).any()


def test_position_bias_feeds_window_attention(device):
    """The bias of a 7 x 7 window as the window attention takes it."""
    g = gen(device, 8)
    table, heads = randn(g, 169, 3, scale=0.5), 3
    at = window_map(7, device)
    bias = bfhip.position_bias(table, at)
    qkv = randn(g, 14 * 21, 96 * heads, scale=0.5, dtype=F16)
    zero = torch.zeros(96 * heads, device=device)
    got = bfhip.window_attention(qkv, zero, bias, 1, 14, 21, heads, 0)
    want = bfhip.window_attention(qkv, zero, table[at.long()].movedim(2, 0).contiguous(), 1, 14, 21, heads, 0)
    assert torch.equal(got, want)


# ------------------------------------------------------------------ attention
def starts(lens, device, first=0):
    return torch.tensor([first] + lens, device=device).cumsum(0).int()


# type, heads, key heads, dim, query lengths, key lengths (None: the same), causal, reach
CASES = [
    (BF16, 4, 2, 128, [130, 1, 0, 64, 65], None, True, None),
    (F16, 3, 3, 32, [49] * 5, None, False, 10),
    (F32, 6, 3, 40, [5, 70, 0, 3, 129], [70, 5, 9, 0, 65], True, None),
    (F32, 2, 1, 128, [150, 65], None, True, 200),
    (BF16, 8, 8, 16, [200], [1500], False, None),
    (F16, 4, 4, 64, [300], None, True, 2047),
    (BF16, 8, 2, 64, [1] * 7, [1, 700, 64, 65, 63, 128, 1025], True, None),
    (F16, 2, 2, 8, [17, 33], [40, 31], False, 3),
    (F16, 4, 1, 80, [100, 200], [90, 260], True, 0),
    (BF16, 6, 2, 96, [257], None, False, 40),
    (F32, 4, 4, 64, [100, 31], [100, 200], False, 17),
    (F32, 8, 1, 16, [3, 1, 2], [500, 640, 2], True, 65),
    (BF16, 1, 1, 128, [1], [1], True, None),
    (BF16, 16, 1, 128, [4, 1], [333, 2000], True, 33),
    (F16, 5, 5, 24, [1] * 130, [3] * 130, True, None),
    (F32, 1, 1, 32, [64], [64], True, 1),
    (BF16, 12, 4, 64, [513], None, True, None),
    (F16, 32, 8, 128, [1, 2, 1], [2500, 1300, 900], True, None),
    (BF16, 3, 3, 128, [7, 0, 5], [0, 9, 4000], False, 500),
    # Key axes that are split: single tokens and few rows, one part to very many.
    (F32, 8, 2, 128, [1, 3], [900, 2000], True, 12),
    (F16, 1, 1, 32, [2], [40001], False, None),
    (BF16, 2, 2, 64, [150], [5000], True, 300),
    (F32, 3, 1, 96, [70, 1], [3000, 40], False, 9),
    (BF16, 32, 4, 80, [1, 1, 2, 0], [0, 1, 6000, 77], True, 5),
    # The longest bias beside the largest rows; queries of a key tile in parts.
    (F32, 2, 1, 128, [70, 5], [90, 300], False, 2047),
    (BF16, 8, 1, 128, [1500, 40], None, True, 2047),
    (F16, 8, 2, 32, [2100], [700], False, None),
]


def inputs(device, case, seed=0, layout="fused"):
    dtype, heads, kv_heads, dim, ql, kl, causal, reach = case
    g = gen(device, seed)
    kl = ql if kl is None else kl
    tq, tk = sum(ql), sum(kl)

    def rows(n, h):
        t = randn(g, n, h, dim, scale=0.8, dtype=dtype)
        if layout == "fused":  # views of one wider row
            wide = torch.full((n, h * dim + 24 * 8), 3.0, dtype=dtype, device=device)
            view = wide[:, 64:64 + h * dim].unflatten(1, (h, dim))
            view.copy_(t)
            return view
        if layout == "heads":  # [heads, tokens, dim]
            return t.movedim(1, 0).contiguous().movedim(0, 1)
        return t

    q, k, v, dout = rows(tq, heads), rows(tk, kv_heads), rows(tk, kv_heads), rows(tq, heads)
    bias = None if reach is None else randn(g, heads, 2 * reach + 1, scale=1.5)
    return dict(q=q, k=k, v=v, q_starts=starts(ql, device), k_starts=starts(kl, device), causal=causal,
                scale=dim ** -0.5 * 1.5, bias=bias), dout


def grads(call, dout, out, lse):
    c = dict(call)
    return bfhip.attention_backward(dout, c.pop("q"), c.pop("k"), c.pop("v"), out, lse, **c)


@pytest.mark.parametrize("layout", ["fused", "heads"])
@pytest.mark.parametrize("case", CASES, ids=str)
def test_attention(device, case, layout):
    call, dout = inputs(device, case, layout=layout)
    want = ref.attention(**call, dout=dout)
    out, lse = bfhip.attention(**call, lse=True)
    assert torch.equal(out, bfhip.attention(**call))
    dead = want["lse"][0] == -math.inf
    assert torch.equal(lse == -math.inf, dead)
    assert not out.movedim(1, 0)[dead].any()
    got = dict(out=out, lse=torch.where(dead, 0.0, lse))
    want["lse"] = torch.where(dead, 0.0, want["lse"][0]), want["lse"][1]
    for name, t in got.items():
        ref.check(name, t, *want[name])
    back = grads(call, dout, out, lse)
    for name, t in zip(("dq", "dk", "dv", "dbias"), back):
        ref.check(name, t, *want[name])
    assert all(torch.equal(a, b) for a, b in zip(back, grads(call, dout, out, lse)))


@pytest.mark.parametrize("scale", [0.0, -0.3, 3.0])
@pytest.mark.parametrize("case", [(F32, 2, 1, 32, [70, 3], [90, 3], True, 4), (BF16, 4, 2, 64, [1, 2], [700, 3], True, None),
                                  (F16, 2, 2, 16, [130], [260], False, None)], ids=str)
def test_attention_scales(device, case, scale):
    """No scale, a negative one and a large one."""
    call, dout = inputs(device, case)
    call["scale"] = scale
    want = ref.attention(**call, dout=dout)
    out, lse = bfhip.attention(**call, lse=True)
    ref.check("out", out, *want["out"])
    for name, t in zip(("dq", "dk", "dv", "dbias"), grads(call, dout, out, lse)):
        ref.check(name, t, *want[name])


@pytest.mark.parametrize("causal", [True, False])
@pytest.mark.parametrize("n", [65, 300, 4100])
def test_attention_of_very_many_sequences(device, n, causal):
    """More sequences than a search step has lanes, most of them a few tokens
    long, some empty, and a long one among single tokens."""
    ql = [(i * 7) % 4 for i in range(n)]
    kl = [(i * 5) % 7 for i in range(n)]
    ql[n // 2], kl[n // 2] = 150, 170
    case = (BF16, 2, 1, 32, ql, kl, causal, None)
    call, dout = inputs(device, case)
    out, lse = bfhip.attention(**call, lse=True)
    back = grads(call, dout, out, lse)
    # The reference goes sequence by sequence: every 9th, and the long one.
    qs, ks = call["q_starts"].tolist(), call["k_starts"].tolist()
    some = [i for i in range(n) if i % max(1, n // 40) == 0 or i == n // 2]
    rows = torch.cat([torch.arange(qs[i], qs[i + 1], device=device) for i in some])
    keys = torch.cat([torch.arange(ks[i], ks[i + 1], device=device) for i in some])
    part = dict(call, q=call["q"][rows], k=call["k"][keys], v=call["v"][keys],
                q_starts=starts([ql[i] for i in some], device), k_starts=starts([kl[i] for i in some], device))
    want = ref.attention(**part, dout=dout[rows])
    for name, t, at in (("out", out, rows), ("dq", back[0], rows), ("dk", back[1], keys), ("dv", back[2], keys)):
        ref.check(name, t[at], *want[name])


def test_attention_of_a_prompt_among_single_tokens(device):
    """A batch that is dealt for single tokens and one that is dealt for
    prompts, the same sequences in both."""
    ql, kl = [1] * 60 + [90], [400] * 60 + [500]
    call, _ = inputs(device, (F16, 4, 2, 64, ql, kl, True, 20))
    ref.check("out", bfhip.attention(**call), *ref.attention(**call)["out"])


@pytest.mark.parametrize("dtype", [F32, F16, BF16])
@pytest.mark.parametrize("reach", [None, 5])
def test_attention_leaves_rows_outside_sequences(device, dtype, reach):
    """Rows before the first and behind the last sequence hold NaN and stay as
    they were, results and gradients alike; their contents reach nothing."""
    case = (dtype, 4, 2, 64, [33, 64, 2], [40, 64, 70], True, reach)
    call, dout = inputs(device, case)
    want, lse = bfhip.attention(**call, lse=True)
    clean = grads(call, dout, want, lse)
    pad = {}
    for name in ("q", "k", "v"):
        t = call[name]
        pad[name] = torch.full((t.shape[0] + 90, *t.shape[1:]), math.nan, dtype=dtype, device=device)
        pad[name][20:20 + t.shape[0]] = t
    wide = dict(call, **pad, q_starts=call["q_starts"] + 20, k_starts=call["k_starts"] + 20)
    n = dout.shape[0]
    out = torch.full_like(pad["q"], 7.0)
    got, lse2 = bfhip.attention(**wide, out=out, lse=True)
    assert torch.equal(got[20:20 + n], want) and (got[:20] == 7).all() and (got[20 + n:] == 7).all()
    assert torch.equal(lse2[:, 20:20 + n], lse)
    g = torch.full_like(pad["q"], math.nan)
    g[20:20 + n] = dout
    back = grads(wide, g, torch.where(got == 7, math.nan, got), lse2)
    for a, b in zip(back[:3], clean[:3]):
        assert torch.equal(a[20:20 + b.shape[0]], b)
    if reach is not None:
        assert torch.equal(back[3], clean[3])


@pytest.mark.parametrize("dtype", [F32, BF16])
def test_attention_masked_keys_hold_anything(device, dtype):
    """Keys a query does not see: infinities, NaN, the type's lowest value."""
    case = (dtype, 2, 2, 32, [100], None, True, None)
    call, _ = inputs(device, case)
    want = bfhip.attention(**call)
    for value in (math.nan, math.inf, -math.inf, torch.finfo(dtype).min):
        k = call["k"].clone()
        k[71:] = value
        got = bfhip.attention(**dict(call, k=k))
        assert torch.equal(got[:71], want[:71]), value


@pytest.mark.parametrize("dtype,size", [(F16, 20.0), (BF16, 100.0), (F32, 100.0)])
@pytest.mark.parametrize("causal", [True, False])
def test_attention_of_large_biases(device, dtype, size, causal):
    """A bias whose own exponential the type does not hold, on tiles that are
    not full: it cancels in the softmax and reaches no gradient by itself."""
    call, dout = inputs(device, (dtype, 4, 2, 32, [70, 3, 130], [70, 90, 131], causal, 6))
    call["bias"][:, :7] += size
    want = ref.attention(**call, dout=dout)
    out, lse = bfhip.attention(**call, lse=True)
    ref.check("out", out, *want["out"])
    for name, t in zip(("dq", "dk", "dv", "dbias"), grads(call, dout, out, lse)):
        ref.check(name, t, *want[name])


@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("causal", [True, False])
@pytest.mark.parametrize("ql", [[33, 200], [1, 2]])
def test_attention_behind_many_other_rows(device, dtype, causal, ql):
    """A first sequence that begins tiles away from the tensor's first row."""
    call, dout = inputs(device, (dtype, 4, 2, 64, [700] + ql, [900, 300, 650], causal, 5))
    for name in ("q_starts", "k_starts"):
        call[name] = call[name][1:].contiguous()
    want = ref.attention(**call, dout=dout)
    out, lse = bfhip.attention(**call, lse=True)
    rows, keys = slice(700, None), slice(900, None)
    ref.check("out", out[rows], want["out"][0][rows], want["out"][1][rows])
    back = grads(call, dout, out, lse)
    for name, t, at in zip(("dq", "dk", "dv", "dbias"), back, (rows, keys, keys, slice(None))):
        ref.check(name, t[at], want[name][0][at], want[name][1][at])


def test_attention_bias_can_mask(device):
    """Scores of -inf: by distance, and for whole rows; the lowest finite value
    masks too, but leaves a softmax where every key has it."""
    case = (F32, 2, 1, 32, [70, 3], None, False, 40)
    call, dout = inputs(device, case)
    bias = call["bias"]
    bias[0, :35] = -math.inf
    bias[1, :] = -math.inf
    call["bias"] = bias
    out, lse = bfhip.attention(**call, lse=True)
    want = ref.attention(**call, dout=dout)
    assert torch.isneginf(lse[1]).all() and not out[:, 1].any()
    ref.check("out", out, *want["out"])
    back = grads(call, dout, out, lse)
    for name, t in zip(("dq", "dk", "dv"), back):
        ref.check(name, t, *want[name])
    assert not back[0][:, 1].any()
    low = dict(call, bias=torch.full_like(bias, torch.finfo(F32).min / 2))
    out = bfhip.attention(**low)
    for b, n in ((0, 70), (70, 3)):
        mean = call["v"][b:b + n].double().mean(0)
        assert ((out[b:b + n].double() - mean).abs() <= 80 * 2.0 ** -24 * call["v"].abs().max()).all()


@pytest.mark.parametrize("case", [(F32, 2, 1, 16, [9, 4], [12, 3], True, 3), (F32, 2, 2, 8, [6], [5], False, 2)], ids=str)
def test_attention_gradient_by_differences(device, case):
    call, dout = inputs(device, case, layout="plain")
    out, lse = bfhip.attention(**call, lse=True)
    back = grads(call, dout, out, lse)
    g = gen(device, 1)
    for name, grad in zip(("q", "k", "v", "bias"), back):
        way = randn(g, *call[name].shape).double()
        step, value = 1e-5, call[name].double()
        loss = [(ref.attention(**dict(call, **{name: value + sign * step * way}))["out"][0] * dout.double()).sum()
                for sign in (1, -1)] if name == "bias" else None
        if loss is None:
            moved = {n: call[n].double() for n in "qkv"}
            loss = []
            for sign in (1, -1):
                moved[name] = value + sign * step * way
                loss.append((ref.attention(**dict(call, **moved))["out"][0] * dout.double()).sum())
        slope = (loss[0] - loss[1]) / (2 * step)
        assert abs((grad.double() * way).sum() - slope) <= 1e-5 * (grad.double() * way).abs().sum(), name


def test_attention_without_rows(device):
    q = torch.empty((0, 2, 32), device=device)
    k = torch.randn((5, 2, 32), device=device)
    at = dict(q_starts=starts([0, 0], device), k_starts=starts([3, 2], device))
    out, lse = bfhip.attention(q, k, k, **at, lse=True)
    bias = torch.zeros((2, 9), device=device)
    dq, dk, dv, db = bfhip.attention_backward(q, q, k, k, out, lse, **at, bias=bias)
    assert out.shape == dq.shape == (0, 2, 32) and not dk.any() and not dv.any() and not db.any()
    # No keys at all: every query is left without.
    out, lse = bfhip.attention(k, q, q, at["k_starts"], at["q_starts"], lse=True)
    assert not out.any() and torch.isneginf(lse).all()
    dq, dk, dv = bfhip.attention_backward(k, k, q, q, out, lse, at["k_starts"], at["q_starts"])
    assert not dq.any() and dk.shape == (0, 2, 32)
    # No sequences: rows stay.
    none = torch.zeros(1, dtype=torch.int32, device=device)
    out = torch.full_like(k, 7.0)
    bfhip.attention(k, k, k, none, none, out=out)
    assert (out == 7).all()
    *_, db = bfhip.attention_backward(k, k, k, k, k, torch.zeros((2, 5), device=device), none, none, bias=bias)
    assert not db.any()


def test_attention_starts_out_of_range_are_clamped(device):
    """Starts past the rows, before them or descending read and write nothing
    outside the rows; sequences that are whole come out right."""
    call, _ = inputs(device, (BF16, 2, 2, 64, [50, 30], None, True, None), layout="plain")
    bad = torch.tensor([0, 50, 80, 10 ** 9, -5, 2 ** 31 - 1], dtype=torch.int32, device=device)
    bad[4] = 80
    out = torch.zeros_like(call["q"])
    got = bfhip.attention(**dict(call, q_starts=bad, k_starts=bad), out=out)
    # (How the work is dealt depends on the number of sequences, so the bits may.)
    ref.check("out", got, *ref.attention(**call)["out"])


# ----------------------------------------------------------------- in sequence
def block(x, w, starts_, table, buckets, dy):
    """One transformer block's attention half and its gradients: norm, fused
    projection, attention with a learned bias, and back."""
    y, mean, rstd = bfhip.layer_norm(x, w["gamma"], w["beta"], stats=True)
    qkv = bfhip.gemm_f32(y, w["qkv"])
    q, k, v = (t.unflatten(1, (-1, 32)) for t in qkv.split([128, 64, 64], 1))
    bias = bfhip.position_bias(table, buckets)
    out, lse = bfhip.attention(q, k, v, starts_, starts_, causal=True, bias=bias, lse=True)
    dq, dk, dv, dbias = bfhip.attention_backward(dy, q, k, v, out, lse, starts_, starts_, causal=True, bias=bias)
    dtable = bfhip.position_bias_backward(dbias, buckets, table.shape[0])
    dqkv = torch.cat([t.flatten(1) for t in (dq, dk, dv)], 1)
    dyn = bfhip.gemm_f32(dqkv, w["qkv_t"])
    dx, dgamma, dbeta = bfhip.layer_norm_backward(dyn, x, mean, rstd, w["gamma"])
    return out, dtable, dx, dgamma, dbeta


def block_inputs(device, seed=0):
    g = gen(device, seed)
    lens = [70, 1, 129]
    n = sum(lens)
    qkv = randn(g, 256, 96, scale=0.1)
    w = dict(gamma=1 + randn(g, 96, scale=0.1), beta=randn(g, 96, scale=0.1), qkv=qkv, qkv_t=qkv.T.contiguous())
    reach = 20
    buckets = (torch.arange(2 * reach + 1, device=device) // 4).int()
    return randn(g, n, 96), w, starts(lens, device), randn(g, 11, 4), buckets, randn(g, n, 4, 32)


def test_operators_in_sequence(device):
    x, w, at, table, buckets, dy = block_inputs(device)
    out, dtable, dx, dgamma, dbeta = block(x, w, at, table, buckets, dy)
    leaves = [t.double().requires_grad_() for t in (x, w["gamma"], w["beta"], table)]
    X, G, B, T = leaves
    h = (X - X.mean(1, keepdim=True)) / (X.var(1, unbiased=False, keepdim=True) + 1e-5).sqrt() * G + B
    qkv = h @ w["qkv"].double().T
    q, k, v = (t.unflatten(1, (-1, 32)) for t in qkv.split([128, 64, 64], 1))
    rows = []
    for s, e in zip(at.tolist(), at.tolist()[1:]):
        n = e - s
        far = torch.arange(n, device=device)[None, :] - torch.arange(n, device=device)[:, None]
        add = T[buckets.long()[far.clamp(-20, 20) + 20]].movedim(2, 0)
        score = (q[s:e].movedim(1, 0) @ k[s:e].repeat_interleave(2, 1).permute(1, 2, 0).contiguous()) * 32 ** -0.5 + add
        p = score.masked_fill(far > 0, -math.inf).softmax(2)
        rows.append((p @ v[s:e].repeat_interleave(2, 1).movedim(1, 0).contiguous()).movedim(0, 1))
    want = torch.cat(rows)
    (want * dy.double()).sum().backward()
    # The linear rounds its operands to bf16 (half a step 2^-8 each, of many
    # independent terms): 1e-2 of the norm holds for everything behind it.
    for name, a, b in (("out", out, want), ("dtable", dtable, T.grad), ("dx", dx, X.grad), ("dgamma", dgamma, G.grad),
                       ("dbeta", dbeta, B.grad)):
        rel = ((a.double() - b.detach()).norm() / b.detach().norm()).item()
        print(f"[rel] {name} {rel:.2e}")
        assert rel <= 2e-2, name


def test_captured_and_replayed(device):
    """Two graphs of the whole run, replayed in turn with eager calls of other
    sizes between, give the eager bits every time."""
    sets = [block_inputs(device, seed) for seed in (1, 2)]
    want = [block(*s) for s in sets]
    torch.cuda.synchronize()
    graphs = []
    for s in sets:
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            out = block(*s)
        graphs.append((g, out))
    small, dout = inputs(device, CASES[0])
    for rep in range(3):
        for (g, out), w in zip(graphs, want):
            for t in out:
                t.zero_()
            g.replay()
            torch.cuda.synchronize()
            assert all(torch.equal(a, b) for a, b in zip(out, w)), rep
            bfhip.attention(**small)
            torch.cuda.synchronize()


@pytest.mark.parametrize("case", [CASES[4], CASES[10], CASES[17], (BF16, 8, 2, 128, [2500], None, True, 60)], ids=str)
def test_split_work_captured_and_replayed(device, case):
    """Keys and queries in parts: a workspace between the launches of a graph."""
    call, dout = inputs(device, case)

    def run():
        out, lse = bfhip.attention(**call, lse=True)
        return out, lse, *grads(call, dout, out, lse)

    want = run()
    torch.cuda.synchronize()
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        got = run()
    for rep in range(3):
        for t in got:
            t.zero_()
        g.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(got, want)), rep
        run()
        torch.cuda.synchronize()


@pytest.mark.parametrize("case", [(F32, 6, 3, 32, [65, 1, 200, 0, 333, 9], [60, 130, 200, 17, 500, 9], True, None),
                                  (F32, 2, 1, 128, [70, 3], [1000, 260], False, None),
                                  (F32, 5, 5, 40, [129, 64], [33, 700], True, None),
                                  (F32, 1, 1, 72, [300], [129], False, None)], ids=str)
def test_queries_on_split_keys(device, case):
    """fp32 gradients whose walks are split where CUs are idle."""
    test_attention(device, case, "fused")
    test_split_work_captured_and_replayed(device, case)


@pytest.mark.parametrize("case", [(BF16, 8, 2, 128, [1] * 40 + [100, 0, 5, 4], [700] * 43 + [0], True, 30),
                                  (F32, 4, 1, 40, [2, 0, 1, 0, 0, 0, 17, 0, 0], [3000, 5, 2000, 0, 7, 8, 900, 1, 0], True, None),
                                  (F16, 3, 3, 64, [1, 16, 17, 3, 0, 0, 1], [90, 4000, 300, 1, 5, 0, 20], False, 4),
                                  (F16, 20, 1, 32, [1, 2, 0, 0, 0, 0, 0, 0, 9], [900] * 9, True, None),
                                  (F16, 20, 1, 32, [3, 0, 1, 0, 1, 0, 0, 2, 0, 0], [900] * 10, True, None),
                                  (BF16, 6, 2, 32, [1] * 70 + [5, 6] + [0] * 8, [64] * 80, False, None)], ids=str)
def test_prompts_among_single_tokens(device, case):
    """Batches whose sequences are dealt in two ways, on either side of the
    border between them."""
    test_attention(device, case, "heads")
    test_split_work_captured_and_replayed(device, case)


def test_on_a_stream_of_its_own(device):
    s = block_inputs(device, 3)
    want = block(*s)
    side = torch.cuda.Stream()
    torch.cuda.synchronize()
    x, w, at, table, buckets, dy = s
    y, mean, rstd = bfhip.layer_norm(x, w["gamma"], w["beta"], stats=True, stream=side)
    bias = bfhip.position_bias(table, buckets, stream=side)
    side.synchronize()
    with torch.cuda.stream(side):
        got = block(*s)
    side.synchronize()
    assert all(torch.equal(a, b) for a, b in zip(got, want))
    assert torch.equal(bias, bfhip.position_bias(table, buckets))
    assert torch.equal(y, bfhip.layer_norm(x, w["gamma"], w["beta"]))
