"""The transformer operators (include/bfhip_transformer.h) where their numbers,
rows or deals come to an edge: biases of any finite size, gradients below a
type's smallest numbers, starts of any value, rows far into a buffer, batches
with empty places."""

import ctypes as C
import math

import pytest
import torch

import bfhip
import transformer_ref as ref
from test_gpu_transformer import BF16, F16, F32, gen, grads, inputs, randn, starts

pytestmark = pytest.mark.gpu


def backward_into(call, dout, out, lse, dq, dk, dv, dbias=None):
    """bfhip_attention_backward into the caller's gradients, dbias or none."""
    q, k, v = call["q"], call["k"], call["v"]
    bias = call["bias"]
    code = {F32: 0, F16: 1, BF16: 2}[q.dtype]
    desc = bfhip.AttentionDesc(code, call["q_starts"].numel() - 1, q.shape[1], k.shape[1], q.shape[2], int(call["causal"]),
                               0 if bias is None else bias.shape[1] // 2, call["scale"], q.shape[0], k.shape[0],
                               call["q_starts"].data_ptr(), call["k_starts"].data_ptr(),
                               None if bias is None else bias.data_ptr())
    lib = bfhip.hip_lib()
    size = lib.bfhip_attention_backward_workspace(desc)
    work = torch.empty(max(size, 1), dtype=torch.uint8, device=q.device)
    row = lambda t: bfhip.Rows(t.data_ptr(), t.stride(0), t.stride(1) if t.shape[1] > 1 else 0)
    err = C.create_string_buffer(256)
    ok = lib.bfhip_attention_backward(desc, row(q), row(k), row(v), row(out), lse.data_ptr(), row(dout), row(dq), row(dk),
                                      row(dv), None if dbias is None else dbias.data_ptr(), work.data_ptr(), size,
                                      torch.cuda.current_stream().cuda_stream, err, 256)
    assert ok, err.value
    return dq, dk, dv

LOWEST = torch.finfo(F32).min

# Prompts, single tokens, single tokens on split keys.
SIZED = [(F32, 2, 1, 32, [70, 3], [90, 3], False, 4), (BF16, 4, 2, 128, [150, 1], [700, 400], False, 20),
         (F16, 4, 1, 64, [1, 2, 1], [40, 3000, 1], True, 9), (BF16, 2, 2, 16, [130, 64], [130, 64], True, 300)]


@pytest.mark.parametrize("value", [LOWEST, LOWEST / 1.3, LOWEST / 2, -1e9, -LOWEST])
@pytest.mark.parametrize("case", SIZED, ids=str)
def test_attention_where_every_key_has_one_large_bias(device, case, value):
    """It swallows the scores and leaves a softmax of equal ones: the mean of
    the seen values."""
    call, _ = inputs(device, case)
    flat = dict(call, q=torch.zeros_like(call["q"]), bias=torch.zeros_like(call["bias"]))
    got = bfhip.attention(**dict(call, bias=torch.full_like(call["bias"], value)))
    ref.check("out", got, *ref.attention(**flat)["out"])


@pytest.mark.parametrize("case", SIZED, ids=str)
def test_attention_lowest_bias_masks(device, case):
    """Keys of the lowest bias beside others: as if they were not there."""
    call, dout = inputs(device, case)
    reach = call["bias"].shape[1] // 2
    results = []
    for value in (-math.inf, LOWEST):
        bias = call["bias"].clone()
        bias[:, :reach] = value  # (a query's own position keeps its bias)
        there = dict(call, bias=bias)
        out, lse = bfhip.attention(**there, lse=True)
        results.append((out, lse, *grads(there, dout, out, lse)))
    lens = [t.diff() for t in (call["q_starts"], call["k_starts"])]
    assert (lens[0] <= lens[1]).all()
    assert all(torch.equal(a, b) for a, b in zip(*results))


@pytest.mark.parametrize("with_dbias", [True, False])
@pytest.mark.parametrize("value", [LOWEST, LOWEST / 2, -1e9, -3e4, 5e5, -LOWEST])
@pytest.mark.parametrize("case", SIZED + [(F32, 2, 1, 128, [3, 70], [600, 300], False, 2047),
                                          (F16, 2, 1, 64, [300], [300], False, 5)], ids=str)
def test_attention_gradients_where_every_key_has_one_large_bias(device, case, value, with_dbias):
    """A constant beside every score of a row leaves its probabilities as they
    are, however large it is (here with scores of zero, which no bias
    swallows); another head has ordinary ones."""
    call, dout = inputs(device, case)
    call["q"].narrow(1, 0, 1).zero_()
    plain = dict(call, bias=call["bias"].clone())
    plain["bias"][0] = 0
    call["bias"] = plain["bias"].clone()
    call["bias"][0] = value
    want = ref.attention(**plain, dout=dout)
    out, lse = bfhip.attention(**call, lse=True)
    if with_dbias:
        back = grads(call, dout, out, lse)
    else:
        back = backward_into(call, dout, out, lse, *(torch.zeros_like(call[n]) for n in "qkv"))
    ref.check("out", out, *want["out"])
    for name, t in zip(("dq", "dk", "dv", "dbias"), back):
        ref.check(name, t, *want[name])


@pytest.mark.parametrize("case", [(F32, 2, 1, 32, [70, 3], [90, 3], True, 8), (BF16, 4, 2, 128, [300, 1], [290, 1], True, 20),
                                  (F16, 4, 1, 64, [700], [700], True, 9)], ids=str)
def test_attention_gradients_of_some_rows_far_from_zero(device, case):
    """The nearest keys masked by a large bias: a sequence's first queries see
    no others."""
    call, dout = inputs(device, case)
    reach = call["bias"].shape[1] // 2
    call["bias"][:, reach - 4:reach + 1] -= 3000.0  # (distances -4 to 0)
    want = ref.attention(**call, dout=dout)
    out, lse = bfhip.attention(**call, lse=True)
    assert (lse < -2000).any() and (lse > -50).any()
    ref.check("out", out, *want["out"])
    for name, t in zip(("dq", "dk", "dv", "dbias"), grads(call, dout, out, lse)):
        ref.check(name, t, *want[name])

# (rows of the tensors, starts): a query's and a key's alike.
STARTS = [[-7, 50, 80, 10 ** 9], [-2 ** 31, -5, 30, 20, 80, 2 ** 31 - 1], [80, 0, 80], [0, 50, 30, 80, 79, 80],
          [300, -1, 40, 40, 80, -3]]


@pytest.mark.parametrize("at", STARTS, ids=str)
@pytest.mark.parametrize("case", [(BF16, 4, 2, 64, None), (F32, 2, 1, 128, None), (F16, 4, 4, 32, 7), (F32, 3, 1, 40, 3)], ids=str)
@pytest.mark.parametrize("few", [False, True])
def test_attention_reads_and_writes_its_rows_only(device, case, at, few):
    """Starts past the rows, before them and descending are clamped: nothing
    outside the rows is read into a result or written, in either direction.
    Where the clamped starts ascend, every sequence comes out right."""
    dtype, heads, kv_heads, dim, reach = case
    tq, guard = 80, 70
    scale_k = 40 if few else 1  # keys per query, so that keys are split
    call, dout = inputs(device, (dtype, heads, kv_heads, dim, [tq], [tq * scale_k], True, reach), layout="plain")
    q_at = torch.tensor(at, dtype=torch.int64).clamp(-2 ** 31, 2 ** 31 - 1)
    k_at = (q_at * scale_k).clamp(-2 ** 31, 2 ** 31 - 1)
    pad = 40 if few else 0  # empty sequences: so few queries per sequence that they are dealt as few
    q_at, k_at = (torch.cat([t, t[-1:].expand(pad)]).int().to(device) for t in (q_at, k_at))

    def inside(t, fill):
        wide = torch.full((t.shape[0] + 2 * guard, *t.shape[1:]), fill, dtype=t.dtype, device=device)
        wide[guard:guard + t.shape[0]] = t
        return wide, wide[guard:guard + t.shape[0]]

    (_, q), (_, k), (_, v), (_, g) = (inside(t, math.nan) for t in (call["q"], call["k"], call["v"], dout))
    wide = {}
    for name, like in (("out", q), ("dq", q), ("dk", k), ("dv", v)):
        wide[name] = inside(torch.zeros_like(like), 7.0)
    there = dict(call, q=q, k=k, v=v, q_starts=q_at, k_starts=k_at)
    out = wide["out"][1]
    _, lse = bfhip.attention(**there, out=out, lse=True)
    clamped = [t.clamp(0, n).tolist() for t, n in ((q_at.cpu(), tq), (k_at.cpu(), tq * scale_k))]
    owned = torch.zeros(tq)
    for a, b in zip(clamped[0], clamped[0][1:]):
        owned[a:max(a, b)] += 1
    lse = torch.where((owned > 0).to(device), lse, 0.0)  # (rows of no sequence have none)
    dbias = None if reach is None else torch.empty_like(call["bias"])
    backward_into(there, g, out, lse, wide["dq"][1], wide["dk"][1], wide["dv"][1], dbias)
    for name, (buffer, _) in wide.items():
        assert (buffer[:guard] == 7).all() and (buffer[-guard:] == 7).all(), name
    for a, b, c, d in zip(clamped[0], clamped[0][1:], clamped[1], clamped[1][1:]):
        if a == b or clamped[0] != sorted(clamped[0]):
            continue
        alone = dict(call, q=q[a:b], k=k[c:d], v=v[c:d], q_starts=starts([b - a], device), k_starts=starts([d - c], device))
        want = ref.attention(**alone, dout=g[a:b])
        for name, rows in (("out", slice(a, b)), ("dq", slice(a, b)), ("dk", slice(c, d)), ("dv", slice(c, d))):
            ref.check(name, wide[name][1][rows], *want[name])


@pytest.mark.parametrize("ql,kl,skip_q", [([5, 70], [200, 300], 140000), ([1, 1], [700, 900], 0)], ids=str)
def test_attention_of_rows_past_four_gib(device, ql, kl, skip_q):
    """A long cache: rows whose offsets no 32-bit number of bytes holds."""
    call, dout = inputs(device, (BF16, 4, 2, 64, ql, kl, True, None), layout="plain")
    stride, skip = 16384, 140000  # 32 KiB a token: 4.6 GB before the first row
    room = torch.zeros(((skip + sum(kl)) * stride,), dtype=BF16, device=device)

    def far(t, at, skip):
        h = t.shape[1] * t.shape[2]
        view = room.view(-1, stride)[:, at:at + h].unflatten(1, t.shape[1:])
        view[skip:skip + t.shape[0]] = t
        return view[:skip + t.shape[0]]

    there = dict(call, q=far(call["q"], 0, skip_q), k=far(call["k"], 1024, skip), v=far(call["v"], 2048, skip),
                 q_starts=call["q_starts"] + skip_q, k_starts=call["k_starts"] + skip)
    out = far(torch.zeros_like(call["q"]), 4096, skip_q)
    _, lse = bfhip.attention(**there, out=out, lse=True)
    want = ref.attention(**call, dout=dout)
    ref.check("out", out[skip_q:], *want["out"])
    skips = dict(q=skip_q, k=skip, v=skip)
    back = backward_into(there, far(dout, 5120, skip_q), out, lse, *(far(torch.zeros_like(call[n]), 6144 + 1024 * i, skips[n])
                                                                     for i, n in enumerate("qkv")))
    for n, t in zip("qkv", back):
        ref.check("d" + n, t[skips[n]:], *want["d" + n])


@pytest.mark.parametrize("case", [(F16, 4, 2, 64, [1] * 60 + [90], [400] * 60 + [500], True, 20),
                                  (BF16, 8, 2, 128, [1] * 30 + [40], [700] * 30 + [60], False, None)], ids=str)
def test_attention_of_the_same_sequences_in_both_deals(device, case):
    """Single tokens and a prompt as a batch of few queries, and with rows of
    no sequence behind them as a batch of prompts."""
    call, dout = inputs(device, case)
    want = ref.attention(**call)["out"]
    n = call["q"].shape[0]
    for extra in (0, 20 * n):
        q = torch.zeros((n + extra, *call["q"].shape[1:]), dtype=call["q"].dtype, device=device)
        q[:n] = call["q"]
        ref.check(f"out, {extra} rows behind", bfhip.attention(**dict(call, q=q))[:n], *want)


@pytest.mark.parametrize("case", [(BF16, 8, 2, 64, 150, 200, 256), (F32, 4, 1, 32, 100, 300, 130)], ids=str)
def test_prompt_in_a_batch_with_empty_places(device, case):
    """A batch of a fixed number of places, most of them empty: its prompt
    takes the prompts' launch, whose bits are those of a batch of prompts."""
    dtype, heads, kv_heads, dim, prompt, keys, places = case
    ql, kl = [1] * 25 + [prompt], [300] * 25 + [keys]
    many, _ = inputs(device, (dtype, heads, kv_heads, dim, [prompt] * 80, [keys] * 80, True, None), layout="plain")
    call, dout = inputs(device, (dtype, heads, kv_heads, dim, ql + [0] * (places - 26), kl + [0] * (places - 26), True, None),
                        layout="plain")
    assert call["q"].shape[0] < places
    for name, n in (("q", prompt), ("k", keys), ("v", keys)):
        call[name][-n:] = many[name][:n]
    out, lse = bfhip.attention(**call, lse=True)
    want = ref.attention(**call, dout=dout)
    ref.check("out", out, *want["out"])
    for name, t in zip(("dq", "dk", "dv"), grads(call, dout, out, lse)):
        ref.check(name, t, *want[name])
    assert torch.equal(out[-prompt:], bfhip.attention(**many)[:prompt])


@pytest.mark.parametrize("case", [(F32, 2, 1, 40, [70, 3], [90, 30], True, 4), (F32, 4, 2, 12 * 8, [1, 1], [900, 65], True, None),
                                  (F32, 3, 3, 8, [130], [200], False, None)], ids=str)
def test_attention_of_rows_on_16_bytes(device, case):
    """fp32 rows that begin at odd multiples of 16 bytes."""
    call, dout = inputs(device, case, layout="plain")

    def odd(t):
        heads, dim = t.shape[1:]
        wide = torch.full((t.shape[0] * (heads * (dim + 4) + 4 * (heads % 2 == 0)) + 4,), 3.0, device=device)
        assert (wide.data_ptr() + 16) % 32 == 16
        view = wide[4:].view(t.shape[0], -1)[:, :heads * (dim + 4)].unflatten(1, (heads, dim + 4))[:, :, :dim]
        assert view.stride(0) % 8 == 4 and view.stride(1) % 8 == 4
        view.copy_(t)
        return view

    call.update({n: odd(call[n]) for n in "qkv"})
    dout = odd(dout)
    want = ref.attention(**call, dout=dout)
    out = odd(torch.zeros_like(dout))
    _, lse = bfhip.attention(**call, out=out, lse=True)
    ref.check("out", out, *want["out"])
    dbias = None if call["bias"] is None else torch.empty_like(call["bias"])
    for name, t in zip(("dq", "dk", "dv"), backward_into(call, dout, out, lse, *(odd(torch.zeros_like(call[n])) for n in "qkv"), dbias)):
        ref.check(name, t, *want[name])


@pytest.mark.parametrize("keys", [2, 300])
def test_attention_gradients_beyond_the_type(device, keys):
    """fp16 gradients that the type does not hold are infinite, not NaN."""
    q = torch.zeros((1, 1, 8), dtype=F16, device=device)
    k = torch.zeros((keys, 1, 8), dtype=F16, device=device)
    v = torch.zeros_like(k)
    k[0, 0, 0], k[1, 0, 0] = 4.0, -4.0
    q[0, 0, 1] = 6.0
    k[0, 0, 1] = k[1, 0, 1] = 6.0  # (the others have almost no weight)
    v[0, 0], v[1, 0] = 300.0, -300.0
    dout = torch.full_like(q, 300.0)
    at = starts([1], device), starts([keys], device)
    out, lse = bfhip.attention(q, k, v, *at, scale=1.0, lse=True)
    dq, dk, dv = bfhip.attention_backward(dout, q, k, v, out, lse, *at, scale=1.0)
    # ds = +-1/2 * 8 * 300 * 300 = +-360000 for the first two keys.
    assert dq[0, 0, 0] == math.inf
    assert dk[0, 0, 1] == math.inf and dk[1, 0, 1] == -math.inf
    assert torch.isfinite(dv).all()


@pytest.fixture
def whole_range(monkeypatch):
    """Bounds without what fp16's smallest numbers would cost inside: only
    results are rounded to them."""
    small = ref.tiny
    monkeypatch.setattr(ref, "tiny", lambda dtype: 0.0)
    return small


@pytest.mark.parametrize("case", [(F16, 2, 1, 64, [40, 3], [300, 60], False, 5), (F16, 2, 2, 32, [200], [600], False, 9),
                                  (F16, 4, 1, 128, [129], None, True, None), (F16, 1, 1, 16, [3], [5000], False, None)], ids=str)
def test_attention_of_small_gradients(device, case, whole_range):
    """fp16: probabilities and score gradients far below the type's smallest
    normal number reach the gradients."""
    call, dout = inputs(device, case)
    if call["bias"] is not None:  # most keys' weights near 2^-24
        call["bias"][:, :3] -= 17.0
    else:
        call["q"].mul_(0.05)
        call["k"].mul_(16.0)
    heads, kv_heads, t = dout.shape[1], call["k"].shape[1], whole_range(F16)
    group = heads // kv_heads
    for size in (1.0, 2.0 ** -17):
        g = (dout * size).contiguous()
        want = ref.attention(**call, dout=g)
        # p enters times 2^12, ds times a power of two that takes the largest
        # |dout . v| to 2^13 or more, in the keys' walk 4 times it: each loses
        # 2^-25 there.
        most = max((g[:, h].double() @ call["v"][:, h // group].double().T).abs().max() for h in range(heads))
        lost = most * 2.0 ** -38 * abs(call["scale"])
        total = lambda x: x.abs().double().sum(0)
        shared = lambda x: total(x).unflatten(0, (kv_heads, group)).sum(1)
        floor = dict(dq=lost * total(call["k"]).repeat_interleave(group, 0) + t, dk=4 * lost * shared(call["q"]) + t,
                     dv=2.0 ** -37 * shared(g) + t, dbias=0.0)
        out, lse = bfhip.attention(**call, lse=True)
        for name, got in zip(("dq", "dk", "dv", "dbias"), grads(call, g, out, lse)):
            value, bound = want[name]
            ref.check(f"{name} x {size}", got, value, bound + floor[name])


def test_attention_gradients_of_uneven_rows(device):
    """fp16: rows and keys whose gradients differ by many powers of two, the
    small ones first and last."""
    call, dout = inputs(device, (F16, 4, 2, 64, [300, 90], [300, 500], True, None))
    size = 2.0 ** torch.randint(-14, 7, (390, 1, 1), generator=gen(device, 5), device=device)
    size[:64], size[-64:] = 2.0 ** -14, 2.0 ** -14
    dout = (dout * size).half()
    want = ref.attention(**call, dout=dout)
    out, lse = bfhip.attention(**call, lse=True)
    for name, t in zip(("dq", "dk", "dv"), grads(call, dout, out, lse)):
        ref.check(name, t, *want[name])


@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("n", [1, 5, 100, 257])
def test_layer_norm_gradients_of_large_equal_rows(device, dtype, n):
    """Rows without spread, far from zero: what lies past their end reaches
    nothing."""
    x = torch.full((3, n), 2.0 ** 112, dtype=dtype, device=device)
    x[1] = -1.0
    g = gen(device, n)
    gamma, dy = 1 + randn(g, n, scale=0.2), randn(g, 3, n, dtype=dtype)
    y, mean, rstd = bfhip.layer_norm(x, gamma, eps=1e-10, stats=True)
    dx, dgamma, dbeta = bfhip.layer_norm_backward(dy, x, mean, rstd, gamma)
    assert torch.equal(mean, x[:, 0].float()) and not y.any()
    want = ref.layer_norm(torch.zeros_like(x), gamma, None, 1e-10, dy)  # (the same centred values)
    for name, got in dict(dx=dx, dgamma=dgamma, dbeta=dbeta).items():
        ref.check(name, got, *want[name])


@pytest.mark.parametrize("case", [(F32, 2, 1, 32, [70], [90], True, None), (BF16, 4, 2, 64, [1, 2], [700, 3], True, 3)], ids=str)
def test_attention_without_scale_takes_no_scores(device, case):
    """Scale 0, and products of queries and keys near 2^120."""
    call, _ = inputs(device, case)
    call["scale"] = 0.0
    want = ref.attention(**dict(call, q=torch.zeros_like(call["q"])))
    for name in "qk":
        call[name].mul_(2.0 ** 58)
    ref.check("out", bfhip.attention(**call), *want["out"])


def test_attention_of_one_token_of_any_stride(device):
    """The stride between tokens means nothing where there is one."""
    call, dout = inputs(device, (F32, 4, 2, 32, [1], [1], True, None), layout="plain")
    want = bfhip.attention(**call)
    for stride in (1, 7, 16):
        odd = {n: call[n].as_strided(call[n].shape, (stride, 32, 1)) for n in "qkv"}
        out = torch.empty_like(want).as_strided(want.shape, (stride, 32, 1))
        got, lse = bfhip.attention(**dict(call, **odd), out=out, lse=True)
        assert torch.equal(got, want)
        back = grads(dict(call, **odd), dout, got, lse)
        assert all(torch.isfinite(t).all() for t in back)


@pytest.mark.parametrize("case", [(BF16, 8, 2, 64, [1] * 12, 4000, True), (F16, 4, 1, 128, [1, 3, 1, 2], 900, True),
                                  (F32, 2, 2, 32, [70, 1, 30], 300, False)], ids=str)
def test_attention_of_caches_with_room(device, case):
    """Keys kept in places of a fixed size: what a place has left over is a
    sequence without queries, whatever lies there."""
    dtype, heads, kv_heads, dim, ql, room, causal = case
    g = gen(device, 7)
    kl = torch.randint(max(ql), room, (len(ql),), generator=g, device=device).tolist()
    call, dout = inputs(device, (dtype, heads, kv_heads, dim, ql, kl, causal, None), layout="plain")
    want = ref.attention(**call, dout=dout)
    wide = {n: torch.full((room * len(ql), kv_heads, dim), math.nan, dtype=dtype, device=device) for n in "kv"}
    rows = torch.cat([torch.arange(room * i, room * i + n, device=device) for i, n in enumerate(kl)])
    for n in "kv":
        wide[n][rows] = call[n]
    q_at, k_at = [0], [0]
    for i, (n, m) in enumerate(zip(ql, kl)):
        q_at += [q_at[-1] + n] * 2
        k_at += [room * i + m, room * (i + 1)]
    there = dict(call, **wide, q_starts=torch.tensor(q_at, device=device).int(), k_starts=torch.tensor(k_at, device=device).int())
    out, lse = bfhip.attention(**there, lse=True)
    ref.check("out", out, *want["out"])
    dq, dk, dv = grads(there, dout, out, lse)
    for name, t in (("dq", dq), ("dk", dk[rows]), ("dv", dv[rows])):
        ref.check(name, t, *want[name])
    left = torch.ones(dk.shape[0], dtype=torch.bool, device=device)
    left[rows] = False
    assert not dk[left].any() and not dv[left].any()


@pytest.mark.parametrize("case", [(BF16, 4, 2, 64, None), (F16, 4, 1, 32, 6), (F32, 2, 1, 128, None)], ids=str)
def test_attention_replayed_with_other_starts(device, case):
    """A captured call reads its starts when it runs."""
    dtype, heads, kv_heads, dim, reach = case
    lens = [([70, 1, 9], [300, 400, 20]), ([1, 78, 1], [20, 100, 600]), ([0, 80, 0], [360, 355, 5])]
    call, dout = inputs(device, (dtype, heads, kv_heads, dim, *lens[0], True, reach))

    def run(c):
        out, lse = bfhip.attention(**c, lse=True)
        return out, lse, *grads(c, dout, out, lse)

    run(call)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got = run(call)
    for ql, kl in lens[1:] + lens[:1]:
        for name, n in (("q_starts", ql), ("k_starts", kl)):
            call[name].copy_(starts(n, device))
        for t in got:
            t.zero_()
        graph.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(got, run(call)))
        torch.cuda.synchronize()


@pytest.mark.parametrize("dtype", [F16, BF16, F32])
@pytest.mark.parametrize("case", [(2, 1, 64, [100, 3], [100, 9], True, None), (2, 2, 32, [70, 30], [500, 30], False, 4),
                                  (1, 1, 16, [40, 3], [3000, 60], False, None)], ids=str)
@pytest.mark.parametrize("value", [math.inf, math.nan])
def test_attention_gradients_that_are_not_finite_show(device, dtype, case, value):
    """An infinite dout: its query's gradient is not finite, nor are those of the
    keys that it sees; other queries' and other sequences' are what they were."""
    call, dout = inputs(device, (dtype, *case))
    want = ref.attention(**call, dout=dout)
    out, lse = bfhip.attention(**call, lse=True)
    dout[17, 0] = value
    dq, dk, dv, *_ = grads(call, dout, out, lse)
    assert not torch.isfinite(dq[17, 0]).any()
    assert not torch.isfinite(dk[:17, 0]).any() and not torch.isfinite(dv[:17, 0]).any()
    others = torch.ones(dq.shape[:2], dtype=torch.bool, device=device)
    others[17, 0] = False
    ref.check("dq", dq[others], want["dq"][0][others], want["dq"][1][others])
    n = call["k_starts"][1]
    for name, t in (("dk", dk), ("dv", dv)):
        ref.check(name, t[n:], want[name][0][n:], want[name][1][n:])


def test_calls_on_two_streams_at_once(device):
    """Split work, gradients and norms in flight on two streams, each call's
    workspace its own."""
    sets = [inputs(device, case) for case in ((BF16, 8, 2, 128, [1500, 40], None, True, 60),
                                              (F16, 8, 8, 16, [200], [4000], False, None))]
    g = gen(device, 9)
    x, gamma = randn(g, 5000, 257, dtype=F16), randn(g, 257)

    def run(call, dout, stream=None):
        out, lse = bfhip.attention(**call, lse=True, stream=stream)
        c = dict(call)
        back = bfhip.attention_backward(dout, c.pop("q"), c.pop("k"), c.pop("v"), out, lse, **c, stream=stream)
        y, mean, rstd = bfhip.layer_norm(x, gamma, stats=True, stream=stream)
        return out, lse, *back, y, *bfhip.layer_norm_backward(x, x, mean, rstd, gamma, stream=stream)

    want = [run(*s) for s in sets]
    streams = [torch.cuda.Stream() for _ in sets]
    torch.cuda.synchronize()
    for _ in range(4):
        got = [[run(*s, stream=stream) for _ in range(3)] for s, stream in zip(sets, streams)]
        torch.cuda.synchronize()
        for rows, expected in zip(got, want):
            assert all(torch.equal(a, b) for row in rows for a, b in zip(row, expected))
