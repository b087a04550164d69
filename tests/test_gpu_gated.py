"""The gated linear (bfhip_gated_linear) and its gradients against 64-bit
formulas."""

import math

import pytest
import torch

import bfhip
import decoder_ref as ref
from gated_paths import HALF, SINGLE
from transformer_ref import check

pytestmark = pytest.mark.gpu
F32, F16, BF16 = torch.float32, torch.float16, torch.bfloat16


def gen(device, seed=0):
    return torch.Generator(device).manual_seed(seed)


def randn(g, *shape, dtype=F32, scale=1.0):
    return (torch.randn(shape, generator=g, device=g.device) * scale).to(dtype)


def inputs(device, dtype, rows, features, hidden, seed=1):
    g = gen(device, seed)
    return dict(x=randn(g, rows, features, dtype=dtype),
                w_gate=randn(g, hidden, features, dtype=dtype, scale=1.5 * features ** -0.5),
                w_up=randn(g, hidden, features, dtype=dtype, scale=features ** -0.5)), randn(g, rows, hidden, dtype=dtype)


def run(call, dh, activation):
    h, gate, up = bfhip.gated_linear(**call, activation=activation, save=True)
    return dict(h=h, gate=gate, up=up), dict(zip(("dx", "dw_gate", "dw_up"),
                                                 bfhip.gated_linear_backward(dh, **call, gate=gate, up=up, activation=activation)))


def check_finite(name, got, value, bound):
    """Within the bound where the type holds the value, infinite beyond."""
    most = torch.finfo(got.dtype).max
    held = value.abs() + bound <= most
    check(name, got[held], value[held], bound[held])
    # (what rounds to the type's next number past its largest is infinite)
    over = value.abs() - bound > most * (1 + torch.finfo(got.dtype).eps)
    assert torch.equal(got[over].double(), value[over].sign() * math.inf), name


def compare(call, dh, activation):
    forward, back = run(call, dh, activation)
    for name, (value, bound) in ref.gated_linear(**call, activation=activation).items():
        check_finite(name, forward[name], value, bound)
    assert torch.equal(bfhip.gated_linear(**call, activation=activation), forward["h"])
    want = ref.gated_linear_backward(dh, **call, gate=forward["gate"], up=forward["up"], activation=activation)
    for name, (value, bound) in want.items():
        check_finite(name, back[name], value, bound)
    return forward, back


# (rows, features, hidden): one of each, sizes that no chunk, tile or step divides,
# fewer and more rows than tiles of each size, long and short contractions.
SIZES = [(1, 1, 1), (3, 5, 2), (1, 512, 300), (16, 1024, 128), (17, 64, 129), (65, 96, 40), (100, 771, 257), (130, 128, 500),
         (257, 264, 136), (5, 4096, 64), (1000, 40, 24), (2100, 33, 65), (600, 1000, 2056)]


@pytest.mark.parametrize("size", SIZES, ids=str)
@pytest.mark.parametrize("dtype", [F32, F16, BF16])
def test_gated_linear(device, dtype, size):
    compare(*inputs(device, dtype, *size), "silu")


@pytest.mark.parametrize("dtype", [F32, F16, BF16])
@pytest.mark.parametrize("rows", [2, 16, 17, 31, 32, 33])
def test_few_rows(device, dtype, rows):
    """Features that leave waves without a step, with one, with many and a rest;
    hidden elements that end inside a block."""
    for features, hidden in ((63, 33), (64, 16), (500, 40), (4096, 100), (3003, 4100)):
        call, dh = inputs(device, dtype, rows, features, hidden)
        forward = dict(zip(("h", "gate", "up"), bfhip.gated_linear(**call, activation="gelu", save=True)))
        for name, (value, bound) in ref.gated_linear(**call, activation="gelu").items():
            check(name, forward[name], value, bound)
    call, dh = inputs(device, dtype, rows, 2816, 4480)  # (weights of more than 48 MiB)
    check("h", bfhip.gated_linear(**call), *ref.gated_linear(**call, activation="silu")["h"])


@pytest.mark.parametrize("activation", ["silu", "gelu", "relu"])
@pytest.mark.parametrize("dtype", [F32, F16, BF16])
def test_activations(device, dtype, activation):
    """Over their whole range: products from -30 to 30, and far ones."""
    call, dh = inputs(device, dtype, 200, 64, 128)
    call["x"] *= 5
    call["x"][::7] *= 0.01
    call["x"][5] *= 40
    compare(call, dh, activation)


@pytest.mark.parametrize("dtype", [F16, BF16])
@pytest.mark.parametrize("size", [(1, 300, 70), (1, 4096, 1000), (7, 64, 2300), (16, 520, 1024), (70, 40, 234), (16384, 24, 1)], ids=str)
def test_few_slopes(device, dtype, size):
    """Up to 16384 slopes reach the gradients with twice the type's precision."""
    rows, features, hidden = size
    assert rows * hidden <= 1 << 14
    call, dh = inputs(device, dtype, rows, features, hidden)
    call["x"][:, 0] = 0  # (a column whose gradients are zeros)
    forward, back = run(call, dh, "gelu")
    want = ref.gated_linear_backward(dh, **call, gate=forward["gate"], up=forward["up"], activation="gelu", left=True)
    for name, (value, bound) in want.items():
        check_finite(name, back[name], value, bound)
    assert not back["dw_gate"][:, 0].any()


@pytest.mark.parametrize("dtype", [F16, BF16])
def test_few_slopes_that_are_infinite(device, dtype):
    """What the rounding of an infinite slope left is nothing, not NaN."""
    call, dh = inputs(device, dtype, 4, 64, 96)
    h, gate, up = bfhip.gated_linear(**call, save=True)
    gate[1], up[1, 5], call["x"][1] = 40.0, math.inf, 1.0
    dh[1] = 1.0
    dx, dw_gate, dw_up = bfhip.gated_linear_backward(dh, **call, gate=gate, up=up)
    rest = torch.arange(96, device=device) != 5
    assert (dw_gate[5] == math.inf).all() and dw_gate[rest].isfinite().all() and dw_up.isfinite().all()
    assert (dx[1].abs() == math.inf).all() and dx[[0, 2, 3]].isfinite().all()


@pytest.mark.parametrize("dtype", [F16, BF16])
def test_large_tiles(device, dtype):
    """Results of more tiles than CUs, whole and ragged."""
    compare(*inputs(device, dtype, 4096, 256, 2048), "silu")
    compare(*inputs(device, dtype, 4100, 520, 2056), "gelu")
    compare(*inputs(device, dtype, 3001, 515, 2051), "relu")


@pytest.mark.parametrize("dtype", [F16, BF16])
def test_large_tiles_of_every_product(device, dtype):
    """All three products by large tiles whose last ones have few rows, few
    columns and few terms, in matrices with NaN behind every row and the last."""
    sizes = dict(x=(4100, 2808), w_gate=(2810, 2808), w_up=(2810, 2808))
    call, dh = inputs(device, dtype, 4100, 2808, 2810)
    wide = {n: torch.full((rows + 256, length + 64), math.nan, dtype=dtype, device=device) for n, (rows, length) in sizes.items()}
    views = {n: wide[n][:rows, :length].copy_(call[n]) for n, (rows, length) in sizes.items()}
    compare(views, dh, "silu")
    compare(*inputs(device, dtype, 4100, 2805, 2810), "relu")


def test_rows_past_4_gib(device):
    """Rows of zeros but for the first and last ones; results of rows in the
    middle are zeros."""
    rows, features, hidden = 600_000, 4096, 128
    call, dh = inputs(device, BF16, 400, features, hidden)
    ends = torch.cat([torch.arange(200), torch.arange(rows - 200, rows)]).to(device)
    x, dy = (torch.zeros((rows, t.shape[1]), dtype=BF16, device=device) for t in (call["x"], dh))
    x[ends], dy[ends] = call["x"], dh
    far = dict(call, x=x)
    forward, back = run(far, dy, "silu")
    for name, (value, bound) in ref.gated_linear(**call, activation="silu").items():
        check(name, forward[name][ends], value, bound)
        assert not forward[name][200:-200].any()
    want = ref.gated_linear_backward(dh, **call, gate=forward["gate"][ends], up=forward["up"][ends], activation="silu")
    check("dx", back["dx"][ends], *want["dx"])
    assert not back["dx"][200:-200].any()
    for name in ("dw_gate", "dw_up"):  # (a sum of more terms, all but 400 of them zero)
        check(name, back[name], *want[name])


def test_large_tiles_f32(device):
    compare(*inputs(device, F32, 2050, 260, 1100), "gelu")


@pytest.mark.parametrize("dtype", [F32, F16, BF16])
def test_rows_of_any_alignment(device, dtype):
    """Views into wider tensors, on and off 16 bytes; the weights' views of one."""
    call, dh = inputs(device, dtype, 70, 72, 136)
    want, grads = run(call, dh, "silu")

    def inside(t, left, right):
        wide = torch.full((t.shape[0], t.shape[1] + left + right), math.nan, dtype=dtype, device=device)
        view = wide[:, left:left + t.shape[1]]
        view.copy_(t)
        return view
    for left, right in ((8, 8), (1, 2), (0, 3)):
        moved = {n: inside(t, left, right) for n, t in call.items()}
        got, back = run(moved, inside(dh, left, right), "silu")
        for a, b in ((want, got), (grads, back)):
            for n in a:
                assert torch.equal(a[n], b[n]), (n, left)
    both = torch.stack([call["w_gate"], call["w_up"]], 1)
    got, back = run(dict(call, w_gate=both[:, 0], w_up=both[:, 1]), dh, "silu")
    assert torch.equal(got["h"], want["h"]) and torch.equal(back["dx"], grads["dx"])


def test_results_only_where_they_belong(device):
    for dtype in (F32, F16, BF16):
        call, _ = inputs(device, dtype, 70, 72, 133)
        wide = torch.full((74, 150), math.nan, dtype=dtype, device=device)
        out = wide[2:72, 3:136]
        want = bfhip.gated_linear(**call)
        bfhip.gated_linear(**call, out=out)
        assert torch.equal(out, want)
        out.fill_(math.nan)
        assert torch.isnan(wide).all()


@pytest.mark.parametrize("dtype", [F32, F16, BF16])
def test_rows_do_not_depend_on_others(device, dtype):
    """Infinities and NaN in one row of x stay in that row."""
    call, dh = inputs(device, dtype, 150, 200, 72)
    want, _ = run(call, dh, "silu")
    for value in (math.inf, math.nan):
        x = call["x"].clone()
        x[33, 7] = value
        h = bfhip.gated_linear(x, call["w_gate"], call["w_up"])
        keep = torch.arange(150, device=device) != 33
        assert torch.equal(h[keep], want["h"][keep]) and not torch.isfinite(h[33]).all()


@pytest.mark.parametrize("size", [(128, 4096, 1100), (999, 771, 2055), (5, 64, 300), (2100, 33, 65), (4100, 2808, 2810)], ids=str)
@pytest.mark.parametrize("dtype", [F32, F16, BF16])
def test_one_gradient(device, dtype, size):
    """The inputs' gradient alone or the weights' alone: the same bits, nothing else
    written, in a workspace of the stated size."""
    call, dh = inputs(device, dtype, *size)
    h, gate, up = bfhip.gated_linear(**call, save=True)
    want = bfhip.gated_linear_backward(dh, **call, gate=gate, up=up)
    lib, error = bfhip.hip_lib(), bfhip._err()
    matrix = lambda t: bfhip.Matrix(t.data_ptr(), t.stride(0))
    desc = bfhip.GatedDesc(bfhip._type_code(dh), 0, *size)
    given = [matrix(call[n]) for n in ("x", "w_gate", "w_up")]
    bytes_ = lib.bfhip_gated_linear_backward_workspace(desc, *given)
    for wanted in ((True, False, False), (False, True, True), (True, True, True)):
        got = [torch.full_like(t, 7) if w else None for t, w in zip(want, wanted)]
        work = torch.full((bytes_ + 256,), 0xa5, dtype=torch.uint8, device=device)
        ok = lib.bfhip_gated_linear_backward(desc, matrix(dh), *given, matrix(gate), matrix(up),
                                             *(t if t is None else matrix(t) for t in got), work.data_ptr(), bytes_,
                                             torch.cuda.current_stream().cuda_stream, error, 512)
        assert ok, error.value
        assert (work[bytes_:] == 0xa5).all()
        for t, g in zip(want, got):
            assert g is None or torch.equal(g, t)


@pytest.mark.parametrize("dtype", [F32, F16, BF16])
def test_no_rows(device, dtype):
    call, dh = inputs(device, dtype, 0, 24, 40)
    forward, back = run(call, dh, "silu")
    assert forward["h"].shape == (0, 40) and back["dx"].shape == (0, 24)
    assert (back["dw_gate"] == 0).all() and (back["dw_up"] == 0).all()


@pytest.mark.parametrize("size", [2.0 ** -20, 2.0 ** -11, 1.0, 2.0 ** 9])
def test_fp16_gradients_of_any_size(device, size):
    """Of a loss that is a mean, and of one that is scaled up: dg of 2^-40 and of
    2^20 in fp16."""
    call, dh = inputs(device, F16, 300, 128, 264)
    dh = (dh * size).to(F16)
    call["w_up"] *= 16 if size > 1 else 2 ** -6 if size < 2.0 ** -19 else 1
    call["w_gate"] *= 2 ** -4 if size > 1 else 1
    h, gate, up = bfhip.gated_linear(**call, save=True)
    back = bfhip.gated_linear_backward(dh, **call, gate=gate, up=up)
    want = ref.gated_linear_backward(dh, **call, gate=gate, up=up, activation="silu")
    for got, name in zip(back, ("dx", "dw_gate", "dw_up")):
        check_finite(name, got, *want[name])


def test_fp16_gradients_that_are_zero_or_infinite(device):
    call, dh = inputs(device, F16, 64, 64, 64)
    h, gate, up = bfhip.gated_linear(**call, save=True)
    for t in bfhip.gated_linear_backward(torch.zeros_like(dh), **call, gate=gate, up=up):
        assert (t == 0).all()
    want = bfhip.gated_linear_backward(dh, **call, gate=gate, up=up)
    dh[5, 6] = math.inf  # reaches row 5 of dx and row 6 of the weights' gradients alone
    got = bfhip.gated_linear_backward(dh, **call, gate=gate, up=up)
    rows = torch.arange(64, device=device)
    assert torch.equal(got[0][rows != 5], want[0][rows != 5]) and not torch.isfinite(got[0][5]).any()
    for a, b in zip(got[1:], want[1:]):
        assert torch.equal(a[rows != 6], b[rows != 6])


@pytest.mark.parametrize("activation", ["silu", "gelu"])
def test_gradients_by_differences(device, activation):
    """sum(dh h) in fp32, by central differences of steps of 2^-6: off by the
    third derivative's share (2^-12 / 6 of it, at most 2 of each slope here) and by
    the roundings of h, 2^-24 sqrt(terms) over the step."""
    call, dh = inputs(device, F32, 20, 24, 32)
    h, gate, up = bfhip.gated_linear(**call, activation=activation, save=True)
    grads = bfhip.gated_linear_backward(dh, **call, gate=gate, up=up, activation=activation)
    step = 2.0 ** -6
    for name, grad in zip(("x", "w_gate", "w_up"), grads):
        for seed in range(3):
            way = randn(gen(device, seed), *call[name].shape)
            way /= way.norm()
            at = lambda s: (bfhip.gated_linear(**dict(call, **{name: call[name] + s * way}), activation=activation).double()
                            * dh.double()).sum()
            slope, want = (at(step) - at(-step)) / (2 * step), (grad.double() * way.double()).sum()
            assert abs(slope - want) <= 2e-3 * grad.double().norm(), (name, slope, want)


def test_equal_calls_give_equal_bits(device):
    for dtype, size in ((BF16, (300, 512, 256)), (F16, (40, 4096, 128)), (F32, (300, 200, 128))):
        call, dh = inputs(device, dtype, *size)
        first = run(call, dh, "gelu")
        for _ in range(3):
            again = run(call, dh, "gelu")
            for a, b in zip(first, again):
                assert all(torch.equal(a[n], b[n]) for n in a)


def test_in_a_graph(device):
    """Forward and backward captured, replayed on other inputs, with eager work
    in between."""
    for dtype, size in ((F16, (64, 2048, 128)), (BF16, (500, 136, 264)), (F32, (3, 512, 64))):
        call, dh = inputs(device, dtype, *size)
        side = torch.cuda.Stream()
        with torch.cuda.stream(side):
            run(call, dh, "silu")
        side.synchronize()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            results = run(call, dh, "silu")
        for seed in (5, 6, 7):
            other, odh = inputs(device, dtype, *size, seed=seed)
            for n in call:
                call[n].copy_(other[n])
            dh.copy_(odh * 2.0 ** -seed)
            graph.replay()
            torch.cuda.synchronize()
            for a, b in zip(results, run(call, dh, "silu")):
                assert all(torch.equal(a[n], b[n]) for n in a)


def test_calls_on_two_streams(device):
    calls = [inputs(device, F16, 200, 1024, 256, seed=s) for s in (1, 2)]
    want = [run(*c, "silu") for c in calls]
    streams = [torch.cuda.Stream() for _ in calls]
    torch.cuda.synchronize()
    for _ in range(5):
        got = []
        for (call, dh), s in zip(calls, streams):
            h, gate, up = bfhip.gated_linear(**call, save=True, stream=s)
            got.append((h, bfhip.gated_linear_backward(dh, **call, gate=gate, up=up, stream=s)))
    torch.cuda.synchronize()
    for (h, back), (f, b) in zip(got, want):
        assert torch.equal(h, f["h"]) and all(torch.equal(x, b[n]) for x, n in zip(back, b))


def test_a_block(device):
    """A feed-forward block with the norm before it, both directions, as a
    program trains it: norm, gated linear, and a plain linear behind them."""
    g = gen(device, 3)
    x, gamma = randn(g, 90, 64), 1 + randn(g, 64, scale=0.1)
    wg, wu, wd = (randn(g, *s, scale=0.2) for s in ((160, 64), (160, 64), (64, 160)))
    dy = randn(g, 90, 64)
    y, mean, rstd = bfhip.layer_norm(x, gamma, stats=True)
    h, gate, up = bfhip.gated_linear(y, wg, wu, save=True)
    dh = dy @ wd
    d_in, dwg, dwu = bfhip.gated_linear_backward(dh, y, wg, wu, gate, up)
    dx, dgamma, _ = bfhip.layer_norm_backward(d_in, x, mean, rstd, gamma)
    leaves = [t.double().cpu().requires_grad_() for t in (x, gamma, wg, wu)]
    X, G, A, B = leaves
    n = torch.nn.functional.layer_norm(X, (64,), G)
    p = n @ A.T
    loss = ((p * torch.sigmoid(p)) * (n @ B.T) @ wd.double().cpu().T * dy.double().cpu()).sum()
    loss.backward()
    for name, got, leaf in zip(("dx", "dgamma", "dwg", "dwu"), (dx, dgamma, dwg, dwu), leaves):
        # sums of at most 160 x 64 x 90 fp32 roundings of random sign: 2^-24 * 1000
        scale = leaf.grad.abs().max()
        assert (got.double().cpu() - leaf.grad).abs().max() <= 6e-5 * scale, name


@pytest.mark.parametrize("rows", [1, 40])
def test_strides_of_no_account(device, rows):
    """One row of any stride, one feature of any, weights that are views of one."""
    call, dh = inputs(device, BF16, rows, 1, 96)
    want, grads = run(call, dh, "silu")
    wide = {n: t.repeat_interleave(3, 1)[:, ::3] for n, t in call.items()}
    if rows == 1:
        wide["x"] = wide["x"].as_strided((1, 1), (0, 5))
    got, back = run(wide, dh, "silu")
    for a, b in ((want, got), (grads, back)):
        assert all(torch.equal(a[n], b[n]) for n in a)
    call, dh = inputs(device, BF16, rows, 72, 96)
    want, grads = run(call, dh, "silu")
    fused = torch.cat([call["w_gate"], call["w_up"]], 1)
    views = dict(x=call["x"], w_gate=fused[:, :72], w_up=fused[:, 72:])
    if rows == 1:
        views["x"] = call["x"].as_strided((1, 72), (0, 1))
    got, back = run(views, dh, "silu")
    for a, b in ((want, got), (grads, back)):
        assert all(torch.equal(a[n], b[n]) for n in a)


@pytest.mark.parametrize("dtype", [F32, F16, BF16])
def test_infinite_weight_of_a_single_hidden_element(device, dtype):
    """dx = dg Wg + du Wu has one term each: an infinite weight makes its feature's
    gradients infinite, with the slope's sign, and no others."""
    rows, features = 65536, 4096
    g = gen(device, 4)
    x = torch.ones((rows, features), dtype=dtype, device=device)
    w_gate, w_up = (randn(g, 1, features, dtype=dtype) for _ in range(2))
    w_gate[0, 7], w_gate[0, 3000] = math.inf, -math.inf
    gate, up = torch.ones((rows, 1), device=device), torch.full((rows, 1), 0.5, device=device)
    dh = torch.where(randn(g, rows, 1) > 0, 1.0, -1.0).to(dtype)
    dx, _, _ = bfhip.gated_linear_backward(dh, x, w_gate, w_up, gate, up)
    assert torch.equal(dx[:, 7:8], dh * math.inf) and torch.equal(dx[:, 3000:3001], -dh * math.inf)
    rest = torch.ones(features, dtype=torch.bool, device=device)
    rest[[7, 3000]] = False
    assert dx[:, rest].isfinite().all()


@pytest.mark.parametrize("dtype", [F32, F16, BF16])
@pytest.mark.parametrize("size", [(7, 72, 300), (130, 520, 100), (1, 4096, 1000)], ids=str)
def test_infinite_operands_of_few_slopes(device, dtype, size):
    """An infinite weight makes its feature's gradients infinite, an infinite x its
    column's, with the slopes' signs; others are within the bound of slopes that
    are rounded once."""
    rows, features, hidden = size
    assert rows * hidden <= 1 << 14
    call, dh = inputs(device, dtype, *size)
    g = gen(device, 9)
    gate, up = 0.5 + torch.rand((rows, hidden), generator=g, device=device), 0.5 + torch.rand((rows, hidden), generator=g, device=device)
    dh = torch.where(dh > 0, dh + 0.5, dh - 0.5).to(dtype)
    want = {n: v.clone() for n, (v, _) in ref.gated_linear_backward(dh, **call, gate=gate, up=up, activation="silu").items()}
    for w, h, f, value in (("w_gate", 3, 9, math.inf), ("w_up", hidden - 1, 70, -math.inf)):
        call[w][h, f] = value
        want["dx"][:, f] = dh[:, h].double().sign() * value
    call["x"][rows - 1, 5] = -math.inf
    want["dw_gate"][:, 5] = want["dw_up"][:, 5] = -dh[rows - 1].double().sign() * math.inf
    finite = {n: t.nan_to_num(0, 0, 0) for n, t in call.items()}
    bounds = ref.gated_linear_backward(dh, **finite, gate=gate, up=up, activation="silu")
    got = bfhip.gated_linear_backward(dh, **call, gate=gate, up=up)
    for t, name in zip(got, ("dx", "dw_gate", "dw_up")):
        far = want[name].isinf()
        assert far.any() and torch.equal(t[far].double(), want[name][far]), name
        check(name, t[~far], bounds[name][0][~far], bounds[name][1][~far])


@pytest.mark.parametrize("dtype", [F32, F16, BF16])
@pytest.mark.parametrize("size", [(0, 24, 40), (3, 64, 100), (300, 72, 136), (999, 771, 2055)], ids=str)
def test_gradients_that_are_not_wanted(device, dtype, size):
    """Are None, and the others have the bits that they have beside them."""
    call, dh = inputs(device, dtype, *size)
    h, gate, up = bfhip.gated_linear(**call, save=True)
    call.update(gate=gate, up=up)
    want = bfhip.gated_linear_backward(dh, **call)
    dx, *none = bfhip.gated_linear_backward(dh, **call, weights=False)
    assert none == [None, None] and torch.equal(dx, want[0])
    none, *dw = bfhip.gated_linear_backward(dh, **call, inputs=False)
    assert none is None and torch.equal(dw[0], want[1]) and torch.equal(dw[1], want[2])


@pytest.mark.parametrize("dtype,size", [(t, s) for t, sizes in ((F32, SINGLE), (F16, HALF), (BF16, HALF)) for s in sizes], ids=str)
def test_every_kernel(device, dtype, size):
    """Sizes that go by every kind of tiles in every product, whole, split and in
    part, and each gradient by itself."""
    activation = ("silu", "gelu", "relu")[sum(size) % 3]
    call, dh = inputs(device, dtype, *size)
    forward, back = compare(call, dh, activation)
    call.update(gate=forward["gate"], up=forward["up"], activation=activation)
    dx, *_ = bfhip.gated_linear_backward(dh, **call, weights=False)
    _, dw_gate, dw_up = bfhip.gated_linear_backward(dh, **call, inputs=False)
    assert torch.equal(dx, back["dx"]) and torch.equal(dw_gate, back["dw_gate"]) and torch.equal(dw_up, back["dw_up"])
