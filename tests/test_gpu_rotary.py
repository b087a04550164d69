"""Rotary positions (bfhip_rotary) against their formula in 64 bits."""

import math

import pytest
import torch

import bfhip
import decoder_ref as ref
from transformer_ref import check

pytestmark = pytest.mark.gpu
F32, F16, BF16 = torch.float32, torch.float16, torch.bfloat16


def gen(device, seed=0):
    return torch.Generator(device).manual_seed(seed)


def randn(g, *shape, dtype=F32):
    return torch.randn(shape, generator=g, device=g.device).to(dtype)


def inputs(device, dtype, tokens, heads, kv_heads, dim, part, far=5000, seed=1):
    g = gen(device, seed)
    rows = randn(g, tokens, (heads + kv_heads) * dim, dtype=dtype)
    q, k = rows.split([heads * dim, kv_heads * dim], 1)
    positions = torch.randint(-far // 8, far, (tokens,), generator=g, device=device, dtype=torch.int32)
    return (q.unflatten(1, (heads, dim)), k.unflatten(1, (kv_heads, dim)), positions,
            bfhip.rotary_frequencies(part, device=device))


# (type, tokens, heads, kv_heads, dim, part): chunks of 16 and 8 bytes and of single
# elements, parts of heads, tails that end inside a chunk, one token, long heads.
CASES = [(F32, 1, 1, 1, 2, 2), (BF16, 1, 32, 8, 128, 128), (F16, 37, 5, 1, 80, 40), (F32, 100, 3, 3, 80, 40),
         (BF16, 9, 2, 2, 64, 24), (F16, 33, 4, 2, 66, 6), (F32, 33, 3, 1, 21, 10), (BF16, 4, 1, 1, 4096, 4096),
         (F16, 5000, 2, 1, 32, 32), (F32, 70000, 1, 1, 8, 4), (BF16, 7, 3, 2, 37, 34)]


@pytest.mark.parametrize("interleaved", [False, True])
@pytest.mark.parametrize("case", CASES, ids=str)
def test_rotary_and_gradient(device, case, interleaved):
    q, k, positions, freq = inputs(device, *case)
    call = dict(interleaved=interleaved, amplitude=1.3)
    for name, f, inverse in (("y", bfhip.rotary, False), ("dx", bfhip.rotary_backward, True)):
        got = f(q, k, positions, freq, **call)
        for x, y in zip((q, k), got):
            check(name, y, *ref.rotary(x, positions, freq, inverse=inverse, **call))
            assert torch.equal(y[..., case[5]:], x[..., case[5]:])
        alone = f(q, None, positions, freq, **call)
        assert torch.equal(alone, got[0])


@pytest.mark.parametrize("dtype", [F32, F16, BF16])
@pytest.mark.parametrize("interleaved", [False, True])
def test_rotary_in_place_is_the_same(device, dtype, interleaved):
    q, k, positions, freq = inputs(device, dtype, 65, 4, 2, 48, 32)
    want = bfhip.rotary(q, k, positions, freq, interleaved)
    got = bfhip.rotary(q, k, positions, freq, interleaved, out=(q, k))
    assert got[0] is q and all(torch.equal(a, b) for a, b in zip(got, want))


def test_rotary_one_in_place_one_not(device):
    q, k, positions, freq = inputs(device, BF16, 65, 4, 2, 48, 32)
    want = bfhip.rotary(q, k, positions, freq)
    other = torch.full_like(k, math.nan).contiguous()
    got = bfhip.rotary(q, k, positions, freq, out=(q, other))
    assert torch.equal(got[0], want[0]) and torch.equal(got[1], want[1])


def test_rotary_writes_its_rows_only(device):
    q, k, positions, freq = inputs(device, F16, 50, 3, 2, 40, 20)
    wide = torch.full((50, 7, 43), math.nan, dtype=F16, device=device)
    out = (wide[:, :3, 1:41], wide[:, 4:6, 2:42])
    want = bfhip.rotary(q, k, positions, freq)
    bfhip.rotary(q, k, positions, freq, out=out)
    assert all(torch.equal(a, b) for a, b in zip(out, want))
    for o in out:
        o.fill_(math.nan)
    assert torch.isnan(wide).all()


def test_rotary_heads_outside_tokens(device):
    """[heads, tokens, head_dim] tensors, seen as rows."""
    q, k, positions, freq = inputs(device, BF16, 77, 4, 2, 64, 64)
    want = bfhip.rotary(q, k, positions, freq)
    qh, kh = (t.transpose(0, 1).contiguous().transpose(0, 1) for t in (q, k))
    out = tuple(torch.empty_like(t) for t in (qh, kh))
    assert out[0].stride(0) < out[0].stride(1)
    bfhip.rotary(qh, kh, positions, freq, out=out)
    assert all(torch.equal(a, b) for a, b in zip(out, want))


@pytest.mark.parametrize("far", [2 ** 20, 2 ** 31 - 1])
def test_rotary_far_positions(device, far):
    """Angles of millions and thousands of millions of radians."""
    q, k, positions, freq = inputs(device, F32, 200, 2, 1, 64, 64)
    positions = torch.linspace(-far, far, 200, dtype=torch.float64).to(torch.int64).clamp(-far, far).int().to(device)
    for x, y in zip((q, k), bfhip.rotary(q, k, positions, freq)):
        check("y", y, *ref.rotary(x, positions, freq))


def test_rotary_of_position_zero_and_of_scores(device):
    """Position 0 leaves a row as it is; scores depend on distances alone."""
    q, k, positions, freq = inputs(device, F32, 64, 2, 2, 64, 64)
    zero = torch.zeros_like(positions)
    assert all(torch.equal(a, b) for a, b in zip(bfhip.rotary(q, k, zero, freq), (q, k)))
    at = torch.arange(64, device=device, dtype=torch.int32)
    scores = []
    for shift in (0, 1000):
        a, b = bfhip.rotary(q, k, at + shift, freq)
        scores.append((a.double().movedim(1, 0) @ b.double().permute(1, 2, 0).contiguous()))
    size = (q.double().abs().movedim(1, 0) @ k.double().abs().permute(1, 2, 0).contiguous())
    # each turned row is off by 12 u of the pair's sizes, twice two rows
    assert ((scores[0] - scores[1]).abs() <= 4 * 4 * 12 * 2.0 ** -24 * size + 1e-6).all()


def test_rotary_gradient_by_differences(device):
    """The gradient of sum(w y) with y in fp32, by central differences of the
    linear map: exact but for the roundings of 2 x 2 evaluations."""
    q, _, positions, freq = inputs(device, F32, 12, 2, 1, 16, 12)
    w = randn(gen(device, 9), 12, 2, 16)
    dq = bfhip.rotary_backward(w, None, positions, freq, amplitude=0.7)
    for e in range(16):
        step = torch.zeros_like(q)
        step[..., e] = 1.0
        up, down = (bfhip.rotary(q + sign * step, None, positions, freq, amplitude=0.7).double() for sign in (1, -1))
        slope = (w.double() * (up - down)).sum(2) / 2
        size = (w.double().abs() * (q.double().abs() + 1)).sum(2)
        assert ((slope - dq[..., e].double()).abs() <= 32 * 2.0 ** -24 * size + 1e-6).all()


def test_rotary_keeps_infinities_to_their_pairs(device):
    q, k, positions, freq = inputs(device, F16, 20, 2, 1, 32, 32)
    want = bfhip.rotary(q, k, positions, freq)
    q = q.clone()
    q[3, 1, 5], q[4, 0, 20] = math.inf, math.nan
    got = bfhip.rotary(q, k, positions, freq)
    bad = torch.zeros_like(q, dtype=torch.bool)
    bad[3, 1, [5, 21]] = True
    bad[4, 0, [4, 20]] = True
    assert torch.equal(got[0][~bad], want[0][~bad]) and not torch.isfinite(got[0][bad]).any()
    assert torch.equal(got[1], want[1])


def test_rotary_in_a_graph_and_on_a_stream(device):
    q, k, positions, freq = inputs(device, BF16, 300, 4, 2, 64, 64)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    want = bfhip.rotary(q, k, positions, freq)
    got = bfhip.rotary(q, k, positions, freq, stream=side)
    side.synchronize()
    assert all(torch.equal(a, b) for a, b in zip(got, want))
    out = tuple(torch.empty_like(t) for t in want)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        bfhip.rotary(q, k, positions, freq, out=out)
    for shift in (0, 7, 100):
        positions += shift
        for o in out:
            o.zero_()
        graph.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(out, bfhip.rotary(q, k, positions, freq)))


@pytest.mark.parametrize("tokens", [1, 5])
def test_rotary_of_broadcast_rows(device, tokens):
    """Rows that share memory, and strides that are of no account."""
    q, _, positions, freq = inputs(device, BF16, tokens, 4, 2, 64, 64)
    for x in (q[:, :1].expand(-1, 4, -1), q[:1].expand(tokens, -1, -1), q[:1, :1].expand(tokens, 3, -1), q[:, :1],
              q.as_strided((tokens, 1, 64), (q.stride(0), 0, 1)), q[:1].as_strided((1, 4, 64), (0, 64, 1))):
        at = positions[:x.shape[0]]
        want = bfhip.rotary(x.contiguous(), None, at, freq)
        assert torch.equal(bfhip.rotary(x, None, at, freq), want)
        for got in bfhip.rotary(x, x, at, freq):
            assert torch.equal(got, want)
