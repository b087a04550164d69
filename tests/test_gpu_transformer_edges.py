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
from test_gpu_transformer import BF16, F16, F32, grads, inputs

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
