"""The transformer operators (include/bfhip_transformer.h) where their numbers,
rows or deals come to an edge: biases of any finite size, gradients below a
type's smallest numbers, starts of any value, rows far into a buffer, batches
with empty places."""

import math

import pytest
import torch

import bfhip
import transformer_ref as ref
from test_gpu_transformer import BF16, F16, F32, grads, inputs

pytestmark = pytest.mark.gpu

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
