"""What the transformer operators' header says of sizes and alignment
(include/bfhip_transformer.h), asked on the CPU."""

import ctypes as C
import pathlib
import random
import re

import pytest
import torch

import bfhip


def _log(rng, low, high):
    return min(high, int(low * (high / low) ** rng.random() + 0.5))


def descriptors(n, seed):
    """Descriptors over the whole range, and such that are near the plans'
    borders: wide groups, very many sequences, a query fewer than a tile."""
    rng = random.Random(seed)
    for _ in range(n):
        kv_heads = _log(rng, 1, 64)
        heads = kv_heads * _log(rng, 1, 512)
        sequences = _log(rng, 1, 4096)
        q = rng.choice((sequences, sequences * rng.randint(1, 20), _log(rng, 1, 1 << 20), 64 * _log(rng, 1, 100) - 1))
        yield bfhip.AttentionDesc(rng.randint(0, 2), sequences, heads, kv_heads, 8 * rng.randint(1, 16), rng.randint(0, 1),
                                  rng.choice((0, 5, 128, 2047)), 0.1, q, _log(rng, 1, 1 << 24), 4096, 4096,
                                  rng.choice((None, 4096)))


def test_attention_forward_workspace_is_bounded():
    size = bfhip.hip_lib().bfhip_attention_forward_workspace
    sizes = [size(d) for d in descriptors(20000, 1)]
    assert max(sizes) <= 1 << 30 and sorted(sizes)[len(sizes) // 2] == 0
    wide = bfhip.AttentionDesc(2, 512, 128, 1, 128, 1, 0, 0.1, 512, 10 ** 6, 4096, 4096, None)
    assert 0 < size(wide) <= 1 << 30


def test_attention_backward_workspace_is_bounded():
    size = bfhip.hip_lib().bfhip_attention_backward_workspace
    for d in descriptors(20000, 2):
        rows, up = (64 if d.type == 0 else 128), lambda n: (n + 255) // 256 * 256
        terms = (3 if d.bias else 2) * up(4 * d.heads * d.q_tokens)
        part = up(4 * d.heads * (2 * d.reach + 1) * (d.q_tokens // rows + d.sequences)) if d.bias else 0
        most = up(16 * d.heads * (d.q_tokens // rows + d.sequences)) if d.type == 1 else 0
        rest = size(d) - terms - part - most
        assert 0 <= rest <= (128 << 20) + ((32 << 20) if d.type == 0 and not d.bias else 0)


def test_attention_backward_workspace_of_a_tile_and_a_half():
    """Sums of split keys alone: 127 queries are two tiles of 64."""
    size = bfhip.hip_lib().bfhip_attention_backward_workspace
    d = bfhip.AttentionDesc(0, 1, 32, 32, 128, 0, 0, 0.1, 127, 4096, 4096, 4096, None)
    assert 0 < size(d) - 2 * 4 * 32 * 127 <= 32 << 20


def test_no_load_of_rows_through_a_fragment_type():
    """Rows begin on 16 bytes.  A load through a type of a larger alignment would
    be undefined for them, whatever it does on a machine that serves it."""
    csrc = pathlib.Path(__file__).resolve().parent.parent / "bevfusion.c_amd" / "csrc"
    for name in ("attention.h", "attention_forward.hip", "attention_backward.hip"):
        text = re.sub(r"//[^\n]*", "", (csrc / name).read_text())
        assert not re.search(r"_cast<\s*(const\s+)?(typename\s+E::Frag|f32x8)\s*\*", text), name


def test_attention_backward_refuses_what_no_launch_holds():
    """A gradient of more biases than a launch's threads can add up is refused
    before anything is launched."""
    lib = bfhip.hip_lib()

    def call(heads, reach):
        d = bfhip.AttentionDesc(0, 1, heads, heads, 8, 0, reach, 0.1, 1, 1, 4096, 4096, 4096)
        row, error = bfhip.Rows(4096, 8 * heads, 8), C.create_string_buffer(256)
        assert not lib.bfhip_attention_backward(d, row, row, row, row, 4096, row, row, row, row, 4096, 4096, 1 << 50, None,
                                                error, 256)
        return error.value

    assert b"too many" in call(65535, 2047) and b"too many" in call(33000, 2047)


def test_python_refuses_heads_of_no_elements():
    empty, at = torch.zeros((4, 2, 0)), torch.zeros(2, dtype=torch.int32)
    with pytest.raises(bfhip.BfHipError):
        bfhip.attention(empty, empty, empty, at, at)
