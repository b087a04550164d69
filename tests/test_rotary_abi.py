"""Rotary positions without a GPU: frequencies, which the host computes, and
refusals, which come before any launch."""

import ctypes as C
import math

import pytest
import torch

import bfhip

P = C.c_void_p(4096)


def frequencies(part, *args, **named):
    return bfhip.rotary_frequencies(part, *args, device="cpu", **named)


@pytest.mark.parametrize("part", [2, 6, 64, 128])
def test_frequencies(part):
    want = torch.tensor([10000.0 ** (-2 * i / part) for i in range(part // 2)], dtype=torch.float64)
    torch.testing.assert_close(frequencies(part), want, rtol=1e-14, atol=0)
    torch.testing.assert_close(frequencies(part, factor=4.0), want / 4, rtol=1e-14, atol=0)


def test_frequencies_by_parts():
    base, factor, length, low, high = 5e5, 8.0, 8192, 1.0, 4.0
    got = frequencies(128, base, factor, length, low, high)
    plain = frequencies(128, base)
    turns = length * plain / (2 * math.pi)
    assert torch.equal(got[turns >= high], plain[turns >= high])
    torch.testing.assert_close(got[turns <= low], plain[turns <= low] / factor, rtol=1e-14, atol=0)
    mid = (turns > low) & (turns < high)
    keep = (turns[mid] - low) / (high - low)
    assert mid.any()
    torch.testing.assert_close(got[mid], plain[mid] * (keep + (1 - keep) / factor), rtol=1e-12, atol=0)


@pytest.mark.parametrize("bad", [dict(part=0), dict(part=3), dict(part=-2), dict(part=4098), dict(base=0.0),
                                 dict(base=float("nan")), dict(factor=0.0), dict(factor=float("inf")), dict(length=-1.0),
                                 dict(low=4.0), dict(high=float("nan"))])
def test_frequencies_refuse(bad):
    with pytest.raises(bfhip.BfHipError, match="frequencies"):
        frequencies(**dict(dict(part=64), **bad))


def row(data=4096, token=256, head=64):
    return bfhip.Rows(data, token, head)


def desc(**change):
    d = dict(type=2, head_dim=64, part=32, interleaved=0, inverse=0, heads=4, heads2=2, amplitude=1.0, tokens=10,
             positions=4096, frequencies=4096)
    d.update(change)
    return bfhip.RotaryDesc(*d.values())


def call(d, x=row(), y=row(8192), x2=row(), y2=row(8192)):
    e = C.create_string_buffer(256)
    ok = bfhip.hip_lib().bfhip_rotary(d, x, y, x2, y2, None, e, 256)
    assert bfhip.hip_lib().bfhip_rotary(d, x, y, x2, y2, None, None, 0) == ok
    return ok, e.value


@pytest.mark.parametrize("bad", [dict(type=3), dict(type=-1), dict(head_dim=0), dict(head_dim=4097), dict(part=0),
                                 dict(part=3), dict(part=66), dict(interleaved=2), dict(inverse=-1), dict(heads=0),
                                 dict(heads=65536), dict(heads2=-1), dict(heads2=65536), dict(amplitude=float("nan")),
                                 dict(amplitude=float("inf")), dict(tokens=-1), dict(tokens=1 << 31)])
def test_rotary_refuses(bad):
    ok, message = call(desc(**bad))
    assert not ok and b"invalid rotary contract" in message


@pytest.mark.parametrize("bad", [None, row(0), row(None), row(8192, -256), row(8192, 256, -64), row(8192, 256, 63),
                                 row(8192, 63), row(8192, 127, 64), row(8192, 64, 639), row(8192, 64, 64)])
def test_rotary_refuses_rows(bad):
    for name in ("y", "y2"):
        ok, message = call(desc(), **{name: bad})
        assert not ok and b"invalid rotary rows" in message, name
    assert b"invalid rotary rows" in call(desc(), x=None)[1]
    assert b"invalid rotary rows" in call(desc(), x=row(4096, -1))[1]


def test_rotary_refuses_in_place_with_other_strides():
    for y in (row(4096, 512), row(4096, 1024, 128)):
        assert b"in place" in call(desc(), x=row(4096), y=y)[1]


def test_rotary_refuses_missing_arrays():
    assert b"invalid" in call(desc(positions=None))[1]
    assert b"invalid" in call(desc(frequencies=None))[1]


def test_rotary_of_no_tokens_is_nothing():
    assert call(desc(tokens=0, positions=None), None, None, None, None)[0]


def test_python_refuses():
    q = torch.zeros((4, 2, 8))
    at, freq = torch.zeros(4, dtype=torch.int32), frequencies(8)
    for args in ((q, q, at, freq), (q.double(), None, at, freq), (q, q[:3], at, freq), (q, q, at.long(), freq),
                 (q, q, at, freq.float()), (q[0], None, at, freq), (q, q.half(), at, freq), (q, q, at[:2], freq)):
        with pytest.raises(bfhip.BfHipError):
            bfhip.rotary(*args)
    with pytest.raises(bfhip.BfHipError):
        bfhip.rotary(q, q, at, freq, out=(q,))
