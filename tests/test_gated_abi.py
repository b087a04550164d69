"""The gated linear's boundary without a GPU: refusals, which come before any
launch, and what its workspaces may take."""

import ctypes as C
import random

import pytest
import torch

import bfhip
from gated_paths import HALF, SINGLE, paths

P = C.c_void_p(4096)


def mat(data=4096, stride=512):
    return bfhip.Matrix(data, stride)


def desc(**change):
    d = dict(type=2, activation=0, rows=10, features=256, hidden=512)
    d.update(change)
    return bfhip.GatedDesc(*d.values())


def call(name, *args):
    e = C.create_string_buffer(256)
    f = getattr(bfhip.hip_lib(), name)
    ok = f(*args, None, e, 256)
    assert f(*args, None, None, 0) == ok
    return ok, e.value


def forward(d, x=mat(), w_gate=mat(), w_up=mat(), h=mat(), gate=mat(), up=mat(), work=P, size=1 << 40):
    return call("bfhip_gated_linear", d, x, w_gate, w_up, h, gate, up, work, size)


def backward(d, dh=mat(), x=mat(), w_gate=mat(), w_up=mat(), gate=mat(), up=mat(), dx=mat(), dw_gate=mat(), dw_up=mat(), work=P,
             size=1 << 50):
    return call("bfhip_gated_linear_backward", d, dh, x, w_gate, w_up, gate, up, dx, dw_gate, dw_up, work, size)


def workspaces(d, x=mat(), w_gate=mat(), w_up=mat()):
    lib = bfhip.hip_lib()
    return [f(d, x, w_gate, w_up) for f in (lib.bfhip_gated_linear_workspace, lib.bfhip_gated_linear_backward_workspace)]


@pytest.mark.parametrize("bad", [dict(type=3), dict(type=-1), dict(activation=3), dict(activation=-1), dict(rows=-1),
                                 dict(rows=0x7fff0001), dict(features=0), dict(features=(1 << 20) + 1), dict(hidden=(1 << 20) + 1), dict(hidden=0), dict(hidden=-1),
                                 dict(rows=1 << 30, features=1 << 11), dict(hidden=1 << 30, features=1 << 11)])
def test_refuses(bad):
    for f in (forward, backward):
        ok, message = f(desc(**bad))
        assert not ok and b"invalid gated linear contract" in message
    assert not any(workspaces(desc(**bad)))


def test_refuses_one_of_two():
    for bad in (dict(gate=None), dict(up=None)):
        assert b"contract" in forward(desc(), **bad)[1]
    for bad in (dict(dw_gate=None), dict(dw_up=None), dict(dx=None, dw_gate=None, dw_up=None)):
        assert b"contract" in backward(desc(), **bad)[1]


@pytest.mark.parametrize("bad", [mat(None), mat(stride=255), mat(stride=-512), mat(stride=1 << 41)])
def test_refuses_matrices(bad):
    for name in ("x", "w_gate", "w_up", "h", "gate", "up"):
        ok, message = forward(desc(), **{name: bad})
        assert not ok and b"invalid gated linear matrices" in message, name
    for name in ("dh", "x", "w_gate", "w_up", "gate", "up", "dx", "dw_gate", "dw_up"):
        ok, message = backward(desc(), **{name: bad})
        assert not ok and b"invalid gated linear matrices" in message, name
    assert b"matrices" in forward(desc(), x=None)[1] and b"matrices" in backward(desc(), x=None)[1]


def test_refuses_weights_of_two_strides():
    for f in (forward, backward):
        assert b"one stride" in f(desc(), w_up=mat(stride=520))[1]


def test_refuses_workspaces():
    wide = {n: mat(stride=4096) for n in ("x", "w_gate", "w_up")}
    d = desc(rows=300, features=4096)
    for f, need in zip((forward, backward), workspaces(d, **wide)):
        assert need > 0
        named = dict(wide, dx=mat(stride=4096), dw_gate=mat(stride=4096), dw_up=mat(stride=4096)) if f is backward else wide
        for bad in (dict(size=need - 1), dict(work=None), dict(work=C.c_void_p(4104))):
            ok, message = f(d, **named, **bad)
            assert not ok and b"workspace" in message


def test_refuses_what_no_launch_holds():
    d = desc(rows=0x7fff0000, features=8, hidden=500)
    x = mat(stride=512)
    assert b"too many" in forward(d, x=x, w_gate=x, w_up=x)[1]
    d = desc(rows=0x7fff0000, features=500, hidden=8)
    for named in (dict(), dict(dw_gate=None, dw_up=None)):
        assert b"too many" in backward(d, **dict(dict.fromkeys(("x", "w_gate", "w_up"), x), **named))[1]


@pytest.mark.parametrize("hidden", [1, 64])
def test_takes_as_many_tiles_as_stated(hidden):
    """Up to 2^23 - 1 tiles of 128 rows in fp32: 2^30 - 128 rows."""
    none = dict(work=None, size=0)
    for rows, message in (((1 << 30) - 128, b"workspace"), (1 << 30, b"too many")):
        d = desc(type=0, rows=rows, features=2, hidden=hidden)
        x = {n: mat(4100, 64) for n in ("x", "w_gate", "w_up")}  # (off 16 bytes: copied, so that there is a workspace)
        assert message in forward(d, **x, **none)[1]
        for left in (dict(), dict(dw_gate=None, dw_up=None)):
            assert message in backward(d, **x, **left, **none)[1]
    d = desc(type=2, rows=0x7fff0000, features=2, hidden=1)
    assert b"workspace" in forward(d, **x, **none)[1] and b"workspace" in backward(d, **x, **none)[1]


def test_nothing_to_do():
    none = mat(None)
    assert forward(desc(rows=0), x=none, h=none, gate=none, up=none, work=None, size=0)[0]
    assert backward(desc(rows=0), dh=none, x=none, gate=none, up=none, dx=none, dw_gate=None, dw_up=None, work=None, size=0)[0]


def test_workspaces_are_bounded():
    rng = random.Random(1)
    log = lambda most: int(most ** rng.random())
    some = 0
    for _ in range(5000):
        d = desc(type=rng.randint(0, 2), rows=log(1 << 20), features=log(1 << 15), hidden=log(1 << 16))
        size, up = (4 if d.type == 0 else 2), lambda n: (n + 7) // 8 * 8
        at, stride = rng.choice(((4096, up(d.features)), (4096, d.features), (4098 if size == 2 else 4100, up(d.features))))
        x = mat(at, stride)
        copied = at % 16 or d.features % (16 // size) or stride % (16 // size)
        copies = (d.rows + 2 * d.hidden) * up(d.features) * size + 1024 if copied else 0
        one, two = workspaces(d, x, x, x)
        assert one <= (256 << 20) + (copies if d.rows > 16 else 0)
        assert two <= (256 << 20) + copies + 2 * (d.rows * up(d.hidden) * size + 256) + 8192
        some += one > 0
    assert some > 300


def test_workspace_holds_copies_where_they_are_needed():
    d = desc(rows=100)
    whole = workspaces(d)
    off = mat(4098, 512)
    for named, bytes_ in ((dict(x=off), 100 * 512), (dict(w_up=off), 2 * 512 * 512), (dict(x=mat(stride=300)), 100 * 512)):
        for a, b in zip(whole, workspaces(d, **named)):
            assert a + bytes_ <= b <= a + bytes_ + 768


def test_python_refuses():
    x, w = torch.zeros((4, 8)), torch.zeros((6, 8))
    for args, named in (((x, w, w), {}), ((x, w, w[:3]), {}), ((x, w.half(), w), {}), ((x[0], w, w), {}),
                        ((x, w, w), dict(activation="tanh")), ((x, w.T.contiguous().T, w), {}), ((x.double(), w, w), {})):
        with pytest.raises(bfhip.BfHipError):
            bfhip.gated_linear(*args, **named)
    with pytest.raises(bfhip.BfHipError):
        bfhip.gated_linear_backward(torch.zeros((4, 5)), x, w, w, torch.zeros((4, 6)), torch.zeros((4, 6)))


def test_python_refuses_no_gradient():
    x, w, rows = torch.zeros((4, 8)), torch.zeros((6, 8)), torch.zeros((4, 6))
    with pytest.raises(bfhip.BfHipError, match="no gradient"):
        bfhip.gated_linear_backward(rows, x, w, w, rows, rows, inputs=False, weights=False)


@pytest.mark.parametrize("dtype,sizes", [(torch.float32, SINGLE), (torch.float16, HALF), (torch.bfloat16, HALF)])
def test_sizes_that_go_by_every_kernel(dtype, sizes):
    """What random sizes go by is what the sizes that are run on the GPU go by: a
    change of the rules that leaves a kernel without a test is found here."""
    covered = set().union(*(paths(dtype, s) for s in sizes))
    kinds = {k for name, (k, *_), *_ in covered if name != "both"}
    assert kinds == {"small", "low", "few"} | (set() if dtype == torch.float32 else {"deep", "large"})
    for kind in kinds - {"few", "small"}:  # every kind in every product that it is for, with and without a split
        for name in ("forward", "inputs") + (("weights",) if kind == "large" else ()):
            found = {p[1][1:] for p in covered if p[0] == name and p[1][0] == kind}
            assert found >= {(True, False), (False, True)} | ({(True, True)} if kind == "large" else set()), (kind, name)
    rng = random.Random(2)
    log = lambda most: int(most ** rng.random())
    tried = 0
    while tried < 6000:
        size = log(20000), log(9000), log(12000)
        if rng.random() < 0.3:
            size = size[0], -(-size[1] // 64) * 64, -(-size[2] // 64) * 64
        if size[0] * size[1] * size[2] <= 1 << 33:
            assert paths(dtype, size) <= covered, size
            tried += 1


def test_plan_refuses():
    lib, plan = bfhip.hip_lib(), (C.c_int * 6)()
    for bad in (dict(hidden=0), dict(type=3)):
        assert not lib.bfhip_gated_linear_plan(desc(**bad), 0, plan, None, 0)
    for product in (-1, 3):
        assert not lib.bfhip_gated_linear_plan(desc(), product, plan, None, 0)
    e = C.create_string_buffer(64)
    assert not lib.bfhip_gated_linear_plan(desc(), 0, None, e, 64) and b"plan" in e.value
