"""The transformer operators' boundary without a GPU: declarations, exports and
refusals (include/bfhip_transformer.h).  Every refusal comes before any launch,
so made-up pointers serve."""

import ctypes as C
import pathlib
import re
import shutil
import subprocess

import pytest
import torch

import bfhip

HEADER = pathlib.Path(__file__).resolve().parent.parent / "include" / "bfhip_transformer.h"
P = C.c_void_p(4096)


def test_declared_exported_and_bound():
    text = re.sub(r"/\*.*?\*/", "", HEADER.read_text(), flags=re.S)
    names = set(re.findall(r"\b(bfhip_[a-z0-9_]+)\s*\(", text))
    assert names == set(bfhip.TRANSFORMER_SIGNATURES)
    lib = bfhip.hip_lib()
    assert all(hasattr(lib, n) for n in names)


def test_header_compiles_as_c(tmp_path):
    if not shutil.which("gcc"):
        pytest.skip("gcc not available")
    src = tmp_path / "t.c"
    src.write_text('#include "bfhip_transformer.h"\n#include <stdio.h>\nint main(void) { printf("%zu %zu",'
                   " sizeof(bfhip_attention_desc), sizeof(bfhip_rows)); return 0; }\n")
    subprocess.run(["gcc", "-std=c11", "-Wall", "-Wextra", "-Werror", f"-I{HEADER.parent}", str(src), "-o",
                    str(tmp_path / "t")], check=True)
    out = subprocess.run([str(tmp_path / "t")], capture_output=True, text=True, check=True).stdout
    assert out == f"{C.sizeof(bfhip.AttentionDesc)} {C.sizeof(bfhip.Rows)}"


def call(name, *args):
    e = C.create_string_buffer(256)
    ok = getattr(bfhip.hip_lib(), name)(*args, None, e, 256)
    assert getattr(bfhip.hip_lib(), name)(*args, None, None, 0) == ok  # no message wanted
    return ok, e.value


def norm(type=0, x=P, xs=96, gamma=P, beta=P, y=P, ys=96, mean=P, rstd=P, rows=10, n=96, eps=1e-5):
    return call("bfhip_layer_norm_forward", type, x, xs, gamma, beta, y, ys, mean, rstd, rows, n, eps)


@pytest.mark.parametrize("bad", [dict(type=3), dict(type=-1), dict(x=None), dict(y=None), dict(mean=None),
                                 dict(rstd=None), dict(rows=-1), dict(n=0), dict(n=65537), dict(eps=-1.0),
                                 dict(eps=float("nan")), dict(ys=95), dict(xs=-1)])
def test_layer_norm_refuses(bad):
    ok, message = norm(**bad)
    assert not ok and b"invalid layer norm" in message


def test_layer_norm_of_no_rows_is_nothing():
    assert norm(rows=0, x=None, y=None)[0]


def norm_back(type=0, dy=P, dys=96, x=P, xs=96, gamma=P, mean=P, rstd=P, dx=P, dxs=96, dgamma=P, dbeta=P, rows=10, n=96,
              work=P, size=1 << 20):
    return call("bfhip_layer_norm_backward", type, dy, dys, x, xs, gamma, mean, rstd, dx, dxs, dgamma, dbeta, rows, n,
                work, size)


@pytest.mark.parametrize("bad", [dict(type=3), dict(dy=None), dict(x=None), dict(dx=None), dict(mean=None),
                                 dict(rstd=None), dict(dgamma=None), dict(dbeta=None), dict(rows=-1), dict(n=0),
                                 dict(dxs=95), dict(dys=-1)])
def test_layer_norm_backward_refuses(bad):
    ok, message = norm_back(**bad)
    assert not ok and b"invalid layer norm" in message


def test_layer_norm_backward_refuses_workspaces():
    size = bfhip.hip_lib().bfhip_layer_norm_backward_workspace
    need = size(1000, 96)
    assert need > 0 and size(-1, 96) == 0 and size(5, 0) == 0
    for bad in (dict(size=need - 1), dict(work=None), dict(work=C.c_void_p(4104))):
        ok, message = norm_back(rows=1000, **bad)
        assert not ok and b"workspace" in message


def bias(name="bfhip_position_bias_forward", table=P, at=P, out=P, count=32, heads=4, n=100, *rest):
    return call(name, table, at, out, count, heads, n, *rest)


@pytest.mark.parametrize("bad", [dict(table=None), dict(at=None), dict(out=None), dict(count=0), dict(heads=0),
                                 dict(n=-1), dict(count=1 << 20, heads=1 << 20), dict(n=1 << 50)])
def test_position_bias_refuses(bad):
    ok, message = bias(**bad)
    assert not ok and b"position bias" in message
    args = dict(table=P, at=P, out=P, count=32, heads=4, n=100)
    args.update(bad)
    ok, message = call("bfhip_position_bias_backward", *args.values(), P, 1 << 40)
    assert not ok and b"position bias" in message


def rows(data=4096, token=128, head=32):
    return bfhip.Rows(data, token, head)


def desc(**change):
    d = dict(type=0, sequences=2, heads=4, kv_heads=2, head_dim=32, causal=1, reach=8, scale=0.2, q_tokens=50,
             k_tokens=60, q_starts=4096, k_starts=4096, bias=4096)
    d.update(change)
    return bfhip.AttentionDesc(*d.values())


def forward(d, q=None, k=None, v=None, out=None, work=P, size=1 << 40):
    r = rows()
    return call("bfhip_attention_forward", d, q or r, k or r, v or r, out or r, P, work, size)


def backward(d, dbias=P, lse=P, work=P, size=1 << 40, **named):
    r = rows()
    t = [named.get(n, r) for n in ("q", "k", "v", "out")]
    g = [named.get(n, r) for n in ("dout", "dq", "dk", "dv")]
    return call("bfhip_attention_backward", d, *t, lse, *g, dbias, work, size)


@pytest.mark.parametrize("bad", [dict(type=3), dict(sequences=-1), dict(heads=0), dict(kv_heads=0), dict(kv_heads=3),
                                 dict(head_dim=0), dict(head_dim=12), dict(head_dim=136), dict(causal=2),
                                 dict(reach=-1), dict(reach=2048), dict(scale=float("nan")), dict(scale=float("inf")),
                                 dict(q_tokens=-1), dict(k_tokens=1 << 31), dict(q_starts=None), dict(k_starts=None)])
def test_attention_refuses(bad):
    d = desc(**bad)
    for f in (forward, backward):
        ok, message = f(d)
        assert not ok and b"invalid attention" in message
    lib = bfhip.hip_lib()
    assert lib.bfhip_attention_forward_workspace(d) == 0 and lib.bfhip_attention_backward_workspace(d) == 0


@pytest.mark.parametrize("bad", [rows(data=4100), rows(data=None), rows(token=130), rows(token=28), rows(head=34),
                                 rows(token=4 << 20), rows(head=-4), rows(token=-128)])
def test_attention_refuses_rows(bad):
    for name in ("q", "k", "v", "out"):
        ok, message = forward(desc(), **{name: bad})
        assert not ok and b"attention rows" in message, name
    for name in ("q", "k", "v", "out", "dout", "dq", "dk", "dv"):
        ok, message = backward(desc(), **{name: bad})
        assert not ok and b"attention rows" in message, name


@pytest.mark.parametrize("bad", [rows(head=0), rows(head=16), rows(token=64), rows(token=36, head=36)])
def test_attention_refuses_results_on_one_another(bad):
    """Rows that overlap are read (broadcast keys), but not written."""
    ok, message = forward(desc(), out=bad)
    assert not ok and b"results on one another" in message
    for name in ("dq", "dk", "dv"):
        ok, message = backward(desc(kv_heads=4), **{name: bad})
        assert not ok and b"results on one another" in message, name
    # Read rows pass that check: the workspace is what is missing here.
    shared = rows(head=0)
    ok, message = backward(desc(), work=None, q=shared, k=shared, v=shared, out=shared, dout=shared)
    assert not ok and b"workspace" in message


def test_attention_refuses_too_many_rows():
    for bad in (dict(q_tokens=0x7fffffff), dict(k_tokens=0x7fffffff)):
        for f in (forward, backward):
            ok, message = f(desc(**bad))
            assert not ok and b"invalid attention" in message


def test_attention_backward_refuses():
    assert b"invalid" in backward(desc(), lse=None)[1]
    assert b"invalid" in backward(desc(bias=None))[1]  # a bias's gradient without one
    need = bfhip.hip_lib().bfhip_attention_backward_workspace(desc())
    assert need > 0
    for bad in (dict(size=need - 1), dict(work=None), dict(work=C.c_void_p(4104))):
        ok, message = backward(desc(), **bad)
        assert not ok and b"workspace" in message


def test_python_refuses():
    """Tensors that the calls do not take: host tensors, types, shapes."""
    x = torch.zeros((4, 8))
    for f in (lambda: bfhip.layer_norm(x), lambda: bfhip.layer_norm(x.double()),
              lambda: bfhip.position_bias(x, torch.zeros(3, dtype=torch.int32)),
              lambda: bfhip.attention(*[torch.zeros((4, 2, 8))] * 3, *[torch.zeros(2, dtype=torch.int32)] * 2)):
        with pytest.raises(bfhip.BfHipError):
            f()
