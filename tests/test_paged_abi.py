"""The paged cache's boundary without a GPU: refusals, which come before any
launch, and what its workspace may take."""

import ctypes as C
import random

import pytest
import torch

import bfhip

P = C.c_void_p(4096)


def row(data=4096, token=256, head=64):
    return bfhip.Rows(data, token, head)


def pool(data=4096, page=16 * 128, token=128, head=64):
    return bfhip.Pages(data, page, token, head)


def desc(**change):
    d = dict(type=2, sequences=3, heads=4, kv_heads=2, head_dim=64, page_size=16, table_pages=50, reach=8, scale=0.2,
             tokens=5, pages=100, table_stride=50, starts=4096, lengths=4096, table=4096, bias=4096)
    d.update(change)
    return bfhip.PagedDesc(*d.values())


def call(name, *args):
    e = C.create_string_buffer(256)
    f = getattr(bfhip.hip_lib(), name)
    ok = f(*args, None, e, 256)
    assert f(*args, None, None, 0) == ok
    return ok, e.value


def append(d, k=row(), v=row(), kp=pool(), vp=pool()):
    return call("bfhip_cache_append", d, k, v, kp, vp)


def attend(d, q=row(), kp=pool(), vp=pool(), out=row(), work=P, size=1 << 40):
    return call("bfhip_paged_attention", d, q, kp, vp, out, P, work, size)


@pytest.mark.parametrize("bad", [dict(type=3), dict(sequences=-1), dict(kv_heads=0), dict(kv_heads=65536), dict(head_dim=0),
                                 dict(head_dim=12), dict(head_dim=136), dict(page_size=0), dict(table_pages=-1),
                                 dict(page_size=1 << 20, table_pages=1 << 12), dict(tokens=-1), dict(tokens=1 << 31),
                                 dict(pages=-1), dict(pages=1 << 31), dict(table_stride=49), dict(table_stride=-1),
                                 dict(starts=None), dict(lengths=None), dict(table=None)])
def test_paged_refuses(bad):
    for f in (append, attend):
        ok, message = f(desc(**bad))
        assert not ok and b"invalid paged" in message
    assert bfhip.hip_lib().bfhip_paged_attention_workspace(desc(**bad)) == 0


@pytest.mark.parametrize("bad", [dict(heads=0), dict(heads=3), dict(heads=65536), dict(scale=float("nan")),
                                 dict(scale=float("inf")), dict(reach=-1), dict(reach=2048)])
def test_paged_attention_refuses(bad):
    ok, message = attend(desc(**bad))
    assert not ok and b"invalid paged attention" in message
    assert bfhip.hip_lib().bfhip_paged_attention_workspace(desc(**bad)) == 0


@pytest.mark.parametrize("bad", [None, pool(None), pool(4100), pool(page=2044), pool(token=130), pool(head=60), pool(page=-2048),
                                 pool(token=-128), pool(head=-64)])
def test_paged_refuses_pages(bad):
    for f in (append, attend):
        for name in ("kp", "vp"):
            ok, message = f(desc(), **{name: bad})
            assert not ok and b"cache pages" in message, name


@pytest.mark.parametrize("bad", [pool(head=0), pool(token=64), pool(page=1024), pool(page=64, token=6400, head=6400)])
def test_append_refuses_pages_on_one_another(bad):
    for name in ("kp", "vp"):
        ok, message = append(desc(), **{name: bad})
        assert not ok and b"on one another" in message
    # they may be read
    assert b"workspace" in attend(desc(), kp=bad, vp=bad, work=None)[1]


def test_append_takes_pages_in_any_order_of_strides():
    for good in (pool(page=64, token=6400, head=16 * 6400), pool(page=64, token=12800, head=6400)):
        assert append(desc(tokens=0), kp=good, vp=good)[0]


@pytest.mark.parametrize("bad", [None, row(None), row(token=-1), row(head=-64)])
def test_append_refuses_rows(bad):
    for name in ("k", "v"):
        ok, message = append(desc(), **{name: bad})
        assert not ok and b"cache rows" in message


@pytest.mark.parametrize("bad", [row(4100), row(None), row(token=258), row(token=56), row(head=34), row(token=4 << 20)])
def test_paged_attention_refuses_rows(bad):
    for name in ("q", "out"):
        ok, message = attend(desc(), **{name: bad})
        assert not ok and b"attention rows" in message
    assert b"on one another" in attend(desc(), out=row(head=0))[1]


def test_paged_attention_refuses_workspaces():
    need = bfhip.hip_lib().bfhip_paged_attention_workspace(desc())
    assert need > 0
    for bad in (dict(size=need - 1), dict(work=None), dict(work=C.c_void_p(4104))):
        ok, message = attend(desc(), **bad)
        assert not ok and b"workspace" in message


def test_paged_attention_refuses_what_no_launch_holds():
    assert b"too many" in attend(desc(tokens=0x7ffff000, heads=64, kv_heads=1), out=row(token=4096))[1]


@pytest.mark.parametrize("heads,kv_heads,most", [(32, 32, 0x7ffff000), (32, 8, 1 << 28), (3, 1, (1 << 30) // 3)])
def test_paged_attention_takes_as_many_rows_as_stated(heads, kv_heads, most):
    """tokens * heads / kv_heads up to 2^30 (and tokens as in any call), whatever
    the heads' number and size are."""
    most = min(most, (1 << 30) * kv_heads // heads)
    for dim in (8, 128):
        wide = row(token=heads * dim, head=dim)
        good, more = (desc(tokens=n, heads=heads, kv_heads=kv_heads, head_dim=dim) for n in (most, most + 1))
        assert b"workspace" in attend(good, q=wide, out=wide, work=None)[1]
        assert b"too many" in attend(more, q=wide, out=wide, work=None)[1]


def test_paged_nothing_to_do():
    for change in (dict(tokens=0), dict(sequences=0)):
        assert append(desc(**change))[0] and attend(desc(**change))[0]


def test_paged_workspace_is_bounded():
    rng, size, some = random.Random(1), bfhip.hip_lib().bfhip_paged_attention_workspace, 0
    for _ in range(20000):
        kv = int(64 ** rng.random())
        n = int(4096 ** rng.random())
        pages = int(1 << rng.randint(0, 14))
        d = desc(type=rng.randint(0, 2), sequences=n, kv_heads=kv, heads=kv * int(512 ** rng.random()),
                 head_dim=8 * rng.randint(1, 16), page_size=int(512 ** rng.random()), table_pages=pages, table_stride=pages,
                 tokens=rng.choice((n, 3 * n, int((1 << 20) ** rng.random()))))
        need = size(d)
        assert need <= (16 << 20) + 8 * (n + 1)
        some += need > 0
    assert some > 10000


def test_python_refuses():
    i32 = dict(dtype=torch.int32)
    k, pages, table = torch.zeros((4, 2, 8)), torch.zeros((5, 16, 2, 8)), torch.zeros((2, 3), **i32)
    starts, lengths = torch.zeros(3, **i32), torch.zeros(2, **i32)
    good = dict(k_pages=pages, v_pages=pages, page_table=table, starts=starts, lengths=lengths)
    for bad in (dict(), dict(k_pages=pages[0]), dict(v_pages=pages[:3]), dict(k_pages=pages.half()), dict(page_table=table[:1]),
                dict(page_table=table.long()), dict(starts=starts[:2]), dict(lengths=lengths.long()),
                dict(page_table=table.T.contiguous().T)):
        with pytest.raises(bfhip.BfHipError):
            bfhip.paged_attention(k, **dict(good, **bad))
        with pytest.raises(bfhip.BfHipError):
            bfhip.cache_append(k, k, **dict(good, **bad))
    for k2, v2 in ((k, k[:3]), (k[:, :1], k[:, :1]), (k[0], k[0])):
        with pytest.raises(bfhip.BfHipError):
            bfhip.cache_append(k2, v2, **good)
    for bad in (dict(k_pages=pages[0, 0], v_pages=pages[0, 0]), dict(page_table=table[0]), dict(starts=starts[:0])):
        with pytest.raises(bfhip.BfHipError):
            bfhip.cache_append(k, k, **dict(good, **bad))
        with pytest.raises(bfhip.BfHipError):
            bfhip.paged_attention(k, **dict(good, **bad))
