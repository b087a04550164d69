"""The paged cache and the attention over it (bfhip_cache_append,
bfhip_paged_attention) against 64-bit formulas."""

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


def cache(device, dtype, kv_heads, dim, size, lens, spare=3, room=2, seed=1, fill=math.nan):
    """Pages in any order, `fill` where no token stands; tables with `room`
    entries past the last, which name no page."""
    g = gen(device, seed)
    used = [-(-n // size) for n in lens]
    total = sum(used) + spare
    order = torch.randperm(total, generator=g, device=device).int()
    table = torch.full((len(lens), max(used, default=0) + room), -1, dtype=torch.int32, device=device)
    pages = []
    for i in range(2):
        pages.append(torch.full((total, size, kv_heads, dim), fill, dtype=dtype, device=device))
    at = 0
    for b, n in enumerate(used):
        table[b, :n] = order[at:at + n]
        at += n
        j = torch.arange(lens[b], device=device)
        for p in pages:
            p[table[b].long()[j // size], j % size] = randn(g, lens[b], kv_heads, dim, dtype=dtype)
    return *pages, table, torch.tensor(lens, dtype=torch.int32, device=device)


def starts_of(device, lens):
    return torch.tensor([0] + list(lens)).cumsum(0).int().to(device)


def inputs(device, case, seed=1, **how):
    dtype, heads, kv_heads, dim, size, q_lens, k_lens, reach = case
    kp, vp, table, lengths = cache(device, dtype, kv_heads, dim, size, k_lens, seed=seed, **how)
    g = gen(device, seed + 100)
    q = randn(g, sum(q_lens), heads, dim, dtype=dtype)
    bias = None if reach is None else randn(g, heads, 2 * reach + 1)
    return dict(q=q, k_pages=kp, v_pages=vp, starts=starts_of(device, q_lens), lengths=lengths, scale=dim ** -0.5,
                bias=bias), table


def compare(call, table):
    out, lse = bfhip.paged_attention(page_table=table, lse=True, **call)
    want = ref.paged_attention(table=table, **call)
    check("out", out, *want["out"])
    dead = torch.isinf(want["lse"][0])
    assert (lse[dead] == -math.inf).all()
    check("lse", lse[~dead], want["lse"][0][~dead], want["lse"][1][~dead])
    assert torch.equal(bfhip.paged_attention(page_table=table, **call), out)
    return out


# (type, heads, kv_heads, dim, page, new tokens, lengths, reach): pages of one token,
# that end inside a tile of 32 keys, larger than one; lengths from none to ones that
# are split; more rows than a tile of 16; sequences without new tokens.
CASES = [(F32, 2, 2, 8, 1, [1], [1], None), (BF16, 32, 8, 128, 16, [1] * 5, [1, 700, 33, 32, 5000], None),
         (F16, 4, 1, 64, 7, [1, 3, 0, 1], [100, 30, 900, 3], None), (F32, 6, 3, 40, 5, [2, 1], [2, 333], 9),
         (BF16, 12, 12, 80, 100, [3] * 4, [1000, 3, 64, 99], 300), (F16, 8, 1, 16, 256, [1] * 70, list(range(1, 71)), None),
         (BF16, 8, 2, 96, 33, [40, 1], [40, 2000], None), (F32, 32, 2, 128, 64, [1, 1], [3000, 17], None),
         (F16, 40, 1, 32, 16, [2, 5], [50, 1200], 2047), (F32, 4, 4, 64, 2048, [1], [20000], None),
         (BF16, 2, 1, 128, 3, [300], [300], 20), (BF16, 4, 4, 128, 16, [1] * 300, [5 * i % 97 + 1 for i in range(300)], None)]


@pytest.mark.parametrize("case", CASES, ids=lambda c: str(c)[:90])
def test_paged_attention(device, case):
    compare(*inputs(device, case))


@pytest.mark.parametrize("dtype", [F32, F16, BF16])
def test_paged_attention_lengths_around_tiles_and_pages(device, dtype):
    lens = [n for m in (16, 32, 48, 64, 96, 128) for n in (m - 1, m, m + 1)]
    for size in (16, 32, 24):
        compare(*inputs(device, (dtype, 4, 2, 32, size, [1] * len(lens), lens, None)))


def test_paged_attention_equals_packed(device):
    """The same keys in one packed tensor."""
    call, table = inputs(device, (BF16, 16, 4, 128, 16, [1, 2, 1, 4], [3000, 500, 1, 4], None))
    got = bfhip.paged_attention(page_table=table, **call)
    k, k_starts = ref.gathered(call["k_pages"], table, call["lengths"])
    v, _ = ref.gathered(call["v_pages"], table, call["lengths"])
    packed = bfhip.attention(call["q"], k, v, call["starts"], k_starts, causal=True)
    # two results of one formula, each within the bound
    want = ref.paged_attention(table=table, **call)["out"]
    check("packed and paged", got, packed.double(), 2 * want[1])


def test_paged_attention_rows_without_keys(device):
    """More new tokens than keys: the first ones see nothing; and an empty
    cache."""
    call, table = inputs(device, (F16, 4, 2, 64, 8, [5, 2, 1], [3, 0, 70], None))
    out, lse = bfhip.paged_attention(page_table=table, lse=True, **call)
    dead = [0, 1, 5, 6]
    assert (out[dead] == 0).all() and (lse[:, dead] == -math.inf).all()
    want = ref.paged_attention(table=table, **call)
    check("out", out, *want["out"])


@pytest.mark.parametrize("value", [-1, 10 ** 6, -2 ** 31, 2 ** 31 - 1])
def test_paged_attention_sees_no_key_of_a_page_that_is_not_there(device, value):
    """As if the sequence had not had those keys."""
    case = (BF16, 8, 2, 64, 16, [1, 1], [800, 90], None)
    call, table = inputs(device, case)
    cut = table.clone()
    cut[0, 3:40] = value
    cut[1, 0] = value
    got = bfhip.paged_attention(page_table=cut, **call)
    left = torch.full_like(table, -1)
    left[0, :13] = torch.cat([table[0, :3], table[0, 40:50]])
    left[1, :5] = table[1, 1:6]
    fewer = dict(call, lengths=torch.tensor([800 - 37 * 16, 90 - 16], dtype=torch.int32, device=device))
    check("out", got, *ref.paged_attention(table=left, **fewer)["out"])
    cut.fill_(value)
    assert (bfhip.paged_attention(page_table=cut, **call) == 0).all()


def test_paged_attention_clamps_lengths(device):
    """To what the table holds, and to zero."""
    call, table = inputs(device, (F32, 4, 2, 32, 16, [1, 1], [64, 64], None), room=0)
    want = bfhip.paged_attention(page_table=table, **call)
    for n in (65, 2 ** 31 - 1):
        call["lengths"][1] = n
        assert torch.equal(bfhip.paged_attention(page_table=table, **call), want)
    for n in (-1, -2 ** 31):
        call["lengths"][1] = n
        got = bfhip.paged_attention(page_table=table, **call)
        assert (got[1] == 0).all() and torch.equal(got[0], want[0])


STARTS = [[-7, 3, 5, 10 ** 9], [-2 ** 31, -5, 2, 1, 6, 2 ** 31 - 1], [6, 0, 6], [0, 4, 2, 6, 5, 6], [300, -1, 3, 3, 6, -3]]


@pytest.mark.parametrize("at", STARTS, ids=str)
@pytest.mark.parametrize("dtype", [F32, BF16])
def test_paged_reads_and_writes_its_rows_only(device, dtype, at):
    """Starts of any value: nothing outside the rows is written, in a result or
    in a page that no sequence has."""
    n = len(at) - 1
    call, table = inputs(device, (dtype, 4, 2, 64, 16, [6], [300 + 500 * i for i in range(n)], None))
    call["starts"] = torch.tensor(at, dtype=torch.int64).clamp(-2 ** 31, 2 ** 31 - 1).int().to(device)
    wide = torch.full((46, 4, 64), math.nan, dtype=dtype, device=device)
    bfhip.paged_attention(page_table=table, out=wide[20:26], **call)
    rest = wide.clone()
    rest[20:26] = math.nan
    assert torch.isnan(rest).all()
    free = torch.ones(call["k_pages"].shape[0], dtype=torch.bool, device=device)
    free[table[table >= 0].long()] = False
    assert free.any()
    k = randn(gen(device), 6, 2, 64, dtype=dtype)
    bfhip.cache_append(k, k, call["k_pages"], call["v_pages"], table, call["starts"], call["lengths"])
    assert torch.isnan(call["k_pages"][free]).all() and torch.isnan(call["v_pages"][free]).all()


def test_paged_rows_of_no_sequence_stay(device):
    call, table = inputs(device, (BF16, 8, 2, 128, 16, [1, 1], [900, 50], None))
    q = randn(gen(device, 5), 7, 8, 128, dtype=BF16)
    q[2:4] = call["q"]
    want = bfhip.paged_attention(page_table=table, **call)
    out = torch.full_like(q, 7.0)
    call = dict(call, q=q, starts=call["starts"] + 2)
    bfhip.paged_attention(page_table=table, out=out, **call)
    assert torch.equal(out[2:4], want) and (out[:2] == 7).all() and (out[4:] == 7).all()


@pytest.mark.parametrize("dtype", [F32, F16, BF16])
def test_paged_strides(device, dtype):
    """Keys and values in one tensor, heads before tokens, tables wider than
    they are used, rows of a fused projection."""
    call, table = inputs(device, (dtype, 8, 4, 64, 16, [1, 2], [700, 80], None))
    want = bfhip.paged_attention(page_table=table, **call)
    both = torch.stack([call["k_pages"], call["v_pages"]], 1).transpose(2, 3).contiguous().transpose(2, 3)
    wide = torch.full((2, 200), 10 ** 6, dtype=torch.int32, device=device)[:, 20:20 + table.shape[1]]
    wide.copy_(table)
    fused = torch.empty((3, 12, 64), dtype=dtype, device=device)
    fused[:, 2:10] = call["q"]
    q = fused[:, 2:10]
    call = dict(call, q=q, k_pages=both[:, 0], v_pages=both[:, 1])
    assert torch.equal(bfhip.paged_attention(page_table=wide, **call), want)


def test_paged_attention_far_into_a_pool(device):
    """Pages beyond 4 GiB."""
    size, dim = 256, 128
    pages = (5 << 30) // (size * dim * 2)
    pool = torch.empty((pages, size, 1, dim), dtype=BF16, device=device)
    lens = [1000, 300]
    used = [4, 2]
    at = torch.tensor([pages - 1, 0, pages // 2, pages - 3, 7, pages - 2], dtype=torch.int32)
    table = torch.zeros((2, 4), dtype=torch.int32, device=device)
    table[0], table[1, :2] = at[:4], at[4:]
    pool[at.long().to(device)] = randn(gen(device), 6, size, 1, dim, dtype=BF16)
    q = randn(gen(device, 2), 2, 4, dim, dtype=BF16)
    call = dict(q=q, k_pages=pool, v_pages=pool, starts=starts_of(device, [1, 1]),
                lengths=torch.tensor(lens, dtype=torch.int32, device=device), scale=dim ** -0.5)
    assert used == [-(-n // size) for n in lens]
    compare(call, table)
    k = randn(gen(device, 3), 2, 1, dim, dtype=BF16)
    bfhip.cache_append(k, -k, pool, torch.zeros_like(pool), table, call["starts"], call["lengths"])
    assert torch.equal(pool[pages - 3, 999 - 768], k[0]) and torch.equal(pool[pages - 2, 299 - 256], k[1])


@pytest.mark.parametrize("scale", [0.0, -0.3, 1e-30, 50.0])
def test_paged_attention_scales(device, scale):
    call, table = inputs(device, (F32, 4, 2, 32, 16, [1, 2], [300, 40], None))
    compare(dict(call, scale=scale), table)


def test_paged_attention_biases_that_mask(device):
    """-inf, the type's lowest value, and a bias that leaves a row nothing."""
    call, table = inputs(device, (BF16, 4, 2, 64, 16, [1, 2], [300, 40], 50))
    call["bias"][0, 10:45] = -math.inf
    call["bias"][1, 10:45] = torch.finfo(F32).min
    call["bias"][2] = -math.inf
    out, lse = bfhip.paged_attention(page_table=table, lse=True, **call)
    assert (out[:, 2] == 0).all() and (lse[2] == -math.inf).all()
    check("out", out, *ref.paged_attention(table=table, **call)["out"])


@pytest.mark.parametrize("dtype", [F32, F16, BF16])
def test_paged_of_nothing(device, dtype):
    """No pages, tables without entries, no sequences, no tokens."""
    i32 = dict(dtype=torch.int32, device=device)
    q = randn(gen(device), 3, 4, 64, dtype=dtype)
    pages = torch.empty((0, 16, 2, 64), dtype=dtype, device=device)
    some = randn(gen(device, 1), 2, 16, 2, 64, dtype=dtype)
    one = dict(starts=starts_of(device, [1, 2]), lengths=torch.tensor([5, 30], **i32))
    for pool, table in ((pages, torch.zeros((2, 2), **i32)), (some, torch.zeros((2, 0), **i32)), (pages, torch.zeros((2, 0), **i32))):
        out, lse = bfhip.paged_attention(q, pool, pool, table, lse=True, **one)
        assert (out == 0).all() and (lse == -math.inf).all()
        before = pool.clone()
        bfhip.cache_append(q[:, :2], q[:, 2:], pool, pool, table, **one)
        assert torch.equal(pool, before)
    none = dict(starts=torch.zeros(1, **i32), lengths=torch.zeros(0, **i32))
    out = torch.full_like(q, 3.0)
    bfhip.paged_attention(q, some, some, torch.zeros((0, 2), **i32), out=out, **none)
    assert (out == 3).all()
    empty = dict(starts=starts_of(device, [0, 0]), lengths=one["lengths"])
    assert bfhip.paged_attention(q[:0], some, some, torch.zeros((2, 2), **i32), **empty).shape == (0, 4, 64)


def test_paged_sequences_that_share_pages(device):
    """A common beginning, and one page twice in a sequence."""
    call, table = inputs(device, (BF16, 8, 2, 64, 16, [1, 1, 2], [700, 90, 320], None))
    table[1, :5] = table[0, :5]
    table[2, 3:9] = table[2, 2]
    compare(call, table)


# ------------------------------------------------------------------- append
@pytest.mark.parametrize("dtype", [F32, F16, BF16])
@pytest.mark.parametrize("size", [1, 5, 16, 64])
def test_append(device, dtype, size):
    """New tokens at the sequences' ends; nothing else changes."""
    lens, new = [70, 5, 1, 33, 400, 9], [3, 5, 1, 0, 131, 1]
    kp, vp, table, lengths = cache(device, dtype, 3, 40, size, lens, fill=7.0)
    g = gen(device, 4)
    fused = randn(g, sum(new) + 5, 6 * 40 + 1, dtype=dtype)[:, 1:]  # (rows of no alignment)
    k, v = (t.unflatten(1, (3, 40)) for t in fused.split(120, 1))
    starts = starts_of(device, new) + 2
    want = [kp.clone(), vp.clone()]
    for b, n in enumerate(new):
        for i in range(n):
            j = lens[b] - n + i
            for w, x in zip(want, (k, v)):
                w[table[b, j // size].long(), j % size] = x[starts[b] + i]
    bfhip.cache_append(k, v, kp, vp, table, starts, lengths)
    assert torch.equal(kp, want[0]) and torch.equal(vp, want[1])


def test_append_writes_nothing_for_pages_that_are_not_there(device):
    kp, vp, table, lengths = cache(device, F16, 2, 64, 4, [6, 30], fill=7.0)
    k = randn(gen(device), 9, 2, 64, dtype=F16)
    table[0, 1], table[1, 7] = 10 ** 6, -3
    before = kp.clone(), vp.clone()
    # sequence 0 has more new tokens than keys: the first two stand before it
    bfhip.cache_append(k, k, kp, vp, table, starts_of(device, [8, 1]), lengths)
    assert torch.equal(kp[table[0, 0].long()], k[2:6])
    for t, old in zip((kp, vp), before):
        t[table[0, 0].long()] = old[table[0, 0].long()]
        assert torch.equal(t, old)
    lengths.fill_(-5)
    bfhip.cache_append(k, k, kp, vp, table, starts_of(device, [8, 1]), lengths)
    assert torch.equal(kp, before[0])


def test_append_of_many_tokens(device):
    lens = [3000, 2500]
    kp, vp, table, lengths = cache(device, BF16, 8, 128, 64, lens, fill=0.0)
    g = gen(device, 4)
    k, v = randn(g, 5500, 8, 128, dtype=BF16), randn(g, 5500, 8, 128, dtype=BF16)
    bfhip.cache_append(k, v, kp, vp, table, starts_of(device, lens), lengths)
    assert torch.equal(ref.gathered(kp, table, lengths)[0], k) and torch.equal(ref.gathered(vp, table, lengths)[0], v)


# ------------------------------------------------------------- in earnest
def test_steps_of_several_sequences(device):
    """Prompts, then single tokens: rotary, append, attention, against packed
    attention over everything so far."""
    heads, kv_heads, dim, size = 8, 2, 64, 16
    freq = bfhip.rotary_frequencies(dim, device=device)
    lens, news = [0, 0, 0], [[37, 5, 100], [1, 1, 1], [1, 0, 1], [1, 3, 1]]
    kp = torch.full((40, size, kv_heads, dim), math.nan, dtype=BF16, device=device)
    vp = kp.clone()
    table = torch.randperm(40, generator=gen(device, 8), device=device).int()[:36].view(3, 12).contiguous()
    g, kept = gen(device, 7), [([], []) for _ in lens]
    for new in news:
        n = sum(new)
        q, k, v = (randn(g, n, (heads + 2 * kv_heads) * dim, dtype=BF16).unflatten(1, (-1, dim))
                   .split([heads, kv_heads, kv_heads], 1))
        positions = torch.cat([torch.arange(a, a + m) for a, m in zip(lens, new)]).int().to(device)
        lens = [a + m for a, m in zip(lens, new)]
        starts = starts_of(device, new)
        lengths = torch.tensor(lens, dtype=torch.int32, device=device)
        bfhip.rotary(q, k, positions, freq, out=(q, k))
        bfhip.cache_append(k, v, kp, vp, table, starts, lengths)
        got = bfhip.paged_attention(q, kp, vp, table, starts, lengths)
        for b, (ks, vs) in enumerate(kept):
            ks.append(k[starts[b]:starts[b + 1]].clone())
            vs.append(v[starts[b]:starts[b + 1]].clone())
        pk, pv = (torch.cat([torch.cat(both[i]) for both in kept]) for i in range(2))
        want = ref.ref.attention(q, pk, pv, starts, starts_of(device, lens), True, dim ** -0.5)
        check("out", got, *want["out"])


def test_paged_in_a_graph(device):
    """Lengths, pages and tokens change between the replays of one capture."""
    call, table = inputs(device, (BF16, 16, 4, 64, 16, [1] * 6, [900, 20, 1, 333, 64, 2000], None), room=70)
    call["lengths"] -= 1
    k, v = (randn(gen(device, s), 6, 4, 64, dtype=BF16) for s in (1, 2))
    out, lse_in = torch.empty_like(call["q"]), None
    args = (call["k_pages"], call["v_pages"], table, call["starts"], call["lengths"])
    side = torch.cuda.Stream()
    with torch.cuda.stream(side):
        bfhip.cache_append(k, v, *args)
        bfhip.paged_attention(call["q"], *args, out=out)
    side.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        bfhip.cache_append(k, v, *args)
        bfhip.paged_attention(call["q"], *args, out=out)
    g = gen(device, 3)
    for lens in ([899, 19, 1, 332, 63, 1999], [900, 20, 1, 333, 64, 2000], [5, 20, 1, 333, 9, 1000]):
        call["lengths"].copy_(torch.tensor(lens, dtype=torch.int32))
        for t in (k, v, call["q"]):
            t.copy_(randn(g, *t.shape, dtype=BF16))
        out.zero_()
        graph.replay()
        torch.cuda.synchronize()
        check("out", out, *ref.paged_attention(table=table, **call)["out"])
        assert torch.equal(out, bfhip.paged_attention(call["q"], *args))


def test_two_calls_on_two_streams(device):
    calls = [inputs(device, (BF16, 16, 4, 128, 16, [1] * 4, [4000, 3000, 100, 5], None), seed=s) for s in (1, 2)]
    want = [bfhip.paged_attention(page_table=t, **c) for c, t in calls]
    streams = [torch.cuda.Stream() for _ in calls]
    torch.cuda.synchronize()
    for _ in range(5):
        got = [bfhip.paged_attention(page_table=t, stream=s, **c) for (c, t), s in zip(calls, streams)]
    torch.cuda.synchronize()
    assert all(torch.equal(a, b) for a, b in zip(got, want))


def test_paged_strides_of_no_account(device):
    """One token of one head: its strides are of no account."""
    call, table = inputs(device, (BF16, 1, 1, 64, 16, [1], [70], None))
    want = bfhip.paged_attention(page_table=table, **call)
    for strides in ((0, 0, 1), (64, 1, 1), (5, 7, 1)):
        q = call["q"].as_strided((1, 1, 64), strides)
        assert torch.equal(bfhip.paged_attention(page_table=table, **dict(call, q=q)), want)
        pools = [call[n].clone() for n in ("k_pages", "v_pages")]
        bfhip.cache_append(q, q, *pools, table, call["starts"], call["lengths"])
        page, row = table[0, 69 // 16], 69 % 16
        assert all(torch.equal(p[page, row], q[0]) for p in pools)


@pytest.mark.parametrize("heads,kv_heads,dim,n", [(128, 128, 8, 5250), (32, 16, 128, 2650)])
def test_paged_attention_of_more_tokens_than_one_launch_joins(device, heads, kv_heads, dim, n):
    """Sequences of new tokens alone, whose number times heads times the padded dim
    / 128 is more than the workgroups of a launch; all sequences have the same
    queries and pages."""
    new = 100 if dim == 8 else 200
    assert n * new * heads * max(dim, 32) // 128 >= 1 << 24
    call, table = inputs(device, (F16, heads, kv_heads, dim, 16, [new], [new], None))
    value, bound = ref.paged_attention(table=table, **call)["out"]
    many = dict(call, q=call["q"].repeat(n, 1, 1), starts=torch.arange(n + 1, dtype=torch.int32, device=device) * new,
                lengths=call["lengths"].repeat(n))
    out = bfhip.paged_attention(page_table=table.repeat(n, 1), **many).view(n, *value.shape)
    for part in range(0, n, 50):  # (all of them: a share's border falls into any sequence)
        share = ((out[part:part + 50].double() - value).abs() / bound).max()
        assert share <= 1, (part, share)


@pytest.mark.parametrize("case", [(BF16, 8, 8, 64, 16, [4] * 40, [4 + 3 * i for i in range(40)], None),
                                  (F16, 8, 2, 128, 16, [1] * 8, [3, 9, 40, 100, 300, 1000, 5000, 20000], None),
                                  (BF16, 16, 2, 32, 7, [1, 20], [700, 200], 30), (F16, 4, 4, 40, 5, [2] * 20, [25] * 20, None)], ids=lambda c: str(c)[:60])
def test_probabilities_have_twice_the_precision(device, case):
    """No rounding of a 16-bit type comes between the scores and the results but
    the results' own."""
    call, table = inputs(device, case)
    out = bfhip.paged_attention(page_table=table, **call)
    check("out", out, *ref.paged_attention(table=table, left=True, **call)["out"])


@pytest.mark.parametrize("dtype", [F32, F16, BF16])
@pytest.mark.parametrize("dim", [24, 64, 128])
def test_infinite_values(device, dtype, dim):
    """An infinite value makes its element's results infinite and nothing else, of
    keys that lie in one share and in many."""
    call, table = inputs(device, (dtype, 8, 2, dim, 16, [1] * 5, [5, 40, 300, 20000, 33], None))
    want = bfhip.paged_attention(page_table=table, **call)
    for b, j, d, value in ((0, 2, 1, math.inf), (1, 35, dim - 1, -math.inf), (2, 0, 5, math.inf), (3, 17000, 9, -math.inf)):
        call["v_pages"][table[b, j // 16].long(), j % 16, 1, d] = value
        want[b, 4:, d] = value
    assert torch.equal(bfhip.paged_attention(page_table=table, **call), want)
