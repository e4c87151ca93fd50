"""Paged 4-bit key/value cache against its definition in 64 bits.

Writing and reading are exact (bitwise).  Attention, per output value: queries and unpacked
keys are exact, so the scores' FP32 accumulation, 8 * 2^-23 of their terms' magnitudes,
moves a weight by that much relative; exponential, sum and division add 2^-18
relative; a weight is rounded to f16, 2^-11 relative or half of f16's least step, 2^-25,
where a reference that is never above the largest weighs 2^7 (2^11 with few rows): 2^-32 of
the largest; the output is rounded once."""

from __future__ import annotations

import ctypes

import pytest
import torch

from lesiondiffusion_mlx_b200 import _lib, kv_cache
from oracle import kv_int4 as oracle

pytestmark = pytest.mark.gpu

UNIT = {torch.float16: 2.0 ** -11, torch.bfloat16: 2.0 ** -8}
TINY = {torch.float16: 2.0 ** -25, torch.bfloat16: 0.0}


def make_cache(pages, heads, dim, page, device, seed, low=88, high=112):
    g = torch.Generator().manual_seed(seed)
    codes = [torch.randint(0, 256, (pages, heads, page, dim // 2), generator=g, dtype=torch.uint8) for _ in range(2)]
    scales = [torch.randint(low, high, (pages, heads, dim // 16, page), generator=g, dtype=torch.uint8)
              for _ in range(2)]
    return kv_cache.KvCacheInt4(*(t.to(device) for t in codes + scales))


def host(cache):
    return [t.cpu().clone() for t in cache]


def make_table(batch, width, seed, spare=3):
    g = torch.Generator().manual_seed(seed)
    pages = batch * width + spare
    return torch.randperm(pages, generator=g)[: batch * width].view(batch, width).to(torch.int32), pages


def ints(values, device):
    return torch.tensor(values, dtype=torch.int32, device=device)


def same_cache(cache, want):
    for got, ref in zip(host(cache), want):
        assert torch.equal(got, ref)


def append_both(want, k, v, table, start, counts):
    heads = want[0].shape[1]
    for at, new in ((0, k), (1, v)):
        oracle.append(want[at], want[at + 2], new.unflatten(-1, (heads, -1)), table, start, counts)


@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16, torch.float32])
@pytest.mark.parametrize("heads,dim,page,tokens,start", [
    (1, 64, 64, 1, [0, 1, 63, 64, 100]), (2, 128, 128, 130, [0, 5, 127]), (3, 32, 16, 40, [0, 15, 16, 7]),
    (2, 64, 32, 33, [31, 0]), (1, 128, 16, 1, [15]), (3, 128, 64, 6, [70, 71, 72, 73])])
def test_append_is_exact(cuda_device, dtype, heads, dim, page, tokens, start):
    """Over random older content, which stays; groups of all magnitudes, among them ones past the
    scales' ends and ones of zeros; 16-bit values meet many ties."""
    batch = len(start)
    table, pages = make_table(batch, (max(start) + tokens + page - 1) // page + 1, 3)
    cache = make_cache(pages, heads, dim, page, cuda_device, 4)
    want = host(cache)
    g = torch.Generator().manual_seed(5)
    k, v = (torch.randn(batch, tokens, heads * dim // 16, 16, generator=g) for _ in range(2))
    k *= torch.exp2(torch.randint(-21, 14, k.shape[:-1], generator=g).float())[..., None]
    v[..., 0, :] = 0.0
    k, v = (t.flatten(-2).to(dtype) for t in (k, v))
    kv_cache.kv_append(cache, k.to(cuda_device), v.to(cuda_device), table.to(cuda_device), ints(start, cuda_device))
    append_both(want, k, v, table, start, [tokens] * batch)
    same_cache(cache, want)
    kv_cache.kv_append(cache, k.to(cuda_device), v.to(cuda_device), table.to(cuda_device), ints(start, cuda_device))
    same_cache(cache, want)
    assert _lib.device_status(reset=True) == 0


def test_every_scale_and_every_tie(cuda_device):
    """Maxima at, just below and just above 7.5 of each scale, and values half way between codes."""
    scales = torch.tensor(oracle.SCALES[1:], dtype=torch.float64)
    rows = []
    for top in (7.5 * scales, 7.5 * scales * (1 - 2.0 ** -9), 7.5 * scales * (1 + 2.0 ** -9)):
        ties = (torch.arange(15) - 7.5)[None] * scales[:, None]
        rows.append(torch.cat((top[:, None], ties.clamp(-top[:, None], top[:, None])), 1))
    x = torch.cat(rows).float()
    x = torch.cat((x, -x), 1).reshape(1, -1, 32)
    table, pages = make_table(1, -(-x.shape[1] // 64), 3)
    for dtype in (torch.float32, torch.float16, torch.bfloat16):
        y = x.to(dtype)
        y = torch.where(torch.isfinite(y), y, torch.zeros_like(y))
        cache = make_cache(pages, 1, 32, 64, cuda_device, 4)
        want = host(cache)
        dev = y.to(cuda_device)
        kv_cache.kv_append(cache, dev, -dev, table.to(cuda_device), ints([0], cuda_device))
        append_both(want, y, -y, table, [0], [y.shape[1]])
        same_cache(cache, want)


def test_append_counts_and_what_is_not_finite(cuda_device):
    heads, dim, page, batch = 2, 32, 16, 3
    table, pages = make_table(batch, 4, 7)
    cache = make_cache(pages, heads, dim, page, cuda_device, 8)
    want = host(cache)
    g = torch.Generator().manual_seed(9)
    at = [0, 14, 40]
    for step in range(12):
        k, v = (torch.randn(batch, 3, heads * dim, generator=g) for _ in range(2))
        if step % 3 == 1:
            k[0, 0, 3], v[0, 0, 17], k[1, 0, 5], v[1, 0] = float("nan"), float("inf"), float("-inf"), 0
        counts = [1, step % 4, 0 if step % 2 else 2]
        kv_cache.kv_append(cache, k.to(cuda_device), v.to(cuda_device), table.to(cuda_device), ints(at, cuda_device),
                           counts=ints(counts, cuda_device))
        append_both(want, k, v, table, at, counts)
        at = [a + c for a, c in zip(at, counts)]
        same_cache(cache, want)
    assert (want[2] == oracle.NAN).any() and _lib.device_status(reset=True) == 0


def test_append_strided_and_out_of_range(cuda_device):
    heads, dim, page, batch = 2, 64, 32, 2
    table, pages = make_table(batch, 3, 1)
    cache = make_cache(pages, heads, dim, page, cuda_device, 2)
    want = host(cache)
    wide = torch.randn(batch, 9, 3 * heads * dim + 5, generator=torch.Generator().manual_seed(3)).to(torch.bfloat16)
    k, v = wide[..., 128:256], wide[..., 261:389]
    dev = wide.to(cuda_device)
    kv_cache.kv_append(cache, dev[..., 128:256], dev[..., 261:389], table.to(cuda_device), ints([4, 30], cuda_device))
    append_both(want, k, v, table, [4, 30], [9, 9])
    same_cache(cache, want)
    assert _lib.device_status(reset=True) == 0
    lost = table.clone()
    lost[0, 0], lost[1, 0] = pages, -1
    for tab, start in ((lost, [0, 0]), (table, [96, 1000]), (table, [-1, -40]), (table, [2 ** 31 - 1, 2 ** 31 - 4])):
        kv_cache.kv_append(cache, dev[..., 128:256], dev[..., 261:389], tab.to(cuda_device), ints(start, cuda_device))
        assert _lib.device_status(reset=True) == 2
    same_cache(cache, want)


@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16, torch.float32])
@pytest.mark.parametrize("heads,dim,page,tokens,start,lengths", [
    (1, 64, 64, 1, [0, 1, 63, 64, 100], [1, 2, 64, 64, 200]), (2, 128, 128, 130, None, [130, 0, 129]),
    (3, 32, 16, 41, [0, 15, 16, 7], [9, 16, 200, 48]), (2, 64, 32, 33, [31, 0], [40, 90]),
    (4, 64, 64, 77, None, [77, 5])])
@pytest.mark.parametrize("eight", [False, True])
def test_read(cuda_device, dtype, heads, dim, page, tokens, start, lengths, eight):
    """Rows of both caches, zeros behind the lengths, whatever lies there."""
    batch = len(lengths)
    table, pages = make_table(batch, -(-200 // page) + 1, 3)
    cache = make_cache(pages, heads, dim, page, cuda_device, 4)
    g = torch.Generator().manual_seed(6)
    if eight:
        codes = [torch.randint(0, 127, (pages, heads, page, dim), generator=g, dtype=torch.uint8) for _ in range(2)]
        codes[0][0, 0, 0, 0] = 0xFF
        scales = [torch.randint(117, 137, (pages, heads), generator=g, dtype=torch.uint8) for _ in range(2)]
        cache = kv_cache.KvCacheFp8(*(t.to(cuda_device).view(kv_cache.CODES) for t in codes),
                                    *(t.to(cuda_device).view(kv_cache.SCALES) for t in scales))
        want = [c.view(torch.float8_e4m3fn).double() * torch.exp2(s.double() - 127)[..., None, None]
                for c, s in zip(codes, scales)]
    else:
        cache.k_scale[0, 0, 0, 0] = oracle.NAN
        k, v, ks, vs = host(cache)
        want = [oracle.values(k, ks), oracle.values(v, vs)]
    at = None if start is None else ints(start, cuda_device)
    got = kv_cache.kv_read(cache, table.to(cuda_device), ints(lengths, cuda_device), tokens=tokens, start=at, dtype=dtype)
    for x, y in zip(got, want):
        assert x.dtype == dtype and x.shape == (batch, tokens, heads * dim)
        ref = torch.zeros(batch, tokens, heads * dim, dtype=torch.float64)
        for b, n in enumerate(lengths):
            first = 0 if start is None else start[b]
            held = oracle.rows(y, table, b, n).transpose(0, 1).flatten(1)[first: first + tokens]
            ref[b, : held.shape[0]] = held
        assert torch.equal(x.cpu().double().nan_to_num(1e9), ref.to(dtype).double().nan_to_num(1e9))
    assert _lib.device_status(reset=True) == 0


def test_read_into_strided_rows_and_out_of_range(cuda_device):
    heads, dim, page = 2, 32, 32
    table, pages = make_table(2, 3, 3)
    cache = make_cache(pages, heads, dim, page, cuda_device, 4)
    k, v, ks, vs = host(cache)
    wide = torch.full((2, 50, 2 * 64 + 3), 7.0, dtype=torch.float16, device=cuda_device)
    out = wide[..., 1:65], wide[..., 66:130]
    kv_cache.kv_read(cache, table.to(cuda_device), ints([96, 40], cuda_device), tokens=50, start=ints([46, 3], cuda_device),
                     out=out)
    for x, c, s in ((out[0], k, ks), (out[1], v, vs)):
        y = oracle.values(c, s)
        assert torch.equal(x[0].cpu().double(), oracle.rows(y, table, 0, 96).transpose(0, 1).flatten(1)[46:])
        assert torch.equal(x[1, :37].cpu().double(), oracle.rows(y, table, 1, 40).transpose(0, 1).flatten(1)[3:])
        assert (x[1, 37:] == 0).all()
    assert (wide[..., [0, 65, 130]] == 7).all() and _lib.device_status(reset=True) == 0
    bad = table.clone()
    bad[0, 1] = pages
    for tab, lengths, start in ((bad, [96, 40], [0, 0]), (table, [97, 40], [0, 0]), (table, [-1, 40], [0, 0]),
                                (table, [96, 40], [-2, 0])):
        x, _ = kv_cache.kv_read(cache, tab.to(cuda_device), ints(lengths, cuda_device), tokens=96,
                                start=ints(start, cuda_device))
        assert _lib.device_status(reset=True) == 2
        y = oracle.values(k, ks)
        assert torch.equal(x[1, :40].cpu().double(), oracle.rows(y, table, 1, 40).transpose(0, 1).flatten(1))
        if lengths[0] < 0 or start[0] < 0:
            assert (x[0] == 0).all()
        elif tab is bad:
            assert (x[0, 32:64] == 0).all()
            assert torch.equal(x[0, :32].cpu().double(), oracle.rows(y, table, 0, 32).transpose(0, 1).flatten(1))


def check_attention(got, ref, dtype):
    bound = ((2.0 ** -11 + 2.0 ** -18 + 2 * 8 * 2.0 ** -23 * ref["score"]) * ref["size"] + 2.0 ** -32 * ref["peak"]
             + UNIT[dtype] * ref["out"].abs() * (1 + 2.0 ** -8) + TINY[dtype])
    err = (got.cpu().double().view(ref["out"].shape) - ref["out"]).abs()
    assert (err <= bound).all(), float((err / bound.clamp(min=1e-300)).max())


def reference(q, cache, table, lengths, group, scale, causal):
    k, v, ks, vs = host(cache)
    return oracle.attention(q, oracle.values(k, ks), oracle.values(v, vs), table, lengths, group, scale, causal)


# as many pairs as SMs, so that a tile of rows has all tokens to itself: its blocks alternate
LONG = [3200, 0, 1, 128, 129, 255, 256, 257, 3199, 2000, 640] + [5] * 26
CASES = [  # lengths, queries, kv heads, group, dim, page, causal
    ([1], 1, 1, 1, 64, 64, False), ([0, 3, 64, 65, 200], 1, 2, 4, 128, 64, True), ([77], 50, 4, 1, 64, 64, False),
    ([129, 17], 5, 1, 3, 32, 16, True), ([40, 0, 7], 12, 2, 2, 64, 32, True), ([300], 1, 1, 16, 128, 128, False),
    ([500, 30], 1, 1, 17, 64, 128, False), ([1500], 1, 2, 1, 128, 16, False), ([260], 130, 1, 2, 128, 64, True),
    ([5], 30, 1, 8, 32, 64, True), ([200, 128, 1], 64, 2, 4, 128, 128, True), ([333], 300, 1, 1, 64, 16, False),
    ([63, 62, 66, 127], 2, 1, 4, 32, 32, True), ([700], 257, 1, 1, 32, 128, True), ([130], 513, 1, 1, 128, 16, False),
    ([1100, 0, 1, 128, 129, 640, 1025], 20, 2, 4, 128, 64, True), ([1300, 257, 3], 50, 1, 1, 64, 16, False),
    (LONG, 25, 4, 4, 128, 64, True), (LONG, 64, 4, 1, 64, 16, False), (LONG, 32, 4, 4, 32, 128, True),
    (LONG, 49, 4, 1, 128, 32, False), ([130000, 70000], 50, 1, 1, 32, 128, True)]


@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
@pytest.mark.parametrize("lengths,queries,heads,group,dim,page,causal", CASES)
def test_attention(cuda_device, dtype, lengths, queries, heads, group, dim, page, causal):
    batch = len(lengths)
    table, pages = make_table(batch, -(-max(lengths) // page) + 1, 11)
    cache = make_cache(pages, heads, dim, page, cuda_device, 12, 96, 112)
    # everything the lengths leave out holds NaN: the tails of last pages, and the pages nobody owns
    owned = set()
    for b, n in enumerate(lengths):
        for slot in range(-(-n // page)):
            owned.add(int(table[b, slot]))
            if n - slot * page < page:
                for t in (cache.k_scale, cache.v_scale):
                    t[int(table[b, slot]), :, :, n - slot * page:] = oracle.NAN
    for at in set(range(pages)) - owned:
        for t in (cache.k_scale, cache.v_scale):
            t[at] = oracle.NAN
    q = 2 * torch.randn(batch, queries, heads * group * dim, generator=torch.Generator().manual_seed(13))
    q = q.to(dtype)
    args = (q.to(cuda_device), cache, table.to(cuda_device), ints(lengths, cuda_device))
    got = kv_cache.kv_attention(*args, scale=dim ** -0.5, causal=causal)
    check_attention(got, reference(q, cache, table, lengths, group, dim ** -0.5, causal), dtype)
    assert torch.equal(kv_cache.kv_attention(*args, scale=dim ** -0.5, causal=causal), got)
    assert _lib.device_status(reset=True) == 0


@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
@pytest.mark.parametrize("causal", [False, True])
@pytest.mark.parametrize("queries,group,dim,page", [(1, 4, 128, 64), (5, 2, 64, 16), (12, 1, 32, 32), (7, 2, 128, 128),
                                                    (70, 1, 64, 64), (130, 2, 128, 16), (300, 1, 32, 128)])
def test_attention_nan_reaches_its_channels_and_the_queries_that_see_it(cuda_device, dtype, causal, queries, group, dim,
                                                                        page):
    """NaN groups of values in tokens that all, some or none of the queries see."""
    heads, lengths = 2, [310, 37]
    table, pages = make_table(2, 320 // page + 1, 21)
    cache = make_cache(pages, heads, dim, page, cuda_device, 22, 96, 112)
    for b, head, tok, group_at in ((0, 0, 309, 0), (0, 1, 305, 0), (0, 1, 306, dim // 16 - 1), (0, 0, 290, 1),
                                   (0, 1, 12, 1), (1, 0, 36, 0), (1, 1, 20, dim // 32)):
        cache.v_scale[int(table[b, tok // page]), head, group_at, tok % page] = oracle.NAN
    q = torch.randn(2, queries, heads * group * dim, generator=torch.Generator().manual_seed(23)).to(dtype)
    ref = reference(q, cache, table, lengths, group, dim ** -0.5, causal)
    got = kv_cache.kv_attention(q.to(cuda_device), cache, table.to(cuda_device), ints(lengths, cuda_device),
                                scale=dim ** -0.5, causal=causal)
    nan = torch.isnan(ref["out"])
    assert nan.any() and not nan.all()
    assert torch.equal(torch.isnan(got.cpu().view(nan.shape)), nan)
    finite = {k: torch.where(torch.isnan(x), torch.zeros_like(x), x) for k, x in ref.items()}
    finite["peak"] = torch.full_like(finite["peak"], 310 * 8 * 30.0)
    check_attention(torch.where(nan.to(cuda_device), 0.0, got.view(nan.shape)), finite, dtype)


@pytest.mark.parametrize("causal", [False, True])
@pytest.mark.parametrize("queries,dim,page", [(60, 128, 64), (100, 64, 16), (128, 32, 128)])
def test_attention_nan_and_lost_pages_among_many_blocks(cuda_device, causal, queries, dim, page):
    """NaN groups of values in blocks of either parity that some queries see, and a page that is not there."""
    heads, lengths, lost, dtype = 4, [1310, 1100] + [1] * 35, 5, torch.float16
    table, pages = make_table(len(lengths), 3264 // page, 21)
    cache = make_cache(pages, heads, dim, page, cuda_device, 22, 96, 112)
    q = torch.randn(len(lengths), queries, heads * dim, generator=torch.Generator().manual_seed(23)).to(dtype)
    need = ctypes.c_size_t()
    _lib.call("ldb_kv_attention_int4_workspace_size", len(lengths), queries, heads, heads, dim, table.shape[1] * page,
              ctypes.byref(need))
    assert need.value == 2 * len(lengths) * heads * queries * (dim + 2) * 4  # (two parts: blocks alternate)
    args = (q.to(cuda_device), cache)
    kept, holes = table.clone(), table.clone()
    kept[:, lost:-1] = table[:, lost + 1:]
    holes[:, lost] = -1
    if not causal:  # (a query's place among the tokens would be another)
        got = kv_cache.kv_attention(*args, holes.to(cuda_device), ints(lengths, cuda_device), scale=dim ** -0.5)
        assert _lib.device_status(reset=True) == 2
        check_attention(got, reference(q, cache, kept, [max(n - page, 1) for n in lengths], 1, dim ** -0.5, False), dtype)
    for b, head, tok, group_at in ((0, 0, 1309, 0), (0, 1, 1275, 1), (1, 0, 1099, 0), (1, 2, 1060, 1)):
        cache.v_scale[int(table[b, tok // page]), head, group_at, tok % page] = oracle.NAN
    ref = reference(q, cache, table, lengths, 1, dim ** -0.5, causal)
    got = kv_cache.kv_attention(*args, table.to(cuda_device), ints(lengths, cuda_device), scale=dim ** -0.5, causal=causal)
    nan = torch.isnan(ref["out"])
    assert nan.any() and _lib.device_status(reset=True) == 0  # (32 channels without a mask: all of it)
    assert torch.equal(torch.isnan(got.cpu().view(nan.shape)), nan)
    finite = {k: torch.where(torch.isnan(x), torch.zeros_like(x), x) for k, x in ref.items()}
    finite["peak"] = torch.full_like(finite["peak"], 1310 * 8 * 30.0)
    check_attention(torch.where(nan.to(cuda_device), 0.0, got.view(nan.shape)), finite, dtype)


@pytest.mark.parametrize("queries", [1, 3, 70])
def test_attention_future_nan_keys_do_not_reach_the_past(cuda_device, queries):
    heads, dim, page, n = 2, 64, 32, 150
    table, pages = make_table(1, 5, 2)
    cache = make_cache(pages, heads, dim, page, cuda_device, 3, 96, 112)
    q = torch.randn(1, queries, heads * dim, generator=torch.Generator().manual_seed(4)).to(torch.float16)
    ref = reference(q, cache, table, [n], 1, 0.125, True)
    cache.k_scale[int(table[0, (n - 1) // page]), :, 2, (n - 1) % page] = oracle.NAN
    got = kv_cache.kv_attention(q.to(cuda_device), cache, table.to(cuda_device), ints([n], cuda_device), scale=0.125,
                                causal=True)
    assert torch.isnan(got[:, -1]).all()
    check_attention(got[:, :-1], {k: x[:, :-1] for k, x in ref.items()}, torch.float16)


@pytest.mark.parametrize("queries", [9, 60, 200])
@pytest.mark.parametrize("value", [float("inf"), float("-inf"), float("nan")])
def test_attention_queries_without_keys_are_zero_whatever_they_hold(cuda_device, queries, value):
    heads, dim, page, n = 1, 64, 64, 6  # the first queries - 6 queries see nothing
    table, pages = make_table(1, 1, 31)
    cache = make_cache(pages, heads, dim, page, cuda_device, 32, 96, 112)
    for dtype in (torch.float16, torch.bfloat16):
        q = torch.randn(1, queries, dim, generator=torch.Generator().manual_seed(33)).to(dtype)
        ref = reference(q, cache, table, [n], 1, 0.125, True)
        q[0, 1, 5] = value
        args = (cache, table.to(cuda_device), ints([n], cuda_device))
        got = kv_cache.kv_attention(q.to(cuda_device), *args, scale=0.125, causal=True)
        assert (got[0, : queries - n] == 0).all()
        check_attention(got, ref, dtype)
        q[0, -2, 5] = value  # one that sees keys becomes NaN, and no other does
        got = kv_cache.kv_attention(q.to(cuda_device), *args, scale=0.125, causal=True)
        assert torch.isnan(got[0, -2]).all()
        rest = [i for i in range(queries) if i != queries - 2]
        check_attention(got[:, rest], {k: x[:, rest] for k, x in ref.items()}, dtype)


@pytest.mark.parametrize("queries,group,dim,page", [(1, 4, 128, 64), (3, 1, 64, 16), (3, 4, 32, 32), (20, 2, 128, 128),
                                                    (90, 1, 64, 16), (130, 2, 128, 64), (64, 1, 32, 128)])
@pytest.mark.parametrize("lost", [-1, 1 << 20])
def test_attention_leaves_out_pages_outside_the_cache(cuda_device, queries, group, dim, page, lost):
    """The result without the tokens of such a page, and a status bit; an item with no other page gives zeros."""
    heads, dtype = 2, torch.bfloat16
    lengths = [3 * page + 5, page - 3]
    table, pages = make_table(2, 4, 41)
    cache = make_cache(pages, heads, dim, page, cuda_device, 42, 96, 112)
    q = torch.randn(2, queries, heads * group * dim, generator=torch.Generator().manual_seed(43)).to(dtype)
    kept = table.clone()
    kept[0, :3] = table[0, [0, 2, 3]]
    ref = reference(q, cache, kept, [2 * page + 5, 0], group, dim ** -0.5, False)
    holes = table.clone()
    holes[0, 1], holes[1, 0] = lost, lost
    got = kv_cache.kv_attention(q.to(cuda_device), cache, holes.to(cuda_device), ints(lengths, cuda_device),
                                scale=dim ** -0.5)
    assert _lib.device_status(reset=True) == 2
    check_attention(got, ref, dtype)
    got = kv_cache.kv_attention(q.to(cuda_device), cache, table.to(cuda_device), ints([4 * page + 1, -1], cuda_device),
                                scale=dim ** -0.5)
    assert _lib.device_status(reset=True) == 2
    check_attention(got, reference(q, cache, table, [4 * page, 0], group, dim ** -0.5, False), dtype)


@pytest.mark.parametrize("queries", [1, 9, 100])
def test_attention_extremes(cuda_device, queries):
    """The largest and the smallest scales, a negative score scale, bf16 queries past f16's range and near zero."""
    heads, dim, page, n = 1, 64, 16, 160
    table, pages = make_table(2, 10, 5)
    g = torch.Generator().manual_seed(7)
    for low, high, size, scale in ((1, 9, 1.0, 64.0), (192, 199, 1.0, 1e-4), (96, 112, 1e30, 1e-31), (96, 112, 1e-36, 1e34),
                                   (96, 112, 1.0, -0.125), (1, 199, 1.0, 1e-5)):
        cache = make_cache(pages, heads, dim, page, cuda_device, 6, low, high)
        q = (size * torch.randn(2, queries, dim, generator=g)).to(torch.bfloat16)
        q[:, :, 3] *= 2.0 ** -12  # channels far below the row's largest are exact too
        got = kv_cache.kv_attention(q.to(cuda_device), cache, table.to(cuda_device), ints([n, 33], cuda_device),
                                    scale=scale)
        check_attention(got, reference(q, cache, table, [n, 33], 1, scale, False), torch.bfloat16)


def test_attention_shared_pages_strides_and_streams(cuda_device):
    heads, group, dim, page, n = 2, 2, 32, 64, 100
    table, pages = make_table(1, 2, 5)
    table = table.expand(3, 2).contiguous()  # three items read one context
    wide_table = torch.full((3, 7), -5, dtype=torch.int32)
    wide_table[:, :2] = table
    cache = make_cache(pages, heads, dim, page, cuda_device, 6, 96, 112)
    width = heads * group * dim
    for queries in (9, 40):
        wide = torch.randn(3, queries, 3 * width + 7, generator=torch.Generator().manual_seed(8)).to(torch.float16)
        for lo in (width, 3):
            q = wide[..., lo: lo + width]
            ref = reference(q.reshape(3, queries, width), cache, table, [n, n, 50], group, 0.2, False)
            out = torch.full((3, queries, 2 * width + 1), 5.0, dtype=torch.float16, device=cuda_device)
            dev = wide.to(cuda_device)[..., lo: lo + width]
            side = torch.cuda.Stream()
            tab, lengths = wide_table.to(cuda_device)[:, :2], ints([n, n, 50], cuda_device)
            side.wait_stream(torch.cuda.current_stream())
            with torch.cuda.stream(side):
                kv_cache.kv_attention(dev, cache, tab, lengths, scale=0.2, out=out[..., 1: width + 1])
            torch.cuda.current_stream().wait_stream(side)
            check_attention(out[..., 1: width + 1], ref, torch.float16)
            assert (out[..., 0] == 5).all() and (out[..., width + 1:] == 5).all()


def test_more_pairs_than_warps_and_pairs_of_many_parts(cuda_device):
    """Many short items, among them idle ones, and one long item whose tiles all warps share."""
    for lengths, heads, dim, queries in (([i % 90 for i in range(700)], 2, 64, 1), ([5000], 1, 128, 1), ([20011], 1, 32, 3)):
        table, pages = make_table(len(lengths), -(-max(lengths) // 64), 5)
        cache = make_cache(pages, heads, dim, 64, cuda_device, 6, 96, 112)
        q = torch.randn(len(lengths), queries, heads * dim, generator=torch.Generator().manual_seed(8)).to(torch.bfloat16)
        got = kv_cache.kv_attention(q.to(cuda_device), cache, table.to(cuda_device), ints(lengths, cuda_device),
                                    scale=0.2, causal=True)
        check_attention(got, reference(q, cache, table, lengths, 1, 0.2, True), torch.bfloat16)


def test_written_read_and_attended_in_one_graph(cuda_device):
    """A decoding step's calls together, captured once and replayed for token after token."""
    heads, group, dim, page, batch, dtype = 2, 2, 64, 32, 3, torch.bfloat16
    table, pages = make_table(batch, 4, 5)
    cache = make_cache(pages, heads, dim, page, cuda_device, 6)
    want = host(cache)
    lengths = [0, 31, 60]
    at, tab = ints(lengths, cuda_device), table.to(cuda_device)
    k, v = (torch.zeros(batch, 1, heads * dim, dtype=dtype, device=cuda_device) for _ in range(2))
    q = torch.zeros(batch, 1, heads * group * dim, dtype=dtype, device=cuda_device)

    def step():
        kv_cache.kv_append(cache, k, v, tab, at)
        after = at + 1
        out = kv_cache.kv_attention(q, cache, tab, after, scale=0.125, causal=True)
        rows = kv_cache.kv_read(cache, tab, after, tokens=1, start=at, dtype=dtype)
        at.copy_(after)
        return out, rows

    saved = [t.clone() for t in cache]
    step()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out, rows = step()
    for t, s in zip(cache, saved):
        t.copy_(s)
    at.copy_(ints(lengths, cuda_device))
    g = torch.Generator().manual_seed(9)
    for _ in range(5):
        new = [torch.randn(t.shape, generator=g).to(dtype) for t in (k, v, q)]
        for t, x in zip((k, v, q), new):
            t.copy_(x)
        graph.replay()
        torch.cuda.synchronize()
        append_both(want, new[0], new[1], table, lengths, [1] * batch)
        lengths = [n + 1 for n in lengths]
        same_cache(cache, want)
        ref = reference(new[2], cache, table, lengths, group, 0.125, True)
        check_attention(out, ref, dtype)
        for got, x in zip(rows, (oracle.values(want[0], want[2]), oracle.values(want[1], want[3]))):
            for b, n in enumerate(lengths):
                assert torch.equal(got[b, 0].cpu().double(), oracle.rows(x, table, b, n)[:, -1].flatten())


@pytest.mark.parametrize("queries", [1, 20, 70])
def test_pages_past_32_bits(cuda_device, queries):
    heads, dim, page, tokens = 8, 128, 128, 300
    pages = 2 ** 32 // (heads * dim // 2 * page) + 9
    cache = kv_cache.KvCacheInt4.empty(pages, heads, dim, page=page, device=cuda_device)
    assert cache.k.numel() > 2 ** 32
    used = [pages - 1, 0, pages - 6]
    table = torch.tensor([used], dtype=torch.int32)
    g = torch.Generator().manual_seed(queries)
    k, v = (torch.randn(1, tokens, heads * dim, generator=g).to(torch.bfloat16) for _ in range(2))
    start = ints([0], cuda_device)
    for t in cache:
        t[used] = 0
    kv_cache.kv_append(cache, k.to(cuda_device), v.to(cuda_device), table.to(cuda_device), start)
    small = kv_cache.KvCacheInt4(*(t[used] for t in cache))
    near = torch.arange(len(used), dtype=torch.int32)[None]
    want = [torch.zeros_like(t) for t in host(small)]
    append_both(want, k, v, near, [0], [tokens])
    same_cache(small, want)
    rows = kv_cache.kv_read(cache, table.to(cuda_device), start + tokens, tokens=tokens, dtype=torch.float32)
    assert torch.equal(rows[1][0].cpu().double(),
                       oracle.rows(oracle.values(want[1], want[3]), near, 0, tokens).transpose(0, 1).flatten(1))
    q = torch.randn(1, queries, heads * dim, generator=g).to(torch.bfloat16)
    got = kv_cache.kv_attention(q.to(cuda_device), cache, table.to(cuda_device), start + tokens, scale=dim ** -0.5,
                                causal=True)
    check_attention(got, reference(q, small, near, [tokens], 1, dim ** -0.5, True), torch.bfloat16)
    assert _lib.device_status(reset=True) == 0


def test_refusals(cuda_device):
    cache = make_cache(4, 2, 64, 32, cuda_device, 1)
    table, one = ints([[0, 1]], cuda_device), ints([3], cuda_device)
    q = torch.zeros(1, 2, 128, device=cuda_device, dtype=torch.float16)
    for call, text in ((lambda: kv_cache.kv_attention(q.float(), cache, table, one, scale=1.0), "float16 or bfloat16"),
                       (lambda: kv_cache.kv_attention(q[..., :64], cache, table, one, scale=1.0), "queries must be"),
                       (lambda: kv_cache.kv_append(cache, q[..., :64], q[..., :64], table, one), "k and v must be"),
                       (lambda: kv_cache.kv_read(cache, table, one.long(), tokens=3), "lengths"),
                       (lambda: kv_cache.kv_read(cache, table[0], one, tokens=3), "table"),
                       (lambda: kv_cache.kv_read(cache, table, one, tokens=-1), "tokens"),
                       (lambda: kv_cache.kv_read(cache, table, one, tokens=2 ** 31), "tokens"),
                       (lambda: kv_cache.kv_attention(q, cache, table, one, scale=None), "kv_attention"),
                       (lambda: kv_cache.kv_read(cache, table, one, tokens=1, dtype=torch.int32), "dtype"),
                       (lambda: kv_cache.kv_read(cache, table, one, tokens=3, start=one.long()), "start"),
                       (lambda: kv_cache.kv_read(cache, table, one, tokens=3, out=(q, q)), "out must")):
        with pytest.raises(ValueError, match=text):
            call()
    with pytest.raises(_lib.LdbError, match="stride"):
        x = torch.zeros(2, 1, 128, device=cuda_device, dtype=torch.float16)[:1].expand(2, 1, 128)
        kv_cache.kv_read(cache, ints([[0], [1]], cuda_device), ints([3, 3], cuda_device), tokens=1, out=(x, x))
