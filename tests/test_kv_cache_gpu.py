"""Paged 8-bit key/value cache against its definition in 64 bits.

Appending is exact (bitwise).  Attention, per output value: the scores
accumulate in FP32, 8 * 2^-23 of their terms' magnitudes, which moves a weight
by that much relative; exponential, sum and division add 2^-18 relative; a weight is rounded to
f16, 2^-11 relative or 2^-25 of the largest weighted scale; the output is
rounded once."""

from __future__ import annotations

import pytest
import torch

from lesiondiffusion_mlx_b200 import _lib, kv_cache
from lesiondiffusion_mlx_b200.fp8 import CODES, SCALES
from oracle import kv_cache as oracle

pytestmark = pytest.mark.gpu

UNIT = {torch.float16: 2.0 ** -11, torch.bfloat16: 2.0 ** -8}
TINY = {torch.float16: 2.0 ** -25, torch.bfloat16: 0.0}


def make_cache(pages, heads, dim, page, device, seed, low=-9, high=-5):
    g = torch.Generator().manual_seed(seed)
    codes = [(60 * torch.randn(pages, heads, page, dim, generator=g)).clamp(-448, 448).to(CODES).to(device)
             for _ in range(2)]
    scales = [(torch.randint(low, high, (pages, heads), generator=g) + 127).to(torch.uint8).view(SCALES).to(device)
              for _ in range(2)]
    return kv_cache.KvCacheFp8(*codes, *scales)


def host(cache):
    return [cache.k.cpu().double(), cache.k_scale.view(torch.uint8).cpu().long() - 127,
            cache.v.cpu().double(), cache.v_scale.view(torch.uint8).cpu().long() - 127]


def make_table(batch, width, device, seed, spare=3):
    g = torch.Generator().manual_seed(seed)
    pages = batch * width + spare
    return torch.randperm(pages, generator=g)[: batch * width].view(batch, width).to(torch.int32), pages


def ints(values, device):
    return torch.tensor(values, dtype=torch.int32, device=device)


def same_cache(cache, want):
    for got, ref in zip(host(cache), want):
        assert torch.equal(torch.isnan(got.double()), torch.isnan(ref.double()))
        assert torch.equal(got.double().nan_to_num(0.0), ref.double().nan_to_num(0.0))


@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16, torch.float32])
@pytest.mark.parametrize("heads,dim,page,tokens,start", [
    (1, 64, 64, 1, [0, 1, 63, 64, 100]), (2, 128, 128, 130, [0, 5, 127]), (3, 32, 16, 40, [0, 15, 16, 7]),
    (2, 64, 32, 33, [31, 0]), (1, 128, 16, 1, [15]), (8, 128, 64, 200, [70])])
def test_append_is_exact(cuda_device, dtype, heads, dim, page, tokens, start):
    batch = len(start)
    width = (max(start) + tokens + page - 1) // page + 1
    table, pages = make_table(batch, width, cuda_device, 3)
    cache = make_cache(pages, heads, dim, page, cuda_device, 4)
    want = host(cache)
    g = torch.Generator().manual_seed(5)
    k, v = (torch.randn(batch, tokens, heads * dim, generator=g).to(dtype) for _ in range(2))
    for b in range(batch):  # some items need a larger scale than the page has, some a smaller one
        k[b] *= 2.0 ** (2 * b - 3)
    kv_cache.kv_append(cache, k.to(cuda_device), v.to(cuda_device), table.to(cuda_device), ints(start, cuda_device))
    for (codes, e), new in zip(((want[0], want[1]), (want[2], want[3])), (k, v)):
        oracle.append(codes, e, new.view(batch, tokens, heads, dim), table, start, [tokens] * batch)
    same_cache(cache, want)
    kv_cache.kv_append(cache, k.to(cuda_device), v.to(cuda_device), table.to(cuda_device), ints(start, cuda_device))
    same_cache(cache, want)  # the same tokens at the same place again change nothing
    assert _lib.device_status(reset=True) == 0


def test_append_token_by_token_and_counts(cuda_device):
    """Pages filled one token at a time, items that get fewer tokens (or none), zeros, NaN and infinity."""
    heads, dim, page, batch = 2, 32, 16, 3
    table, pages = make_table(batch, 4, cuda_device, 7)
    cache = make_cache(pages, heads, dim, page, cuda_device, 8)
    want = host(cache)
    g = torch.Generator().manual_seed(9)
    at = [0, 14, 40]
    for step in range(20):
        k, v = (torch.randn(batch, 2, heads * dim, generator=g) * 2.0 ** (step % 7 - 3) for _ in range(2))
        if step == 4:
            k[0], v[0, 0, 3], k[1, 0, 5] = 0, float("nan"), float("inf")
        counts = [1, step % 3, 0 if step % 2 else 2]
        counts[2] = min(counts[2], 64 - at[2])
        kv_cache.kv_append(cache, k.to(cuda_device), v.to(cuda_device), table.to(cuda_device), ints(at, cuda_device),
                           counts=ints(counts, cuda_device))
        for (codes, e), new in zip(((want[0], want[1]), (want[2], want[3])), (k, v)):
            oracle.append(codes, e, new.view(batch, 2, heads, dim), table, at, counts)
        at = [a + c for a, c in zip(at, counts)]
        same_cache(cache, want)
    assert _lib.device_status(reset=True) == 0


def test_append_strided_and_out_of_range(cuda_device):
    """Channel slices of a fused projection at odd offsets; positions and pages outside the cache are
    reported and leave every page as it was."""
    heads, dim, page, batch = 2, 64, 32, 2
    table, pages = make_table(batch, 3, cuda_device, 1)
    cache = make_cache(pages, heads, dim, page, cuda_device, 2)
    want = host(cache)
    wide = torch.randn(batch, 9, 3 * heads * dim + 5, generator=torch.Generator().manual_seed(3)).to(torch.bfloat16)
    k, v = wide[..., 128:256], wide[..., 261:389]
    dev = wide.to(cuda_device)
    kv_cache.kv_append(cache, dev[..., 128:256], dev[..., 261:389], table.to(cuda_device), ints([4, 30], cuda_device))
    for (codes, e), new in zip(((want[0], want[1]), (want[2], want[3])), (k, v)):
        oracle.append(codes, e, new.reshape(batch, 9, heads, dim), table, [4, 30], [9, 9])
    same_cache(cache, want)
    assert _lib.device_status(reset=True) == 0
    lost = table.clone()
    lost[0, 0], lost[1, 0] = pages, -1
    for tab, start in ((lost, [0, 0]), (table, [96, 1000]), (table, [-1, -40])):
        kv_cache.kv_append(cache, dev[..., 128:256], dev[..., 261:389], tab.to(cuda_device), ints(start, cuda_device))
        assert _lib.device_status(reset=True) == 2
    same_cache(cache, want)


def check_attention(got, ref, dtype):
    bound = ((2.0 ** -11 + 2.0 ** -18 + 2 * 8 * 2.0 ** -23 * ref["score"]) * ref["size"]
             + 448 * 2.0 ** -25 * ref["peak"] + UNIT[dtype] * ref["out"].abs() * (1 + 2.0 ** -8) + TINY[dtype])
    err = (got.cpu().double().view(ref["out"].shape) - ref["out"]).abs()
    assert (err <= bound).all(), float((err / bound.clamp(min=1e-300)).max())


CASES = [  # lengths, queries, kv heads, group, dim, page, causal
    ([1], 1, 1, 1, 64, 64, False), ([0, 3, 64, 65, 200], 1, 2, 4, 128, 64, True), ([77], 50, 4, 1, 64, 64, False),
    ([129, 17], 5, 1, 3, 32, 16, True), ([40, 0, 7], 12, 2, 2, 64, 32, True), ([300], 1, 1, 16, 128, 128, False),
    ([500, 30], 1, 1, 17, 64, 128, False), ([1500], 1, 2, 1, 128, 16, False), ([260], 130, 1, 2, 128, 64, True),
    ([5], 30, 1, 8, 32, 64, True), ([200, 128, 1], 64, 2, 4, 128, 128, True), ([333], 300, 1, 1, 64, 16, False)]


@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
@pytest.mark.parametrize("lengths,queries,heads,group,dim,page,causal", CASES)
def test_attention(cuda_device, dtype, lengths, queries, heads, group, dim, page, causal):
    batch = len(lengths)
    table, pages = make_table(batch, -(-max(lengths) // page) + 1, cuda_device, 11)
    cache = make_cache(pages, heads, dim, page, cuda_device, 12)
    want = host(cache)
    # everything the lengths leave out holds NaN: the tails of last pages, and the pages nobody owns
    owned = set()
    for b, n in enumerate(lengths):
        for slot in range(-(-n // page)):
            owned.add(int(table[b, slot]))
            tail = n - slot * page
            if tail < page:
                for t in (cache.k, cache.v):
                    t.view(torch.uint8)[int(table[b, slot]), :, tail:] = 0x7F
    for at in set(range(pages)) - owned:
        for t in (cache.k, cache.v):
            t.view(torch.uint8)[at] = 0xFF
    q = 2 * torch.randn(batch, queries, heads * group * dim, generator=torch.Generator().manual_seed(13))
    q = q.to(dtype)
    got = kv_cache.kv_attention(q.to(cuda_device), cache, table.to(cuda_device), ints(lengths, cuda_device),
                                scale=dim ** -0.5, causal=causal)
    ref = oracle.attention(q, *want, table, lengths, group, dim ** -0.5, causal)
    check_attention(got, ref, dtype)
    again = kv_cache.kv_attention(q.to(cuda_device), cache, table.to(cuda_device), ints(lengths, cuda_device),
                                  scale=dim ** -0.5, causal=causal)
    assert torch.equal(again, got)
    assert _lib.device_status(reset=True) == 0


@pytest.mark.parametrize("queries", [1, 3, 70])
def test_attention_future_nan_does_not_reach_the_past(cuda_device, queries):
    """NaN keys and values in the last token: only the queries that see it become NaN."""
    heads, dim, page, n = 2, 64, 32, 150
    table, pages = make_table(1, 5, cuda_device, 2)
    cache = make_cache(pages, heads, dim, page, cuda_device, 3)
    want = host(cache)
    q = torch.randn(1, queries, heads * dim, generator=torch.Generator().manual_seed(4)).to(torch.float16)
    ref = oracle.attention(q, *want, table, [n], 1, 0.125, True)
    at, slot = int(table[0, (n - 1) // page]), (n - 1) % page
    for which in (cache.k, cache.v):
        kept = which.view(torch.uint8)[at, :, slot].clone()
        which.view(torch.uint8)[at, :, slot, 7] = 0x7F
        got = kv_cache.kv_attention(q.to(cuda_device), cache, table.to(cuda_device), ints([n], cuda_device),
                                    scale=0.125, causal=True)
        assert torch.isnan(got[:, -1].view(heads, dim)[:, 7]).all()
        if queries > 1:
            check_attention(got[:, :-1], {k: x[:, :-1] for k, x in ref.items()}, torch.float16)
        which.view(torch.uint8)[at, :, slot] = kept


def test_attention_scale_extremes(cuda_device):
    """Pages whose scales lie far apart, keys that dwarf the rest, bf16 queries past f16's range."""
    heads, dim, page, n = 1, 64, 16, 160
    table, pages = make_table(2, 10, cuda_device, 5)
    cache = make_cache(pages, heads, dim, page, cuda_device, 6, low=-30, high=12)
    k_e = cache.k_scale.view(torch.uint8)
    k_e.copy_(torch.full_like(k_e, 127 - 9))
    want = host(cache)
    q = torch.randn(2, 4, dim, generator=torch.Generator().manual_seed(7))
    q[1] *= 1e6
    for dtype, scale in ((torch.bfloat16, 0.125), (torch.bfloat16, 1e-6)):
        ref = oracle.attention(q.to(dtype), *want, table, [n, 33], 1, scale, False)
        got = kv_cache.kv_attention(q.to(cuda_device, dtype), cache, table.to(cuda_device),
                                    ints([n, 33], cuda_device), scale=scale)
        keep = slice(0, 1) if scale == 0.125 else slice(0, 2)  # 1e6 * 0.125: a hard maximum, beyond any bound
        check_attention(got[keep], {k: x[keep] for k, x in ref.items()}, dtype)
        assert torch.isfinite(got).all()


def test_attention_shared_pages_strides_and_streams(cuda_device):
    heads, group, dim, page, n = 2, 2, 32, 64, 100
    table, pages = make_table(1, 2, cuda_device, 5)
    table = table.expand(3, 2).contiguous()  # three items read one context
    wide_table = torch.full((3, 7), -5, dtype=torch.int32)
    wide_table[:, :2] = table
    cache = make_cache(pages, heads, dim, page, cuda_device, 6)
    want = host(cache)
    width = heads * group * dim
    wide = torch.randn(3, 9, 3 * width + 7, generator=torch.Generator().manual_seed(8)).to(torch.float16)
    for lo in (width, 3):
        q = wide[..., lo : lo + width]
        ref = oracle.attention(q.reshape(3, 9, width), *want, table, [n, n, 50], group, 0.2, False)
        out = torch.full((3, 9, 2 * width + 1), 5.0, dtype=torch.float16, device=cuda_device)
        dev = wide.to(cuda_device)[..., lo : lo + width]
        side = torch.cuda.Stream()
        tab, lengths = wide_table.to(cuda_device)[:, :2], ints([n, n, 50], cuda_device)
        side.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(side):
            kv_cache.kv_attention(dev, cache, tab, lengths, scale=0.2, out=out[..., 1 : width + 1])
        torch.cuda.current_stream().wait_stream(side)
        check_attention(out[..., 1 : width + 1], ref, torch.float16)
        assert (out[..., 0] == 5).all() and (out[..., width + 1 :] == 5).all()


def test_attention_reports_what_lies_outside(cuda_device):
    """Page numbers and lengths outside the cache: a status bit, no access outside, other items as they were."""
    heads, dim, page = 1, 64, 64
    table, pages = make_table(2, 3, cuda_device, 5)
    cache = make_cache(pages, heads, dim, page, cuda_device, 6)
    q = torch.randn(2, 3, dim, generator=torch.Generator().manual_seed(7)).to(torch.float16)
    ref = oracle.attention(q, *host(cache), table, [150, 150], 1, 0.125, False)
    for bad, lengths in ((pages, [150, 150]), (-1, [150, 150]), (1 << 30, [150, 150]), (None, [150, 193]), (None, [150, -1])):
        tab = table.clone()
        if bad is not None:
            tab[1, 1] = bad
        got = kv_cache.kv_attention(q.to(cuda_device), cache, tab.to(cuda_device), ints(lengths, cuda_device), scale=0.125)
        check_attention(got[:1], {k: x[:1] for k, x in ref.items()}, torch.float16)
        assert _lib.device_status(reset=True) == 2


def test_refusals(cuda_device):
    cache = make_cache(4, 2, 64, 32, cuda_device, 1)
    table, one = ints([[0, 1]], cuda_device), ints([3], cuda_device)
    q = torch.zeros(1, 2, 128, device=cuda_device, dtype=torch.float16)
    with pytest.raises(ValueError, match="float16 or bfloat16"):
        kv_cache.kv_attention(q.float(), cache, table, one, scale=1.0)
    with pytest.raises(ValueError, match="queries must be"):
        kv_cache.kv_attention(q[..., :64], cache, table, one, scale=1.0)
    with pytest.raises(ValueError, match="lengths"):
        kv_cache.kv_attention(q, cache, table, one.long(), scale=1.0)
    with pytest.raises(ValueError, match="table"):
        kv_cache.kv_attention(q, cache, table[0], one, scale=1.0)
    with pytest.raises(ValueError, match="out must"):
        kv_cache.kv_attention(q, cache, table, one, scale=1.0, out=q.float())
    with pytest.raises(ValueError, match="k and v must be"):
        kv_cache.kv_append(cache, q[..., :64], q[..., :64], table, one)
    with pytest.raises(ValueError, match="counts"):
        kv_cache.kv_append(cache, q, q, table, one, counts=ints([1, 1], cuda_device))
    with pytest.raises(ValueError, match="share dtype"):
        kv_cache.kv_append(cache, q, q.float(), table, one)


@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
@pytest.mark.parametrize("causal", [False, True])
@pytest.mark.parametrize("queries,group,dim,page", [(1, 4, 128, 64), (5, 2, 64, 16), (12, 1, 32, 32), (7, 2, 128, 128),
                                                    (70, 1, 64, 64), (130, 2, 128, 16), (300, 1, 32, 128)])
def test_attention_nan_values_stay_in_their_channel(cuda_device, dtype, causal, queries, group, dim, page):
    """NaN values in tokens that all, some or none of the queries see: exactly the formula's outputs are NaN."""
    heads, lengths = 2, [310, 37]
    table, pages = make_table(2, 320 // page + 1, cuda_device, 21)
    cache = make_cache(pages, heads, dim, page, cuda_device, 22)
    for b, head, tok, channel, code in ((0, 0, 309, 3, 0x7F), (0, 1, 305, 0, 0xFF), (0, 1, 306, dim - 1, 0x7F),
                                        (0, 0, 290, 17, 0x7F), (0, 1, 12, 9, 0xFF), (1, 0, 36, 1, 0x7F),
                                        (1, 1, 20, 30, 0x7F)):
        cache.v.view(torch.uint8)[int(table[b, tok // page]), head, tok % page, channel] = code
    want = host(cache)
    q = torch.randn(2, queries, heads * group * dim, generator=torch.Generator().manual_seed(23)).to(dtype)
    ref = oracle.attention(q, *want, table, lengths, group, dim ** -0.5, causal)
    got = kv_cache.kv_attention(q.to(cuda_device), cache, table.to(cuda_device), ints(lengths, cuda_device),
                                scale=dim ** -0.5, causal=causal)
    nan = torch.isnan(ref["out"])
    assert nan.any() and not nan.all()
    assert torch.equal(torch.isnan(got.cpu().view(nan.shape)), nan)
    finite = {k: torch.where(torch.isnan(x), torch.zeros_like(x), x) for k, x in ref.items()}
    check_attention(torch.where(nan.to(cuda_device), 0.0, got.view(nan.shape)), finite, dtype)


@pytest.mark.parametrize("queries", [9, 60, 200])
@pytest.mark.parametrize("value", [float("inf"), float("-inf"), float("nan")])
def test_attention_queries_without_keys_are_zero_whatever_they_hold(cuda_device, queries, value):
    heads, dim, page, n = 1, 64, 64, 6  # the first queries - 6 queries see nothing
    table, pages = make_table(1, 1, cuda_device, 31)
    cache = make_cache(pages, heads, dim, page, cuda_device, 32)
    q = torch.randn(1, queries, dim, generator=torch.Generator().manual_seed(33)).to(torch.float16)
    ref = oracle.attention(q, *host(cache), table, [n], 1, 0.125, True)
    q[0, 1, 5] = value
    got = kv_cache.kv_attention(q.to(cuda_device), cache, table.to(cuda_device), ints([n], cuda_device), scale=0.125,
                                causal=True)
    assert (got[0, : queries - n] == 0).all()
    check_attention(got, ref, torch.float16)
    q[0, -2, 5] = value  # one that sees keys becomes NaN, and no other does
    got = kv_cache.kv_attention(q.to(cuda_device), cache, table.to(cuda_device), ints([n], cuda_device), scale=0.125,
                                causal=True)
    assert torch.isnan(got[0, -2]).all()
    rest = [i for i in range(queries) if i != queries - 2]
    check_attention(got[:, rest], {k: x[:, rest] for k, x in ref.items()}, torch.float16)


@pytest.mark.parametrize("queries,group,dim,page", [(1, 4, 128, 64), (3, 1, 64, 16), (3, 4, 32, 32), (20, 2, 128, 128),
                                                    (90, 1, 64, 16), (130, 2, 128, 64), (64, 1, 32, 128)])
@pytest.mark.parametrize("lost", [-1, 1 << 20])
def test_attention_leaves_out_pages_outside_the_cache(cuda_device, queries, group, dim, page, lost):
    """The result without the tokens of such a page, and a status bit; an item with no other page gives zeros."""
    heads, dtype = 2, torch.bfloat16
    lengths = [3 * page + 5, page - 3]
    table, pages = make_table(2, 4, cuda_device, 41)
    cache = make_cache(pages, heads, dim, page, cuda_device, 42)
    q = torch.randn(2, queries, heads * group * dim, generator=torch.Generator().manual_seed(43)).to(dtype)
    kept = table.clone()
    kept[0, :3] = table[0, [0, 2, 3]]
    ref = oracle.attention(q, *host(cache), kept, [2 * page + 5, 0], group, dim ** -0.5, False)
    holes = table.clone()
    holes[0, 1], holes[1, 0] = lost, lost
    got = kv_cache.kv_attention(q.to(cuda_device), cache, holes.to(cuda_device), ints(lengths, cuda_device),
                                scale=dim ** -0.5)
    assert _lib.device_status(reset=True) == 2
    check_attention(got, ref, dtype)


def test_attention_refuses_items_that_overlap_in_the_output(cuda_device):
    cache = make_cache(4, 1, 64, 32, cuda_device, 1)
    table, lengths = ints([[0], [1]], cuda_device), ints([3, 3], cuda_device)
    q = torch.zeros(2, 1, 64, device=cuda_device, dtype=torch.float16)
    with pytest.raises(_lib.LdbError, match="item stride"):
        kv_cache.kv_attention(q, cache, table, lengths, scale=1.0, out=q[:1].expand(2, 1, 64))


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("page", [16, 32, 64, 128])
@pytest.mark.parametrize("dim", [32, 64, 128])
def test_append_every_page_size(cuda_device, dtype, dim, page):
    """Each page of each head width, over older tokens, with a short item, three heads and an infinity."""
    heads, tokens, start, counts = 3, 2 * page + 5, [0, page - 1, 7], [2 * page + 5, page + 3, 0]
    table, pages = make_table(3, 4, cuda_device, dim + page)
    cache = make_cache(pages, heads, dim, page, cuda_device, page)
    want = host(cache)
    g = torch.Generator().manual_seed(dim)
    k, v = (torch.randn(3, tokens, heads * dim, generator=g) for _ in range(2))
    k[1] *= 64
    v[0, 3, 5] = float("inf")
    k, v = k.to(dtype), v.to(dtype)
    kv_cache.kv_append(cache, k.to(cuda_device), v.to(cuda_device), table.to(cuda_device), ints(start, cuda_device),
                       counts=ints(counts, cuda_device))
    for (codes, e), new in zip(((want[0], want[1]), (want[2], want[3])), (k, v)):
        oracle.append(codes, e, new.view(3, tokens, heads, dim), table, start, counts)
    same_cache(cache, want)
    assert _lib.device_status(reset=True) == 0
