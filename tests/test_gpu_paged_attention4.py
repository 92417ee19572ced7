"""cb_paged_attention4 against attention in 64 bits over the values that the pages hold.

Bound, per output with probabilities p_j (exact), values v_j = low_j + step_j c_j and
u = eps / 2 of the output type:

* a factor p step' is rounded to fp16: 2^-11 relative, so at most 2^-11 sum p step' c
  (below 2^-14 it is a subnormal: the reference keeps the largest of a call's factors
  over 2^-5, so such a factor is off by 2^-25 / 2^-5 = 2^-20 of the largest p step',
  which over n keys is at most n 2^-20 15 max(p step'));
* exp2, the fp32 sums and the logits: a logit is a sum of 2 x 64 products over fp32 with
  terms of size A = scale log2e sum |q| |k| (codes and lowest value apart), off by at most
  2^-24 (128 + 8) A, which changes p by that much relative: 2^-16 A;
* the result is rounded once: u |out|.

    |got - want| <= u |want| + (2^-11 + 2^-15 A) sum p (step c + |low|) + n 2^-16 max(p step) + tiny
"""

from __future__ import annotations

import math

import pytest
import torch

from cacheblend_b200 import PagedKV4, append_paged_kv4, gather_paged_kv4, paged_attention4
from cacheblend_b200.attention import paged_attention4_workspace_bytes

pytestmark = pytest.mark.gpu


def _pages(device, lens, block, kv_heads, head, seed, step=(0.15, 0.35), low=(-2.7, -1.2), spare=2):
    """(cache with random pages, block table) for sequences of ``lens`` keys."""
    gen = torch.Generator().manual_seed(seed)
    pages = [-(-n // block) for n in lens]
    blocks = sum(pages) + spare
    order = torch.randperm(blocks, generator=gen).to(torch.int32)
    table = torch.full((len(lens), max(max(pages), 1) + 1), -1, dtype=torch.int32)  # unused entries are padding
    at = 0
    for i, n in enumerate(pages):
        table[i, :n] = order[at:at + n]
        at += n
    codes = torch.randint(0, 256, (2, blocks, kv_heads, block, head // 2), generator=gen, dtype=torch.uint8)
    pairs = torch.rand(2, blocks, kv_heads, block, head // 64, 2, generator=gen)
    pairs[..., 0] = step[0] + pairs[..., 0] * (step[1] - step[0])
    pairs[..., 1] = low[0] + pairs[..., 1] * (low[1] - low[0])
    pairs = pairs.half()
    for i, n in enumerate(lens):  # rows behind a sequence's end: whatever memory held
        if n % block:
            pairs[:, table[i, n // block], :, n % block:] = torch.nan
            codes[:, table[i, n // block], :, n % block:] = 255
    return PagedKV4(codes.to(device), pairs.to(device)), table.to(device)


def _parts(cache, table_row, n, plane):
    """(step * code, low) in 64 bits, [n, kv_heads, head]."""
    block = cache.block_size
    pages = table_row[:-(-n // block)].long()
    codes = cache.codes[plane][pages]
    codes = torch.stack((codes & 15, codes >> 4), -1).flatten(-2).double().unflatten(-1, (-1, 64))
    pair = cache.scales[plane][pages].double()
    varied, low = codes * pair[..., :1], pair[..., 1:].expand_as(codes)
    order = lambda x: x.flatten(-2).transpose(1, 2).flatten(0, 1)[:n]  # noqa: E731
    return order(varied), order(low)


def _check(got, query, cache, table, lens, scale, start=None):
    groups = query.shape[1] // cache.num_heads
    info = torch.finfo(query.dtype)
    worst = 0.0
    for i, n in enumerate(lens):
        a, b = (start[i], start[i + 1]) if start is not None else (i, i + 1)
        if n == 0:
            assert int((got[a:b] != 0).sum()) == 0
            continue
        kv, kl = _parts(cache, table[i], n, 0)
        vv, vl = _parts(cache, table[i], n, 1)
        for j in range(a, b):
            seen = n - (b - a) + (j - a) + 1
            if seen <= 0:
                assert int((got[j] != 0).sum()) == 0
                continue
            q = query[j].double().unflatten(0, (cache.num_heads, groups))
            w = torch.einsum("hgd,lhd->hgl", q, kv[:seen] + kl[:seen]) * scale
            size = torch.einsum("hgd,lhd->hgl", q.abs(), kv[:seen] + kl[:seen].abs()).amax(-1) * abs(scale) * math.log2(math.e)
            p = torch.softmax(w, -1)
            want = torch.einsum("hgl,lhd->hgd", p, vv[:seen] + vl[:seen])
            mass = torch.einsum("hgl,lhd->hgd", p, vv[:seen] + vl[:seen].abs())
            largest = torch.einsum("hgl,lhd->hgld", p, vv[:seen]).amax(2)
            bound = want.abs() * (info.eps / 2) + (2.0 ** -11 + 2.0 ** -15 * size[..., None]) * mass \
                + seen * 2.0 ** -20 * largest + info.smallest_normal
            off = (got[j].double().unflatten(0, (cache.num_heads, groups)) - want).abs()
            worst = max(worst, float((off / bound).max()))
    assert worst <= 1, worst


CASES = [
    # lens, block, heads, kv_heads, head, dtype, tokens per sequence
    ([1], 16, 32, 8, 128, torch.bfloat16, None),
    ([0, 1, 31, 32, 33, 0], 16, 8, 2, 128, torch.float16, None),
    ([1000], 16, 8, 1, 64, torch.bfloat16, None),
    ([257, 5, 4100, 63], 24, 28, 4, 128, torch.bfloat16, None),      # groups of 7, pages that end inside a tile
    ([700, 64], 1, 5, 5, 64, torch.float16, None),                   # one head a group, pages of one row
    ([2049, 100], 64, 64, 2, 128, torch.bfloat16, None),             # groups of 32: four row blocks
    ([40000], 128, 16, 2, 128, torch.bfloat16, None),
    ([300, 9, 2, 1200], 16, 16, 4, 128, torch.bfloat16, [3, 1, 5, 4]),   # more tokens than keys in one
    ([90, 0, 513], 24, 12, 4, 64, torch.float16, [17, 2, 40]),
    ([3, 60], 7, 96, 2, 128, torch.float16, [1, 2]),
]


@pytest.mark.parametrize("case", CASES, ids=str)
def test_against_64_bits(cuda, case):
    lens, block, heads, kv_heads, head, dtype, counts = case
    cache, table = _pages(cuda, lens, block, kv_heads, head, 3)
    gen = torch.Generator(device=cuda).manual_seed(4)
    start = None if counts is None else [0, *torch.tensor(counts).cumsum(0).tolist()]
    total = len(lens) if counts is None else start[-1]
    query = torch.randn(total, heads, head, generator=gen, device=cuda).to(dtype)
    lengths = torch.tensor(lens, dtype=torch.int32, device=cuda)
    begin = None if start is None else torch.tensor(start, dtype=torch.int32, device=cuda)
    got = paged_attention4(query, cache, table, lengths, head ** -0.5, query_start=begin)
    _check(got, query, cache, table, lens, head ** -0.5, start)
    again = paged_attention4(query, cache, table, lengths, head ** -0.5, query_start=begin)
    assert torch.equal(got, again)


@pytest.mark.parametrize("step,low,q", [((1e-4, 3e-4), (-1e-3, 1e-3), 1.0), ((40.0, 900.0), (-8000.0, 100.0), 1e-4),
                                        ((0.0, 0.0), (-1.0, 1.0), 1.0), ((0.1, 0.2), (-1.0, 0.0), 30.0)])
def test_sizes_of_values(cuda, step, low, q):
    """Small, large and constant rows, and peaked logits."""
    lens = [1500, 40]
    cache, table = _pages(cuda, lens, 16, 2, 128, 5, step, low)
    query = (torch.randn(2, 8, 128, device=cuda, generator=torch.Generator(device=cuda).manual_seed(6)) * q).to(torch.bfloat16)
    got = paged_attention4(query, cache, table, torch.tensor(lens, dtype=torch.int32, device=cuda), 0.09)
    _check(got, query, cache, table, lens, 0.09)


def test_strides_rows_behind_and_bad_pages(cuda):
    lens, heads, head = [200, 77], 8, 128
    cache, table = _pages(cuda, lens, 16, 4, head, 7)
    wide = torch.randn(6, heads + 3, head + 1, device=cuda, generator=torch.Generator(device=cuda).manual_seed(8)).to(torch.bfloat16)
    query = wide[:, 1:1 + heads, 1:]  # rows that are not 16-byte aligned
    start = torch.tensor([1, 2, 4], dtype=torch.int32, device=cuda)
    lengths = torch.tensor(lens, dtype=torch.int32, device=cuda)
    out = torch.full((6, heads, head + 2), 5.0, device=cuda, dtype=torch.bfloat16)[..., 1:1 + head]
    got = paged_attention4(query, cache, table, lengths, head ** -0.5, query_start=start, out=out)
    assert got is out
    _check(got, query, cache, table, lens, head ** -0.5, [1, 2, 4])
    assert (got[0] == 5).all() and (got[4:] == 5).all()  # rows of no sequence
    # a page outside the cache is left out: the same as a sequence without its keys
    short = table.clone()
    short[0, -(-lens[0] // 16) - 1] = cache.num_blocks + 4
    cut = paged_attention4(query, cache, short, lengths, head ** -0.5, query_start=start)
    fewer = torch.tensor([192, 77], dtype=torch.int32, device=cuda)
    assert torch.equal(cut[2:4], got[2:4])
    same = paged_attention4(query, cache, table, fewer, head ** -0.5, query_start=start)
    assert torch.equal(cut[1], same[1])
    # lengths past the table, starts past the rows: clamped
    over = paged_attention4(query, cache, table[:, :5].contiguous(), torch.tensor([10 ** 6, 77], dtype=torch.int32, device=cuda),
                            head ** -0.5, query_start=torch.tensor([1, 2, 99], dtype=torch.int32, device=cuda))
    want = paged_attention4(query, cache, table, torch.tensor([80, 77], dtype=torch.int32, device=cuda), head ** -0.5,
                            query_start=torch.tensor([1, 2, 6], dtype=torch.int32, device=cuda))
    assert torch.equal(over[1:], want[1:])


def test_not_finite(cuda):
    """A NaN row reaches the tokens that see it and no other."""
    lens = [100]
    for plane in (0, 1):
        cache, table = _pages(cuda, lens, 16, 1, 64, 9)
        cache.scales[plane, table[0, 6], 0, 2, 0, 0] = torch.nan  # key 98
        query = torch.randn(3, 2, 64, device=cuda, generator=torch.Generator(device=cuda).manual_seed(1)).to(torch.float16)
        got = paged_attention4(query, cache, table, torch.tensor(lens, dtype=torch.int32, device=cuda), 0.125,
                               query_start=torch.tensor([0, 3], dtype=torch.int32, device=cuda))
        assert bool(got[0].isfinite().all()) and bool(got[1:].isnan().all())
    cache, table = _pages(cuda, [100, 50], 16, 1, 64, 9)
    query[0, 1] = torch.inf  # a bad query head keeps to itself
    got = paged_attention4(query[:2], cache, table, torch.tensor([100, 50], dtype=torch.int32, device=cuda), 0.125)
    assert bool(got[0, 1].isnan().all()) and bool(got[0, 0].isfinite().all()) and bool(got[1].isfinite().all())


@pytest.mark.parametrize("scale", [-0.07, 0.0])
def test_scales_that_are_not_positive(cuda, scale):
    lens = [300, 41]
    cache, table = _pages(cuda, lens, 16, 2, 128, 21)
    query = torch.randn(2, 8, 128, device=cuda, generator=torch.Generator(device=cuda).manual_seed(1)).to(torch.bfloat16)
    got = paged_attention4(query, cache, table, torch.tensor(lens, dtype=torch.int32, device=cuda), scale)
    _check(got, query, cache, table, lens, scale)


def test_empty_cache_and_no_sequences(cuda):
    """No pages at all: every sequence is empty."""
    empty = PagedKV4(torch.zeros(2, 0, 2, 16, 64, dtype=torch.uint8, device=cuda),
                     torch.zeros(2, 0, 2, 16, 2, 2, dtype=torch.float16, device=cuda))
    query = torch.randn(2, 8, 128, device=cuda).to(torch.bfloat16)
    table, lens = torch.zeros(2, 3, dtype=torch.int32, device=cuda), torch.tensor([20, 0], dtype=torch.int32, device=cuda)
    cache, _ = _pages(cuda, [20], 16, 2, 128, 1)
    with pytest.raises(ValueError, match="null page"):
        paged_attention4(query, empty, table, lens, 0.1)
    none = torch.full_like(table, cache.num_blocks)  # every page outside the cache
    assert int((paged_attention4(query, cache, none, lens, 0.1) != 0).sum()) == 0
    assert int((paged_attention4(query, cache, table[:, :0], lens, 0.1) != 0).sum()) == 0
    assert paged_attention4(query[:0], cache, table[:0], lens[:0], 0.1).shape == (0, 8, 128)


def test_calls_at_once_and_again(cuda):
    """Calls of different shapes on two streams at once, many times: always the same bits."""
    problems = []
    for seed, (lens, heads, kv_heads, head) in enumerate([([5000, 3, 900], 16, 2, 128), ([40] * 90, 8, 4, 64), ([12000], 8, 1, 128)]):
        cache, table = _pages(cuda, lens, 16, kv_heads, head, seed)
        query = torch.randn(len(lens), heads, head, device=cuda, generator=torch.Generator(device=cuda).manual_seed(seed)).to(torch.bfloat16)
        problems.append((query, cache, table, torch.tensor(lens, dtype=torch.int32, device=cuda), 0.1))
    want = [paged_attention4(*p) for p in problems]
    torch.cuda.synchronize()
    sides = [torch.cuda.Stream(cuda) for _ in range(2)]
    got = [(i, paged_attention4(*problems[i], stream=sides[n % 2])) for n in range(30) for i in range(3)]
    torch.cuda.synchronize()
    assert all(torch.equal(out, want[i]) for i, out in got)


def test_many_sequences(cuda):
    """More sequences than threads of a CTA, most of them empty or short."""
    gen = torch.Generator().manual_seed(10)
    lens = (torch.rand(700, generator=gen) ** 4 * 300).long().tolist()
    cache, table = _pages(cuda, lens, 16, 2, 64, 11)
    query = torch.randn(700, 4, 64, device=cuda, generator=torch.Generator(device=cuda).manual_seed(1)).to(torch.bfloat16)
    got = paged_attention4(query, cache, table, torch.tensor(lens, dtype=torch.int32, device=cuda), 0.125)
    _check(got, query, cache, table, lens, 0.125)


def test_offsets_past_32_bits(cuda):
    """Pages that lie past a 32-bit byte offset of the codes."""
    block, kv_heads, head = 128, 8, 128
    blocks = (1 << 32) // (block * kv_heads * head // 2) + 30
    codes = torch.empty(2, blocks, kv_heads, block, head // 2, dtype=torch.uint8, device=cuda)
    scales = torch.zeros(2, blocks, kv_heads, block, 2, 2, dtype=torch.float16, device=cuda)
    small, table = _pages(cuda, [500, 130], block, kv_heads, head, 12)
    moved = torch.where(table >= 0, table + blocks - small.num_blocks, table)
    codes[:, -small.num_blocks:], scales[:, -small.num_blocks:] = small.codes, small.scales
    query = torch.randn(2, 32, head, device=cuda, generator=torch.Generator(device=cuda).manual_seed(1)).to(torch.bfloat16)
    lengths = torch.tensor([500, 130], dtype=torch.int32, device=cuda)
    want = paged_attention4(query, small, table, lengths, head ** -0.5)
    assert torch.equal(paged_attention4(query, PagedKV4(codes, scales), moved, lengths, head ** -0.5), want)


def test_streams_workspace_and_graph(cuda):
    lens = [900, 33]
    cache, table = _pages(cuda, lens, 16, 2, 128, 13)
    query = torch.randn(2, 8, 128, device=cuda, generator=torch.Generator(device=cuda).manual_seed(1)).to(torch.bfloat16)
    lengths = torch.tensor(lens, dtype=torch.int32, device=cuda)
    want = paged_attention4(query, cache, table, lengths, 0.1)
    torch.cuda.synchronize()
    side = torch.cuda.Stream(cuda)
    got = paged_attention4(query, cache, table, lengths, 0.1, stream=side)
    side.synchronize()
    assert torch.equal(got, want)
    size = paged_attention4_workspace_bytes(2, 2, 8, 2, 128)
    dirty = torch.full((size,), 255, dtype=torch.uint8, device=cuda)
    assert torch.equal(paged_attention4(query, cache, table, lengths, 0.1, workspace=dirty), want)
    with pytest.raises(ValueError, match="workspace"):
        paged_attention4(query, cache, table, lengths, 0.1, workspace=dirty[:size - 32])
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        inside = paged_attention4(query, cache, table, lengths, 0.1)
    lengths.copy_(torch.tensor([300, 20], dtype=torch.int32))  # the next step's lengths
    graph.replay()
    torch.cuda.synchronize()
    _check(inside, query, cache, table, [300, 20], 0.1)


def test_append_then_attend(cuda):
    """A prompt and decode steps through the pages, as a serving loop makes them."""
    block, kv_heads, heads, head = 16, 2, 8, 128
    gen = torch.Generator(device=cuda).manual_seed(20)
    cache = PagedKV4.allocate(12, block, kv_heads, head, cuda)
    table = torch.tensor([[3, 0, 7, 9], [1, 11, 2, 4]], dtype=torch.int32, device=cuda)
    lens = torch.tensor([30, 7], dtype=torch.int32, device=cuda)

    def fresh(n):
        return (torch.randn(n, kv_heads, head, generator=gen, device=cuda).to(torch.bfloat16) for _ in range(2))

    for i, n in enumerate(lens.tolist()):
        k, v = fresh(n)
        at = torch.arange(n, device=cuda)
        append_paged_kv4(None, None, k, v, cache, table[i, at // block].long() * block + at % block)
    for _ in range(4):
        k, v = fresh(2)
        at = lens.long()
        append_paged_kv4(None, None, k, v, cache, table[torch.arange(2, device=cuda), at // block].long() * block + at % block)
        lens += 1
        query = torch.randn(2, heads, head, generator=gen, device=cuda).to(torch.bfloat16)
        got = paged_attention4(query, cache, table, lens, head ** -0.5)
        _check(got, query, cache, table, lens.tolist(), head ** -0.5)
    assert gather_paged_kv4(cache, table[0, :1].long() * block).isfinite().all()


@pytest.mark.parametrize("length,count", [(200, 3), (130, 5), (129, 2)])
def test_several_tokens_of_a_length_past_the_table(cuda, length, count):
    """Keys past the table's width are left out; which of the rest a token sees goes by the whole length."""
    cache, table = _pages(cuda, [200], 16, 2, 128, 14)
    table = table[:, :8].contiguous()  # 128 keys
    query = torch.randn(count, 8, 128, device=cuda, generator=torch.Generator(device=cuda).manual_seed(1)).to(torch.bfloat16)
    got = paged_attention4(query, cache, table, torch.tensor([length], dtype=torch.int32, device=cuda), 128 ** -0.5,
                           query_start=torch.tensor([0, count], dtype=torch.int32, device=cuda))
    seen = [min(length - count + j + 1, 128) for j in range(count)]
    assert bool(got.isfinite().all())
    _check(got, query, cache, table.expand(count, -1), seen, 128 ** -0.5)


@pytest.mark.parametrize("head", [64, 128])
@pytest.mark.parametrize("step", [math.inf, 65504.0, 1e-7])
def test_steps_that_a_row_does_not_see(cuda, head, step):
    """The step of a later token's V row changes no bit of the tokens before it."""
    lens, start = [123], torch.tensor([0, 3], dtype=torch.int32, device=cuda)
    cache, table = _pages(cuda, lens, 16, 1, head, 9)
    query = torch.randn(3, 2, head, device=cuda, generator=torch.Generator(device=cuda).manual_seed(1)).to(torch.float16)
    lengths = torch.tensor(lens, dtype=torch.int32, device=cuda)
    clean = paged_attention4(query, cache, table, lengths, head ** -0.5, query_start=start)
    cache.scales[1, table[0, 7], 0, 10, 0, 0] = step  # key 122
    got = paged_attention4(query, cache, table, lengths, head ** -0.5, query_start=start)
    assert torch.equal(got[:2], clean[:2])
    assert bool(got[:2].isfinite().all())
    if step < 1:
        assert bool(got.isfinite().all())
        _check(got, query, cache, table, lens, head ** -0.5, [0, 3])


@pytest.mark.parametrize("head", [64, 128])
def test_rows_of_very_different_step(cuda, head):
    """V rows of large step that hardly weigh take no bits of those that do.

    Two keys have a logit of 60, the others of -60, and a key in 32, of the latter, has a V row of step 4,000
    where the rest have about 2e-6.  The reference keeps the largest factor p step' over 2^10, so fp16
    subnormals (off by 2^-25) are off by 2^-35 of the largest p step' at most: the term of _check covers
    them, as long as p and step' are taken from the same key."""
    n = 500
    cache, table = _pages(cuda, [n], 16, 2, head, 15, step=(1e-6, 4e-6), low=(-2e-5, 2e-5))
    at = torch.arange(3, n, 32, device=cuda)
    page, row = table[0].long()[at // 16], at % 16
    cache.scales[1, page, :, row, :, 0], cache.scales[1, page, :, row, :, 1] = 4000.0, -20000.0
    cache.scales[0, ..., 0], cache.scales[0, ..., 1] = 0.0, -1.0
    for key in (11, 331):  # beside keys 3 and 323 in a lane
        cache.scales[0, table[0, key // 16], :, key % 16, :, 1] = 1.0
    query = torch.ones(1, 8, head, device=cuda, dtype=torch.bfloat16)
    got = paged_attention4(query, cache, table, torch.tensor([n], dtype=torch.int32, device=cuda), 60.0 / head)
    assert bool(got.isfinite().all())
    _check(got, query, cache, table, [n], 60.0 / head)


@pytest.mark.parametrize("step", [math.nan, math.inf])
@pytest.mark.parametrize("group", [0, 1])
@pytest.mark.parametrize("key", [5, 995])  # in a whole tile, in the last one
def test_not_finite_keeps_to_its_group(cuda, step, group, key):
    """A V row's group that is not finite reaches its own 64 dimensions, in the rows that see it."""
    lens, heads, head = [1000, 77], 8, 128
    cache, table = _pages(cuda, lens, 16, 2, head, 16)
    query = torch.randn(2, heads, head, device=cuda, generator=torch.Generator(device=cuda).manual_seed(1)).to(torch.bfloat16)
    lengths = torch.tensor(lens, dtype=torch.int32, device=cuda)
    clean = paged_attention4(query, cache, table, lengths, head ** -0.5)
    bad = PagedKV4(cache.codes, cache.scales.clone())
    bad.scales[1, table[0, key // 16], 0, key % 16, group, 0] = step  # KV head 0: query heads 0 to 3
    got = paged_attention4(query, bad, table, lengths, head ** -0.5)
    hit = torch.zeros(2, heads, head, dtype=torch.bool, device=cuda)
    hit[0, :4, 64 * group:64 * group + 64] = True
    assert not bool(got[hit].isfinite().any()) and bool(got[~hit].isfinite().all())
    _check(torch.where(hit, clean, got), query, cache, table, lens, head ** -0.5)


@pytest.mark.parametrize("size", [2.0 ** 105, 2.0 ** 118, torch.finfo(torch.bfloat16).max])
@pytest.mark.parametrize("sign", [1, -1])
def test_logits_past_fp32(cuda, size, sign):
    """Logits that fp32 does not tell apart, or does not hold: the value of the highest, or not finite -- never
    the zeros of a row that sees no key, and the same in whole tiles and in cut ones."""
    lens, best = [20, 64, 1100, 0], (7, 40, 1030)
    cache, table = _pages(cuda, lens, 16, 2, 128, 17)
    cache.scales[0, ..., 0], cache.scales[0, ..., 1] = 0.0, 1.0  # rows of K that are 1 throughout, one of them 1 +- 1/2
    for i, key in enumerate(best):
        cache.scales[0, table[i, key // 16], :, key % 16, :, 1] = 1.0 + 0.5 * sign
    query = torch.full((4, 8, 128), sign * size, device=cuda, dtype=torch.bfloat16)
    got = paged_attention4(query, cache, table, torch.tensor(lens, dtype=torch.int32, device=cuda), 1.0)
    assert int((got[3] != 0).sum()) == 0
    u = torch.finfo(query.dtype).eps / 2
    for i, key in enumerate(best):
        varied, low = (x[key].repeat_interleave(4, 0) for x in _parts(cache, table[i], lens[i], 1))
        # one factor p step rounded to fp16, and the result
        off, bound = (got[i].double() - varied - low).abs(), u * (varied + low).abs() + (2.0 ** -11 + 2.0 ** -20) * (varied + low.abs())
        assert bool(((off <= bound) | ~got[i].isfinite()).all())
    # several tokens, the first of which sees nothing
    got = paged_attention4(query[:3], cache, table[:1], torch.tensor([2], dtype=torch.int32, device=cuda), 1.0,
                           query_start=torch.tensor([0, 3], dtype=torch.int32, device=cuda))
    assert int((got[0] != 0).sum()) == 0 and bool((got[1:] != 0).any(-1).all())


@pytest.mark.parametrize("lens,block", [([40000], 128), ([9000, 300, 7001], 24)])
@pytest.mark.parametrize("head", [64, 128])
def test_every_part_counts(cuda, lens, block, head):
    """Uniform weights and values that are zero but in one stretch of 256 keys (a CTA's round), swept over
    the sequence: a part of a cut piece that is lost, or joined twice, changes an output by all of it.

    Logits are 0, so exp2 and M are the same for every key.  A value is 15 steps of 1/8 over a lowest value
    of 0: its factor is rounded to fp16 (2^-11) and weighs with 15 - 8 and, in fp32, 8; sums of up to
    40,000 terms in fp32, in parts of at most some hundred a lane and then by tree: 2^-14.  The result is
    rounded once."""
    cache, table = _pages(cuda, lens, block, 2, head, 18, step=(0.0, 0.0), low=(0.0, 0.0))
    cache.codes[1] = 255
    query = torch.randn(len(lens), 8, head, device=cuda, generator=torch.Generator(device=cuda).manual_seed(1)).to(torch.float16)
    lengths = torch.tensor(lens, dtype=torch.int32, device=cuda)
    got, want = [], []
    for first in range(0, max(lens), 256):
        marked = PagedKV4(cache.codes, cache.scales.clone())
        counts = []
        for i, n in enumerate(lens):
            keys = torch.arange(min(first, n), min(first + 256, n), device=cuda)
            marked.scales[1, table[i].long()[keys // block], :, keys % block, :, 0] = 0.125
            counts.append(1.875 * len(keys) / n)
        got.append(paged_attention4(query, marked, table, lengths, head ** -0.5))
        want.append(counts)
    want = torch.tensor(want, dtype=torch.float64, device=cuda)[..., None, None]
    off = (torch.stack(got).double() - want).abs()
    u = torch.finfo(torch.float16).eps / 2
    assert bool((off <= want * (u + 2.0 ** -11 + 2.0 ** -14) + 2.0 ** -24).all())


@pytest.mark.parametrize("key", [0, 255, 256, 511, 512, 8191, 16384, 20000, 32767, 39999])
def test_one_key_takes_all(cuda, key):
    """One key of 40,000 whose logit is far over the rest, anywhere: the output is its value."""
    cache, table = _pages(cuda, [40000], 128, 2, 128, 19)
    query = torch.ones(1, 16, 128, device=cuda, dtype=torch.bfloat16)
    cache.scales[0, table[0, key // 128], :, key % 128] = 4.0  # values of 4 to 64, the others' -2.7 to 4.1
    got = paged_attention4(query, cache, table, torch.tensor([40000], dtype=torch.int32, device=cuda), 0.25)
    vv, vl = _parts(cache, table[0], 40000, 1)
    want, mass = (vv + vl)[key].repeat_interleave(8, 0), (vv + vl.abs())[key].repeat_interleave(8, 0)
    # its logit is some 1,000 over the others': p is 1 and 0, one factor rounded to fp16, and the result
    u = torch.finfo(query.dtype).eps / 2
    assert bool(((got[0].double() - want).abs() <= u * want.abs() + (2.0 ** -11 + 2.0 ** -20) * mass).all())


@pytest.mark.parametrize("case", CASES, ids=str)
def test_outputs_are_finite(cuda, case):
    """_check takes a maximum, which passes over NaN: whatever the pages hold behind a sequence's end, none comes out."""
    lens, block, heads, kv_heads, head, dtype, counts = case
    cache, table = _pages(cuda, lens, block, kv_heads, head, 3)
    total = len(lens) if counts is None else sum(counts)
    query = torch.randn(total, heads, head, generator=torch.Generator(device=cuda).manual_seed(4), device=cuda).to(dtype)
    begin = None if counts is None else torch.tensor([0, *torch.tensor(counts).cumsum(0).tolist()], dtype=torch.int32, device=cuda)
    got = paged_attention4(query, cache, table, torch.tensor(lens, dtype=torch.int32, device=cuda), head ** -0.5, query_start=begin)
    assert bool(got.isfinite().all())


def _centred_bound(q, step, varied, low, key_step, keys, p, scale, info):
    """What one query head of 64 bits may be off by, whatever the steps and lowest values are.

    With factors f_j = p_j step_j, codes c_j and middles m_j = low_j + 8 step_j:

    * a factor is rounded to fp16 and weighs with c - 8: 2^-11 sum f |c - 8| (and the subnormals, see
      test_rows_of_very_different_step);
    * a product of the matrix unit lines its terms up by the fp16 exponents of the operands, and a code is a
      subnormal 2^-24 c, whose exponent counts as 2^-14: sums are cut 2^10 above fp32's 2^-24 (measured:
      2^-18.6 of 8 f), at most 2^-13 of each product's largest factor: 2^-13 sum f.  The same for the logits:
      4 products a group cut at 2^-13 max |q| step, in log2 scale log2e; 2^-10 scale max |q| max step covers both
      groups, twice (numerator and sum);
    * fp32 logits, exp2 and sums: 2^-15 (A + 1) of sum p |m| + f |c - 8|, A = scale log2e sum |q| |k|;
    * the result is rounded once."""
    e = torch.einsum("hgl,lhd->hgd", p, (varied - 8 * step).abs())
    everything = e + torch.einsum("hgl,lhd->hgd", p, (low + 8 * step).abs())
    factors = torch.einsum("hgl,lhd->hgd", p, step)
    largest = torch.einsum("hgl,lhd->hgld", p, step).amax((2, 3))[..., None]
    size = torch.einsum("hgd,lhd->hgl", q.abs(), keys).amax(-1)[..., None] * abs(scale) * math.log2(math.e)
    cut = 2.0 ** -9 * abs(scale) * q.abs().amax(-1)[..., None] * key_step
    return 2.0 ** -11 * e + 2.0 ** -13 * factors + (2.0 ** -15 * (size + 1) + cut) * everything \
        + len(step) * 2.0 ** -32 * largest + info.smallest_normal


@pytest.mark.parametrize("step", [(1e-3, 5.0), (0.0, 0.01)])
@pytest.mark.parametrize("low", [(-30.0, 10.0), (-0.1, 0.1)])
@pytest.mark.parametrize("lens,block,heads,kv_heads,head,dtype", [
    ([1, 20, 700, 3], 16, 16, 2, 128, torch.bfloat16), ([16, 1, 5, 2000], 24, 10, 5, 64, torch.float16),
    ([9000], 128, 8, 8, 128, torch.float16), ([2] * 40, 33, 24, 8, 64, torch.bfloat16)])
def test_wide_steps_and_lowest_values(cuda, lens, block, heads, kv_heads, head, dtype, step, low):
    cache, table = _pages(cuda, lens, block, kv_heads, head, 22, step, low)
    query = torch.randn(len(lens), heads, head, device=cuda, generator=torch.Generator(device=cuda).manual_seed(1)).to(dtype)
    scale = head ** -0.5
    got = paged_attention4(query, cache, table, torch.tensor(lens, dtype=torch.int32, device=cuda), scale)
    info = torch.finfo(dtype)
    key_step = float(cache.scales[0, ..., 0].nan_to_num(0).max())
    for i, n in enumerate(lens):
        kv, kl = _parts(cache, table[i], n, 0)
        vv, vl = _parts(cache, table[i], n, 1)
        pages = table[i, :-(-n // block)].long()
        steps = cache.scales[1][pages][..., :1].double().expand(-1, -1, -1, -1, 64).flatten(-2).transpose(1, 2).flatten(0, 1)[:n]
        q = query[i].double().unflatten(0, (kv_heads, -1))
        p = torch.softmax(torch.einsum("hgd,lhd->hgl", q, kv + kl) * scale, -1)
        want = torch.einsum("hgl,lhd->hgd", p, vv + vl)
        bound = want.abs() * (info.eps / 2) + _centred_bound(q, steps, vv, vl, key_step, kv + kl.abs(), p, scale, info)
        off = (got[i].double().unflatten(0, (kv_heads, -1)) - want).abs()
        assert bool((off <= bound).all()), (i, float((off / bound).max()))
