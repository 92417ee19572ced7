"""cb_prompt_attention against attention in 64 bits, sequence by sequence.

Bound, with exact probabilities p_j, values v_j and u = eps / 2 of the type:

* each unnormalized probability is rounded once to the type: at most u sum p |v|
  (an fp16 one below 2^-14 is a subnormal, off by 2^-25; the largest of a row is at least
  2^-8 -- the reference moves when the maximum grows by 2^8 -- so n keys add at most
  n 2^-17 max |v|);
* exp2 and the fp32 sums, and the logits: D products and sums in fp32 of size
  A = scale log2e sum |q| |k|, off by at most 2^-24 (D + 8) A <= 2^-16 A for D 128, which
  changes p by that much relative, once in the numerator and once in the sum: 2^-15 A;
* the result is rounded once: u |out|.

    |got - want| <= u |want| + (u + 2^-15 (A + 1)) sum p |v| + [fp16] n 2^-17 max |v| + tiny
"""

from __future__ import annotations

import math

import pytest
import torch

from cacheblend_b200 import prompt_attention
from cacheblend_b200.attention import prompt_attention_workspace_bytes

pytestmark = pytest.mark.gpu


def _starts(lengths, device, first=0):
    return torch.tensor([first, *(first + torch.tensor(lengths).cumsum(0)).tolist()], dtype=torch.int32, device=device)


def _want(q, k, v, scale):
    """(out, bound without the rounding of the result) of one sequence in 64 bits."""
    n, heads, _ = q.shape
    keys, kv_heads, _ = k.shape
    groups = heads // kv_heads
    last = torch.arange(n, device=q.device) + keys - n
    hidden = torch.arange(keys, device=q.device)[None, :] > last[:, None]
    out, bound = torch.zeros(q.shape, dtype=torch.float64, device=q.device), torch.zeros(q.shape, dtype=torch.float64, device=q.device)
    u = torch.finfo(q.dtype).eps / 2
    if keys == 0:
        return out, bound
    for h in range(heads):
        qh, kh, vh = q[:, h].double(), k[:, h // groups].double(), v[:, h // groups].double()
        w = (qh @ kh.T * scale).masked_fill(hidden, -math.inf)
        size = (qh.abs() @ kh.abs().T).masked_fill(hidden, 0).amax(-1, keepdim=True) * scale * math.log2(math.e)
        p = torch.softmax(w, -1).nan_to_num(0.0)  # a row that sees nothing: zeros
        out[:, h] = p @ vh
        bound[:, h] = (u + 2.0 ** -15 * (size + 1)) * (p @ vh.abs())
        if q.dtype == torch.float16:
            bound[:, h] += keys * 2.0 ** -17 * vh.abs().amax()
    return out, bound


def _check(got, q, k, v, starts, key_starts, scale):
    info = torch.finfo(q.dtype)
    worst = 0.0
    for a, b, c, d in zip(starts, starts[1:], key_starts, key_starts[1:]):
        if a == b:
            continue
        want, bound = _want(q[a:b], k[c:d], v[c:d], scale)
        bound += want.abs() * (info.eps / 2) + info.smallest_normal
        worst = max(worst, float(((got[a:b].double() - want).abs() / bound).max()))
    assert worst <= 1, worst


def _inputs(device, tokens, keys, heads, kv_heads, head, dtype, seed):
    gen = torch.Generator(device=device).manual_seed(seed)
    return tuple(torch.randn(n, h, head, generator=gen, device=device).to(dtype)
                 for n, h in ((tokens, heads), (keys, kv_heads), (keys, kv_heads)))


CASES = [
    # query lengths, cached prefixes, heads, kv_heads, head, dtype
    ([1], [0], 32, 8, 128, torch.bfloat16),
    ([301], [0], 32, 8, 128, torch.bfloat16),
    ([1, 64, 65, 0, 63, 128, 129], None, 8, 2, 128, torch.float16),
    ([200, 77], [0, 0], 4, 4, 64, torch.bfloat16),            # one head a group: 128 queries a tile
    ([300, 5, 260], [100, 0, 13], 28, 4, 128, torch.bfloat16),  # groups of 7
    ([140], [1000], 6, 2, 64, torch.float16),                 # groups of 3
    ([33, 40], [0, 128], 128, 1, 128, torch.bfloat16),        # one query a tile
    ([70, 9], [0, 3], 80, 1, 64, torch.bfloat16),             # one query a tile, 48 idle rows
    ([2500], [0], 8, 1, 128, torch.bfloat16),
    ([700, 1, 1, 900, 30], [0, 5000, 1, 200, 0], 16, 2, 128, torch.float16),
    ([17] * 90, None, 16, 2, 64, torch.bfloat16),
]


@pytest.mark.parametrize("case", CASES, ids=lambda c: f"{len(c[0])}x{max(c[0])}-{c[2]}-{c[3]}-{c[4]}-{c[5]}"[:60])
def test_against_64_bits(cuda, case):
    lengths, prefix, heads, kv_heads, head, dtype = case
    key_lengths = lengths if prefix is None else [n + p for n, p in zip(lengths, prefix)]
    q, k, v = _inputs(cuda, sum(lengths), sum(key_lengths), heads, kv_heads, head, dtype, 1)
    start, key_start = _starts(lengths, cuda), None if prefix is None else _starts(key_lengths, cuda)
    error = torch.zeros(1, dtype=torch.int32, device=cuda)
    got = prompt_attention(q, k, v, start, head ** -0.5, key_start=key_start, device_error=error)
    assert int(error) == 0
    _check(got, q, k, v, start.tolist(), (start if key_start is None else key_start).tolist(), head ** -0.5)
    again = prompt_attention(q, k, v, start, head ** -0.5, key_start=key_start)
    assert torch.equal(got, again)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
def test_peaked_and_growing_logits(cuda, dtype):
    """Maxima that grow by far more than 2^8 from tile to tile, and by less."""
    q, k, v = _inputs(cuda, 520, 520, 4, 1, 128, dtype, 2)
    k = (k.float() * torch.linspace(0.1, 12, 520, device=cuda)[:, None, None]).to(dtype)
    start = _starts([520], cuda)
    got = prompt_attention(q, k, v, start, 0.1)
    _check(got, q, k, v, [0, 520], [0, 520], 0.1)
    k = k.flip(0).contiguous()
    _check(prompt_attention(q, k, v, start, 0.1), q, k, v, [0, 520], [0, 520], 0.1)


def test_more_queries_than_keys(cuda):
    """The first queries of a sequence see nothing: zeros."""
    q, k, v = _inputs(cuda, 400 + 300, 150 + 300, 4, 2, 64, torch.bfloat16, 3)
    start, key_start = _starts([400, 300], cuda), _starts([150, 300], cuda)
    got = prompt_attention(q, k, v, start, 0.125, key_start=key_start)
    assert int((got[:250] != 0).sum()) == 0
    _check(got, q, k, v, start.tolist(), key_start.tolist(), 0.125)
    # a sequence with no keys at all, beside one that has some
    q, k, v = _inputs(cuda, 90, 50, 4, 2, 64, torch.bfloat16, 4)
    got = prompt_attention(q, k, v, _starts([40, 50], cuda), 0.125, key_start=_starts([0, 50], cuda))
    assert int((got[:40] != 0).sum()) == 0
    _check(got, q, k, v, [0, 40, 90], [0, 0, 50], 0.125)


@pytest.mark.parametrize("lengths,keys", [
    ([2500], [2500]),  # one sequence, several items per CTA
    ([70, 1, 400, 33, 64, 900, 16] * 6, [0, 1, 300, 0, 20, 1200, 500] * 6),  # many that see nothing, among others
    ([40] * 90, [0] * 89 + [7]),  # almost only those
    ([17] * 200, [17] * 200),  # one tile each: the next item follows at once
])
def test_several_items_per_cta(cuda, lengths, keys):
    q, k, v = _inputs(cuda, sum(lengths), sum(keys), 16, 8, 64 if len(lengths) > 100 else 128, torch.bfloat16, 11)
    starts, key_starts = _starts(lengths, cuda), _starts(keys, cuda)
    workspace = torch.full((prompt_attention_workspace_bytes(len(q), len(lengths), 16, 8, q.shape[2]),), 255, dtype=torch.uint8,
                           device=cuda)
    error = torch.zeros(1, dtype=torch.int32, device=cuda)
    got = prompt_attention(q, k, v, starts, 0.1, key_start=key_starts, workspace=workspace, device_error=error)
    for _ in range(3):  # the workspace as the call before left it
        again = prompt_attention(q, k, v, starts, 0.1, key_start=key_starts, workspace=workspace, device_error=error)
        assert bool((got.view(torch.int16) == again.view(torch.int16)).all())
    assert int(error) == 0
    _check(got, q, k, v, starts.tolist(), key_starts.tolist(), 0.1)


@pytest.mark.parametrize("lengths,keys,kv_heads", [
    ([3, 0, 70, 1, 65], [3, 0, 70, 9, 200], 4),
    ([1] * 32, [1, 130] * 16, 2),  # as many as a warp has lanes
    ([1] * 33, [1, 130, 5] * 11, 2),
    ([0, 0, 129, 0], [7, 0, 129, 0], 1),
    ([130, 20, 0, 300], [0, 500, 0, 300], 2),
])
def test_few_items(cuda, lengths, keys, kv_heads):
    q, k, v = _inputs(cuda, sum(lengths), sum(keys), 4 * kv_heads, kv_heads, 128, torch.float16, 12)
    starts, key_starts = _starts(lengths, cuda), _starts(keys, cuda)
    got = prompt_attention(q, k, v, starts, 0.09, key_start=key_starts)
    _check(got, q, k, v, starts.tolist(), key_starts.tolist(), 0.09)


def test_strides_and_rows_behind(cuda):
    """Slices of one projection's output; rows of no sequence stay as they were."""
    heads, kv_heads, head, tokens = 8, 2, 128, 333
    fused = torch.randn(tokens, (heads + 2 * kv_heads) * head + 8, device=cuda,
                        generator=torch.Generator(device=cuda).manual_seed(5)).to(torch.bfloat16)
    q, k, v = (x.unflatten(-1, (-1, head)) for x in fused[:, 8:].split([heads * head, kv_heads * head, kv_heads * head], -1))
    out = torch.full((tokens, heads + 1, head), 7.0, dtype=torch.bfloat16, device=cuda)[:, 1:]
    start = _starts([100, 180], cuda, first=3)
    got = prompt_attention(q, k, v, start, head ** -0.5, out=out)
    assert got is out
    _check(got, q, k, v, start.tolist(), start.tolist(), head ** -0.5)
    assert (got[:3] == 7).all() and (got[283:] == 7).all()
    # heads before tokens
    swapped = k.transpose(0, 1).contiguous().transpose(0, 1)
    assert torch.equal(prompt_attention(q, swapped, v, start, head ** -0.5)[3:283], got[3:283])
    # starts past the rows are clamped
    over = prompt_attention(q, k, v, torch.tensor([3, 103, 10 ** 6], dtype=torch.int32, device=cuda), head ** -0.5)
    _check(over, q, k, v, [3, 103, tokens], [3, 103, tokens], head ** -0.5)
    with pytest.raises(NotImplementedError, match="aligned"):
        prompt_attention(fused[:, 4:4 + heads * head].unflatten(-1, (heads, head)), k, v, start, 0.1)


@pytest.mark.parametrize("dtype,groups", [(torch.bfloat16, 4), (torch.float16, 1), (torch.bfloat16, 7)])
def test_not_finite_in_masked_places(cuda, dtype, groups):
    """NaN and infinities in keys and values that a row does not see -- later tokens, other
    sequences, rows behind the last -- reach no output of that row; a row that sees one has it."""
    lengths = [150, 90]
    q, k, v = _inputs(cuda, 300, 300, 2 * groups, 2, 128, dtype, 6)
    start = _starts(lengths, cuda)
    clean = prompt_attention(q, k, v, start, 0.09)
    bad_k, bad_v = k.clone(), v.clone()
    for x in (bad_k, bad_v):
        x[240:] = torch.nan
        x[260:] = torch.inf
    got = prompt_attention(q, bad_k, bad_v, start, 0.09)
    assert torch.equal(got[:240], clean[:240])
    bad_v[101, 0, 5], bad_v[149, 0, 7], bad_v[170, 1, 100] = torch.nan, torch.inf, -torch.inf
    got = prompt_attention(q, bad_k, bad_v, start, 0.09)
    expect = clean[:240].clone()
    expect[101:150, :groups, 5] = torch.nan
    expect[149:150, :groups, 7] = torch.inf
    expect[170:240, groups:, 100] = -torch.inf
    assert torch.equal(got[:240].isnan(), expect.isnan())
    fine = expect.isfinite()
    assert torch.equal(got[:240][fine], expect[fine])
    assert torch.equal(got[:240].isinf(), expect.isinf())
    bad_k[120, 1, 0] = torch.nan
    got = prompt_attention(q, bad_k, v, start, 0.09)
    assert torch.equal(got[:120], clean[:120]) and torch.equal(got[:240, :groups], clean[:240, :groups])
    assert bool(got[120:150, groups:].isnan().all()) and torch.equal(got[150:240], clean[150:240])
    bad_q = q.clone()
    bad_q[10, 0] = torch.nan
    got = prompt_attention(bad_q, k, v, start, 0.09)
    rest = torch.ones(300, 2 * groups, dtype=torch.bool, device=cuda)
    rest[10, 0] = False
    rest[240:] = False
    assert bool(got[10, 0].isnan().all()) and torch.equal(got[rest], clean[rest])


def test_streams_workspace_and_graph(cuda):
    q, k, v = _inputs(cuda, 500, 500, 8, 2, 128, torch.bfloat16, 7)
    start = _starts([120, 300], cuda)
    want = prompt_attention(q, k, v, start, 0.1)
    torch.cuda.synchronize()
    side = torch.cuda.Stream(cuda)
    got = prompt_attention(q, k, v, start, 0.1, stream=side)
    side.synchronize()
    assert torch.equal(got[:420], want[:420])
    size = prompt_attention_workspace_bytes(500, 2, 8, 2, 128)
    dirty = torch.full((size,), 255, dtype=torch.uint8, device=cuda)
    assert torch.equal(prompt_attention(q, k, v, start, 0.1, workspace=dirty)[:420], want[:420])
    with pytest.raises(ValueError, match="workspace"):
        prompt_attention(q, k, v, start, 0.1, workspace=dirty[:size - 16])
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        inside = prompt_attention(q, k, v, start, 0.1)
    start.copy_(torch.tensor([0, 400, 500], dtype=torch.int32))  # the next batch
    graph.replay()
    torch.cuda.synchronize()
    _check(inside, q, k, v, [0, 400, 500], [0, 400, 500], 0.1)


def test_dimensions_of_one(cuda):
    """One token, one head: whatever strides such dimensions carry."""
    q, k, v = _inputs(cuda, 1, 1, 1, 1, 64, torch.bfloat16, 9)
    odd = [torch.as_strided(t, (1, 1, 64), (3, 7, 1)) for t in (q, k, v)]
    got = prompt_attention(*odd, _starts([1], cuda), 0.1)
    assert torch.equal(got, v)


def test_calls_at_once_and_again(cuda):
    """Calls of different shapes on two streams at once, many times: always the same bits."""
    problems = []
    for seed, (lengths, heads, kv_heads, head) in enumerate([([700, 3, 2100], 16, 2, 128), ([40] * 30, 8, 4, 64), ([900], 14, 2, 128)]):
        q, k, v = _inputs(cuda, sum(lengths), sum(lengths), heads, kv_heads, head, torch.bfloat16, seed)
        problems.append((q, k, v, _starts(lengths, cuda), 0.1))
    want = [prompt_attention(*p) for p in problems]
    torch.cuda.synchronize()
    sides = [torch.cuda.Stream(cuda) for _ in range(2)]
    error = torch.zeros(1, dtype=torch.int32, device=cuda)
    torch.cuda.synchronize()
    got = [(i, prompt_attention(*problems[i], stream=sides[n % 2], device_error=error)) for n in range(20) for i in range(3)]
    torch.cuda.synchronize()
    assert int(error) == 0 and all(torch.equal(out, want[i]) for i, out in got)


def test_long_prompt(cuda):
    """A prompt of many tiles per row, checked on its last rows."""
    q, k, v = _inputs(cuda, 9000, 9000, 4, 1, 128, torch.bfloat16, 8)
    got = prompt_attention(q, k, v, _starts([9000], cuda), 128 ** -0.5)
    want, bound = _want(q[8900:], k, v, 128 ** -0.5)
    bound += want.abs() * 2.0 ** -8 + 1e-30
    assert float(((got[8900:].double() - want).abs() / bound).max()) <= 1


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("head", [64, 128])
def test_logits_of_minus_infinity(cuda, dtype, head):
    """A row whose seen logits are all -inf is NaN, as of any softmax of them; beside a finite one they weigh
    nothing; a row that sees no key is zeros."""
    q, k, v = _inputs(cuda, 300 + 200 + 40, 300 + 200, 8, 2, head, dtype, 13)
    q[..., 0] = 1.0
    k[:300, :, 0] = -torch.inf
    k[100, :, 0] = 0.0  # the only finite logit of the first sequence
    start, key_start = _starts([300, 200, 40], cuda), _starts([300, 200, 0], cuda)
    got = prompt_attention(q, k, v, start, 0.1, key_start=key_start)
    assert bool(got[:100].isnan().all())
    assert torch.equal(got[100:300], v[100].repeat_interleave(4, 0).expand(200, -1, -1))
    assert int((got[500:] != 0).sum()) == 0
    assert bool(got[100:].isfinite().all())
    _check(got[300:500], q[300:500], k[300:], v[300:], [0, 200], [0, 200], 0.1)


@pytest.mark.parametrize("last", [False, True], ids=["peak first", "peak last"])
def test_small_fp16_probabilities(cuda, last):
    """Many keys of small weight beside one of large weight and value 0.

    Their probabilities, 2^-25.2 of the largest, are what the output consists of.  An fp16 probability of
    2^7 2^-25.2 (the reference lies 2^7 below the maximum, or more where a later one is larger) is a subnormal,
    off by 2^-25 at most: n keys by n 2^-32 max |v|, against an output of n 2^-25.2.  The logits are exact
    (one dimension, multiples of 2^-4); exp2 and the sums as in the bound above."""
    n, head = 4096, 128
    q, k, v = (torch.zeros(m, 1, head, dtype=torch.float16, device=cuda) for m in (1, n + 1, n + 1))
    q[..., 0], k[..., 0] = 1.0, -25.1875
    k[n if last else 0, :, 0] = 0.0
    v[:] = 1.0
    v[n if last else 0] = 0.0
    scale = math.log(2.0)  # logits as powers of two
    got = prompt_attention(q, k, v, _starts([1], cuda), scale, key_start=_starts([n + 1], cuda))
    want, _ = _want(q, k, v, scale)
    off = (got.double() - want).abs()
    assert float((off / (want * (2.0 ** -11 + 2.0 ** -15 * 27) + (n + 1) * 2.0 ** -32)).max()) <= 1


def test_no_keys_at_all(cuda):
    """Zeros in the rows of the sequences, the rest as it was."""
    q, k, v = _inputs(cuda, 90, 0, 4, 2, 64, torch.bfloat16, 14)
    for lengths in ([40, 45], [1] * 40):  # found by the CTAs themselves, and from a list
        out = torch.full_like(q, 3.0)
        starts = _starts(lengths, cuda, first=2)
        got = prompt_attention(q, k, v, starts, 0.125, key_start=torch.zeros_like(starts), out=out)
        end = 2 + sum(lengths)
        assert int((got[2:end] != 0).sum()) == 0 and bool((got[:2] == 3).all()) and bool((got[end:] == 3).all())


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("queries,keys,head", [(1, 5001, 128), (5, 5001, 64), (200, 5001, 128)])
def test_every_tile_counts(cuda, dtype, queries, keys, head):
    """Uniform weights, and per KV head values that are 1 in one tile of 128 keys and 0 elsewhere: a tile
    that is lost or taken twice changes an output by all of it.

    Logits are 0 and probabilities a power of two, so the sums are exact (up to 5,001 ones); the quotient
    is off by 2 ulp of fp32 and the result is rounded once."""
    tiles = -(-keys // 128)
    q, k, v = _inputs(cuda, queries, keys, tiles, tiles, head, dtype, 15)
    k.zero_()
    at = torch.arange(keys, device=cuda)
    v[:] = (at[:, None] // 128 == torch.arange(tiles, device=cuda)).to(dtype)[..., None]
    got = prompt_attention(q, k, v, _starts([queries], cuda), head ** -0.5, key_start=_starts([keys], cuda))
    seen = keys - queries + 1 + torch.arange(queries, device=cuda)[:, None]
    count = (seen - torch.arange(tiles, device=cuda) * 128).clamp(0, 128)
    want = (count.double() / seen)[..., None]
    assert bool(((got.double() - want).abs() <= want * (torch.finfo(dtype).eps / 2 + 2.0 ** -20)).all())


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
def test_one_key_of_a_long_prefix_takes_all(cuda, dtype):
    """Per KV head one key far over the rest, in the first tile, the last and each between.

    fp16: the probabilities' subnormals are off by n 2^-32 max |v| (see above)."""
    keys, head, kv_heads = 5001, 128, 40
    q, k, v = _inputs(cuda, 3, keys, kv_heads, kv_heads, head, dtype, 16)
    planted = torch.arange(kv_heads, device=cuda) * 128 + torch.arange(kv_heads, device=cuda) * 37 % 128
    planted = planted.clamp(max=keys - 3)
    heads = torch.arange(kv_heads, device=cuda)
    q[:] = q[:1]
    k[planted, heads] = q[0]  # a logit of |q|^2 / 4, about 32, against +-2.8
    got = prompt_attention(q, k, v, _starts([3], cuda), 0.25, key_start=_starts([keys], cuda))
    want, bound = _want(q, k, v, 0.25)
    if dtype == torch.float16:
        bound -= keys * (2.0 ** -17 - 2.0 ** -32) * v.double().abs().amax((0, 2))[:, None]
    bound += want.abs() * (torch.finfo(dtype).eps / 2) + 2.0 ** -24
    assert float(((got.double() - want).abs() / bound).max()) <= 1
    assert float((want - v[planted, heads].double()).abs().max()) < 0.05  # the planted key's value it is


@pytest.mark.parametrize("case", CASES, ids=lambda c: f"{len(c[0])}x{max(c[0])}-{c[2]}-{c[3]}-{c[4]}-{c[5]}"[:60])
def test_outputs_are_finite(cuda, case):
    """_check takes a maximum, which passes over NaN: no output is one."""
    lengths, prefix, heads, kv_heads, head, dtype = case
    key_lengths = lengths if prefix is None else [n + p for n, p in zip(lengths, prefix)]
    q, k, v = _inputs(cuda, sum(lengths), sum(key_lengths), heads, kv_heads, head, dtype, 1)
    got = prompt_attention(q, k, v, _starts(lengths, cuda), head ** -0.5, key_start=_starts(key_lengths, cuda))
    assert bool(got.isfinite().all())
