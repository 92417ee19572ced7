"""cb_append_paged_kv / cb_append_paged_kv4 / cb_gather_paged_kv4 against plain forms.

Rotation bound: with table values c, s exact, the kernel rounds a c, b s and their
difference to fp32 (each within 2^-24 relative) and the result once to the element type
(u = eps / 2 relative, or half the smallest subnormal), so

    |got - exact| <= (1 + u) 2^-24 (|a c| + |b s| + |exact| + 2^-23 (...)) + u |exact| + tiny / 2
                  <= 2^-22 (|a c| + |b s|) + u |exact| + tiny

The 4-bit rows are compared code for code with the same fp32 steps in numpy (IEEE), and
with the values in 64 bits: a code is off by at most half a step, the lowest value by
2^-11 |low| and fifteen steps by 15 * 2^-11 step (fp16), plus fp32 rounding.
"""

from __future__ import annotations

from types import SimpleNamespace

import numpy as np
import pytest
import torch

from cacheblend_b200 import PagedKV4, append_paged_kv, append_paged_kv4, gather_paged_kv4

pytestmark = pytest.mark.gpu

MAX_POSITION = 5000


def _rope(head, rotary, neox, dtype, device):
    inverse = 1.0 / (1e4 ** (torch.arange(0, rotary, 2, dtype=torch.float64) / rotary))
    angles = torch.arange(MAX_POSITION, dtype=torch.float64)[:, None] * inverse
    table = torch.cat((angles.cos(), angles.sin()), -1).to(dtype).to(device)
    return SimpleNamespace(head_size=head, rotary_dim=rotary, is_neox_style=neox, cos_sin_cache=table)


def _turn(x, positions, rope, real):
    """(rotated, |a c| + |b s|) in ``real`` arithmetic, one op at a time."""
    width = rope.rotary_dim
    row = rope.cos_sin_cache[positions].to(real)[:, None]
    cos, sin = row[..., :width // 2], row[..., width // 2:]
    x = x.to(real)
    out, size = x.clone(), torch.zeros_like(x)
    one, two = (slice(0, width // 2), slice(width // 2, width)) if rope.is_neox_style else \
        (slice(0, width, 2), slice(1, width, 2))
    a, b = x[..., one], x[..., two]
    out[..., one], out[..., two] = a * cos - b * sin, b * cos + a * sin
    size[..., one], size[..., two] = (a * cos).abs() + (b * sin).abs(), (b * cos).abs() + (a * sin).abs()
    return out, size


def _check_turn(got, x, positions, rope):
    exact, size = _turn(x, positions, rope, torch.float64)
    info = torch.finfo(got.dtype)
    bound = size * 2.0 ** -22 + exact.abs() * (info.eps / 2) + info.smallest_normal * info.eps
    over = (got.double() - exact).abs() - bound
    assert float(over.max()) <= 0
    same, _ = _turn(x, positions, rope, torch.float32)
    assert torch.equal(got, same.to(got.dtype))  # the same fp32 steps: the same bits


def _inputs(device, tokens, heads, kv_heads, head, dtype, seed, pad=0):
    gen = torch.Generator(device=device).manual_seed(seed)
    fused = torch.randn(tokens, (heads + 2 * kv_heads) * head + pad, generator=gen, device=device).to(dtype)
    q, k, v = fused[:, :(heads + 2 * kv_heads) * head].split([heads * head, kv_heads * head, kv_heads * head], -1)
    positions = torch.randint(0, MAX_POSITION, (tokens,), generator=gen, device=device)
    return q.unflatten(-1, (heads, head)), k.unflatten(-1, (kv_heads, head)), v.unflatten(-1, (kv_heads, head)), positions


def _slots(device, tokens, total, seed):
    gen = torch.Generator(device=device).manual_seed(seed)
    return torch.randperm(total, generator=gen, device=device)[:tokens]


CASES = [
    # tokens, heads, kv_heads, head, rotary, neox, block, dtype, table, pad
    (1, 32, 8, 128, 128, True, 16, torch.bfloat16, torch.float32, 0),
    (77, 32, 8, 128, 128, True, 16, torch.bfloat16, torch.bfloat16, 0),
    (33, 14, 2, 64, 64, False, 24, torch.float16, torch.float32, 0),
    (130, 6, 3, 96, 48, True, 7, torch.bfloat16, torch.float32, 0),     # 48 / 2 = 24: whole pieces of 8
    (65, 4, 4, 80, 40, True, 16, torch.float16, torch.float16, 0),     # 40 / 2 = 20: piece by piece does not fit
    (19, 5, 1, 20, 6, False, 5, torch.bfloat16, torch.float32, 3),      # odd rows and strides
    (40, 2, 2, 64, 32, False, 1, torch.float32, torch.float32, 0),
    (9, 3, 3, 1, 0, True, 16, torch.float32, torch.float32, 0),         # heads of one value
    (300, 64, 8, 256, 256, True, 128, torch.bfloat16, torch.float32, 8),
    # enough tokens for several heads per thread, head counts that four does not divide
    (3001, 10, 5, 128, 128, True, 16, torch.bfloat16, torch.float32, 0),
    (5003, 7, 7, 64, 32, False, 16, torch.float16, torch.float32, 0),
    (4001, 6, 3, 128, 32, True, 32, torch.float32, torch.float32, 0),
]


@pytest.mark.parametrize("case", CASES, ids=str)
def test_append_16_bit(cuda, case):
    tokens, heads, kv_heads, head, rotary, neox, block, dtype, table, pad = case
    rope = _rope(head, rotary, neox, table, cuda) if rotary else None
    q, k, v, positions = _inputs(cuda, tokens, heads, kv_heads, head, dtype, 3, pad)
    blocks = tokens * 2 // block + 2
    slots = _slots(cuda, tokens, blocks * block, 4)
    if tokens > 8:
        slots[-3:] = -1  # padding behind the last sequence
    pages = torch.randn(2, blocks, block, kv_heads, head, device=cuda).to(dtype)
    before = pages.clone()
    turned = append_paged_kv(rope, positions, k, v, pages, slots, block, query=q)
    kept = slots >= 0
    flat, was = pages.view(2, -1, kv_heads, head), before.view(2, -1, kv_heads, head)
    if rope is not None:
        _check_turn(turned, q, positions, rope)
        _check_turn(flat[0][slots[kept]], k[kept], positions[kept], rope)
    else:
        assert torch.equal(turned, q) and torch.equal(flat[0][slots[kept]], k[kept])
    assert torch.equal(flat[1][slots[kept]], v[kept])
    rest = torch.ones(flat.shape[1], dtype=torch.bool, device=cuda)
    rest[slots[kept]] = False
    assert torch.equal(flat[:, rest], was[:, rest])  # nothing else is touched


@pytest.mark.parametrize("layout", ["merged_block", "pair", "hnd", "padded_block"])
def test_append_layouts(cuda, layout):
    tokens, kv_heads, head, block, blocks, dtype = 50, 4, 64, 16, 9, torch.bfloat16
    rope = _rope(head, head, True, torch.float32, cuda)
    _, k, v, positions = _inputs(cuda, tokens, 1, kv_heads, head, dtype, 5)
    slots = _slots(cuda, tokens, blocks * block, 6)
    want = torch.zeros(2, blocks, block, kv_heads, head, dtype=dtype, device=cuda)
    append_paged_kv(rope, positions, k, v, want, slots, block)
    if layout == "merged_block":
        layer = torch.zeros(blocks, 2, block, kv_heads, head, dtype=dtype, device=cuda)
        got = layer.transpose(0, 1)
    elif layout == "pair":
        got = torch.zeros_like(want)
        layer = (got[0], got[1])
    elif layout == "hnd":
        layer = torch.zeros(2, blocks, kv_heads, block, head, dtype=dtype, device=cuda).transpose(2, 3)
        got = layer
    else:  # vLLM may use fewer rows of a block than it holds
        layer = torch.zeros(2, blocks, block + 3, kv_heads, head, dtype=dtype, device=cuda)
        got = layer[:, :, :block]
    append_paged_kv(rope, positions, k, v, layer, slots, block)
    assert torch.equal(got, want)
    if layout == "padded_block":
        assert int(layer[:, :, block:].abs().sum()) == 0


def test_append_leaves_bad_tokens_out(cuda):
    """Device slots outside the cache and positions outside the table: nothing is written."""
    rope = _rope(64, 64, True, torch.float32, cuda)
    q, k, v, positions = _inputs(cuda, 6, 2, 2, 64, torch.bfloat16, 7)
    slots = torch.tensor([0, 32, -5, 2 ** 40, 3, 31], device=cuda)
    positions[4], positions[0] = MAX_POSITION, -1
    pages = torch.zeros(2, 2, 16, 2, 64, dtype=torch.bfloat16, device=cuda)
    turned = append_paged_kv(rope, positions, k, v, pages, slots, 16, query=q)
    written = pages.view(2, 32, -1).abs().sum(-1) > 0
    assert written.nonzero().tolist() == [[0, 31], [1, 31]]
    assert torch.equal(turned[0], torch.zeros_like(turned[0])) and torch.equal(turned[4], torch.zeros_like(turned[4]))
    good = torch.tensor([1, 2, 3, 5], device=cuda)
    _check_turn(turned[good], q[good], positions[good], rope)
    cache = PagedKV4.allocate(2, 16, 2, 64, cuda)
    append_paged_kv4(rope, positions, k, v, cache, slots)
    touched = cache.scales.abs().sum((2, 4, 5)).view(2, 32) > 0
    assert touched.nonzero().tolist() == [[0, 31], [1, 31]]


def test_append_host_indices_and_no_tokens(cuda):
    rope = _rope(64, 64, True, torch.float32, cuda)
    q, k, v, positions = _inputs(cuda, 3, 2, 2, 64, torch.bfloat16, 8)
    pages = torch.zeros(2, 2, 16, 2, 64, dtype=torch.bfloat16, device=cuda)
    other = torch.zeros_like(pages)
    append_paged_kv(rope, positions.cpu(), k, v, pages, torch.tensor([4, -1, 9], dtype=torch.int32), 16)
    append_paged_kv(rope, positions, k, v, other, torch.tensor([4, -1, 9], device=cuda), 16)
    assert torch.equal(pages, other) and int((pages != 0).any(-1).any(-1).sum()) == 4
    with pytest.raises(IndexError):
        append_paged_kv(rope, positions.cpu(), k, v, pages, torch.tensor([4, -1, 32]), 16)
    with pytest.raises(IndexError):
        append_paged_kv(rope, torch.tensor([0, MAX_POSITION, 1]), k, v, pages, torch.tensor([4, -1, 9]), 16)
    none = append_paged_kv(rope, positions[:0], k[:0], v[:0], pages, positions[:0], 16, query=q[:0])
    assert none.shape == (0, 2, 64)
    cache = PagedKV4.allocate(2, 16, 2, 64, cuda)
    append_paged_kv4(rope, positions[:0], k[:0], v[:0], cache, positions[:0])
    assert gather_paged_kv4(cache, positions[:0]).shape == (2, 0, 2, 64)


def _held(x: np.ndarray):
    """(codes, step, low) of fp32 rows [..., 64 g] by the kernel's fp32 steps, and in numpy's IEEE arithmetic."""
    x = x.reshape(*x.shape[:-1], -1, 64).astype(np.float32)
    low = np.maximum(x.min(-1, keepdims=True), np.float32(-65504))
    step = ((np.minimum(x.max(-1, keepdims=True), np.float32(65504)) - low) * np.float32(1 / 15)).astype(np.float16)
    low16 = low.astype(np.float16)
    with np.errstate(divide="ignore"):
        inverse = np.where(step > 0, np.float32(1) / step.astype(np.float32), np.float32(0))
    codes = np.clip(np.rint((x - low16.astype(np.float32)) * inverse), 0, 15)
    return codes, step, low16


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16, torch.float32])
@pytest.mark.parametrize("tokens,kv_heads,head,rotary,neox,block,pad", [
    (1, 1, 64, 64, True, 16, 0), (50, 3, 128, 128, True, 24, 0), (33, 8, 128, 64, False, 16, 0), (7, 2, 128, 24, True, 1, 1),
    (6007, 3, 128, 128, True, 16, 0), (6007, 5, 128, 64, True, 16, 0), (9001, 5, 64, 32, True, 16, 0), (9001, 5, 64, 64, False, 16, 0)])
def test_append_4_bit(cuda, dtype, tokens, kv_heads, head, rotary, neox, block, pad):
    rope = _rope(head, rotary, neox, torch.float32, cuda)
    q, k, v, positions = _inputs(cuda, tokens, 2, kv_heads, head, dtype, 9, pad)
    v = (v.float() * torch.linspace(0.01, 30, tokens, device=cuda)[:, None, None] - 4).to(dtype)
    if tokens > 5:
        v[3] = 2.5                       # a constant row: step 0
        v[4, 0, :5] = 0                  # an outlier beside zeros
        v[4, 0, 5:64] = 0
        v[4, 0, 9] = 7
        v[5, 0, :60] = 1.5               # beyond fp16's range, where the type goes there: held at its end
        v[5, 0, 7], v[5, 0, 30] = min(torch.finfo(dtype).max, 1e30), max(torch.finfo(dtype).min, -3e38)
        v[6, 0, :64] = -min(torch.finfo(dtype).max, 2e8)
        v[6, 0, 3] = 17.0
    blocks = tokens // block + 2
    slots = _slots(cuda, tokens, blocks * block, 10)
    cache = PagedKV4.allocate(blocks, block, kv_heads, head, cuda)
    cache.codes.random_(0, 256)
    before = cache.codes.clone()
    turned = append_paged_kv4(rope, positions, k, v, cache, slots, query=q)
    _check_turn(turned, q, positions, rope)
    rows = _turn(k, positions, rope, torch.float32)[0].to(dtype)
    got = gather_paged_kv4(cache, slots, torch.float32)
    for plane, x in ((0, rows), (1, v)):
        codes, step, low = _held(x.float().cpu().numpy())
        page, at = slots // block, slots % block
        bytes_ = cache.codes[plane][page, :, at].cpu().numpy()
        have = np.stack((bytes_ & 15, bytes_ >> 4), -1).reshape(codes.shape)
        assert np.array_equal(have, codes)
        pair = cache.scales[plane][page, :, at].cpu().numpy()
        assert np.array_equal(pair[..., 0], step[..., 0]) and np.array_equal(pair[..., 1], low[..., 0])
        value = (low.astype(np.float32) + step.astype(np.float32) * codes.astype(np.float32)).reshape(x.shape)
        assert np.array_equal(got[plane].cpu().numpy(), value)
        step64, low64 = step.astype(np.float64), low.astype(np.float64)
        bound = step64 / 2 + 2.0 ** -11 * (np.abs(low64) + 15 * step64) + 16 * 2.0 ** -25
        held = x.double().cpu().numpy().reshape(codes.shape).clip(-65504, 65504)
        off = np.abs(value.reshape(codes.shape) - held)
        assert (off <= bound * (1 + 1e-5)).all()
    rest = torch.ones(blocks * block, dtype=torch.bool, device=cuda)
    rest[slots] = False
    assert torch.equal(cache.codes.transpose(2, 3).flatten(1, 2)[:, rest], before.transpose(2, 3).flatten(1, 2)[:, rest])


def test_4_bit_extremes(cuda):
    """NaN and infinity make their own group NaN; values past fp16 are held at its end."""
    v = torch.zeros(4, 1, 128, dtype=torch.bfloat16, device=cuda)
    v[0, 0, 3], v[1, 0, 70], v[2, 0, 0], v[3] = torch.nan, torch.inf, 3e38, -1e30
    k = torch.ones_like(v)
    cache = PagedKV4.allocate(1, 4, 1, 128, cuda)
    append_paged_kv4(None, None, k, v, cache, torch.arange(4, device=cuda))
    got = gather_paged_kv4(cache, torch.arange(4, device=cuda), torch.float32)
    assert torch.equal(got[0], torch.ones_like(got[0]))
    nan = got[1].isnan().view(4, 2, 64)
    assert nan[0, 0].all() and nan[1, 1].all() and int(nan.sum()) == 128
    # the fp16 step 65504 / 15 is within 2^-11, so the highest value is within 32 of fp16's end
    assert abs(float(got[1, 2, 0, 0]) - 65504) <= 32 and torch.equal(got[1, 3], torch.full_like(got[1, 3], -65504.0))


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16, torch.float32])
def test_gather_4_bit_views_and_padding(cuda, dtype):
    gen = torch.Generator(device=cuda).manual_seed(2)
    pool = torch.randint(0, 256, (3, 2, 5, 2, 7, 64), generator=gen, device=cuda, dtype=torch.uint8)
    scale_pool = torch.randn(3, 2, 5, 2, 7, 2, 2, generator=gen, device=cuda).half()
    cache = PagedKV4(pool[1], scale_pool[1])  # one layer of a pool
    slots = torch.tensor([0, 34, -1, 35, 8, 8], device=cuda)
    out = torch.full((2, 6, 2, 130), 9.0, device=cuda, dtype=dtype)[..., 1:129]  # rows that are not 16-byte aligned
    got = gather_paged_kv4(cache, slots, dtype, out=out)
    assert got is out
    codes = torch.stack((pool[1] & 15, pool[1] >> 4), -1).flatten(-2).double().unflatten(-1, (2, 64))
    want = (codes * scale_pool[1][..., :1].double() + scale_pool[1][..., 1:].double()).flatten(-2).transpose(2, 3).flatten(1, 2)
    info = torch.finfo(dtype)
    for i, s in enumerate(slots.tolist()):
        if not 0 <= s < 35:
            assert int((got[:, i] != 0).sum()) == 0
            continue
        # one fp32 rounding of the sum, one to the type
        bound = want[:, s].abs() * (info.eps / 2 + 2.0 ** -23) + info.smallest_normal * info.eps
        assert ((got[:, i].double() - want[:, s]).abs() <= bound).all()


def test_append_offsets_past_32_bits(cuda):
    """A plane of more than 4 GiB: the last block lies past a 32-bit byte offset."""
    kv_heads, head, block = 8, 128, 16
    blocks = (1 << 32) // (block * kv_heads * head * 2) + 40
    pages = torch.zeros(2, blocks, block, kv_heads, head, dtype=torch.bfloat16, device=cuda)
    _, k, v, positions = _inputs(cuda, 5, 1, kv_heads, head, torch.bfloat16, 12)
    slots = blocks * block - 1 - torch.arange(5, device=cuda)
    append_paged_kv(None, None, k, v, pages, slots, block)
    assert torch.equal(pages[0].view(-1, kv_heads, head)[slots], k)
    assert torch.equal(pages[1].view(-1, kv_heads, head)[slots], v)
    assert int((pages[0, :10] != 0).sum()) == 0


def test_append_streams_and_graph(cuda):
    rope = _rope(128, 128, True, torch.float32, cuda)
    q, k, v, positions = _inputs(cuda, 20, 4, 2, 128, torch.bfloat16, 13)
    slots = _slots(cuda, 20, 64, 14)
    want, cache_want = torch.zeros(2, 4, 16, 2, 128, dtype=torch.bfloat16, device=cuda), PagedKV4.allocate(4, 16, 2, 128, cuda)
    turned = append_paged_kv(rope, positions, k, v, want, slots, 16, query=q)
    append_paged_kv4(rope, positions, k, v, cache_want, slots)
    side = torch.cuda.Stream(cuda)
    side.wait_stream(torch.cuda.current_stream(cuda))
    pages = torch.zeros_like(want)
    torch.cuda.synchronize()
    on_side = append_paged_kv(rope, positions, k, v, pages, slots, 16, query=q, stream=side)
    side.synchronize()
    assert torch.equal(pages, want) and torch.equal(on_side, turned)
    pages.zero_()
    cache = PagedKV4.allocate(4, 16, 2, 128, cuda)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        in_graph = append_paged_kv(rope, positions, k, v, pages, slots, 16, query=q)
        append_paged_kv4(rope, positions, k, v, cache, slots)
        read = gather_paged_kv4(cache, slots)
    pages.zero_(), cache.codes.zero_(), cache.scales.zero_()
    graph.replay()
    torch.cuda.synchronize()
    assert torch.equal(pages, want) and torch.equal(in_graph, turned) and torch.equal(cache.codes, cache_want.codes)
    assert torch.equal(read, gather_paged_kv4(cache_want, slots))


@pytest.mark.parametrize("pad", [0, 1], ids=["aligned", "unaligned"])
def test_4_bit_groups_at_the_ends_of_bf16(cuda, pad):
    """Finite groups whose ends add up to more than fp32 holds: held at fp16's end, not NaN."""
    top = torch.finfo(torch.bfloat16).max
    x = torch.ones(4, 1, 128 + pad, dtype=torch.bfloat16, device=cuda)[..., pad:]
    x[0], x[1], x[2], x[2, 0, ::2], x[3, 0, :64] = -top, top, top, -top, -2e38
    cache = PagedKV4.allocate(1, 4, 1, 128, cuda)
    append_paged_kv4(None, None, x, x, cache, torch.arange(4, device=cuda))
    want = torch.ones(4, 1, 128, device=cuda)
    want[0], want[1], want[3, 0, :64] = -65504, 65504, -65504
    want[2], want[2, 0, ::2] = 15 * 8736 - 65504, -65504  # a step of fp16(131008 / 15) = 8736
    got = gather_paged_kv4(cache, torch.arange(4, device=cuda), torch.float32)
    assert torch.equal(got[0], want) and torch.equal(got[1], want)


def test_fp16_values_at_its_end_read_back_finite(cuda):
    """A step is rounded, so a group's highest code may stand for more than fp16 holds: read at its end."""
    x = torch.zeros(3, 1, 128, dtype=torch.float16, device=cuda)
    x[0, 0, 5], x[1, 0, 70], x[2, 0, :64:2], x[2, 0, 1:64:2] = 65504.0, -65504.0, 65504.0, -65504.0
    cache, at = PagedKV4.allocate(1, 3, 1, 128, cuda), torch.arange(3, device=cuda)
    append_paged_kv4(None, None, x, x, cache, at)
    wide = gather_paged_kv4(cache, at, torch.float32)
    assert float(wide.max()) > 65504
    for out in (None, torch.empty(2, 3, 1, 129, dtype=torch.float16, device=cuda)[..., 1:]):
        got = gather_paged_kv4(cache, at, torch.float16, out=out)
        assert torch.equal(got, wide.clamp(-65504, 65504).half())
    cache.scales[0, 0, 0, 0, 0, 0], cache.scales[0, 0, 0, 1, 1, 1] = torch.nan, torch.inf  # what is not finite stays so
    got = gather_paged_kv4(cache, at, torch.float16)
    assert bool(got[0, 0, 0, :64].isnan().all()) and bool((got[0, 1, 0, 64:] == torch.inf).all())


def test_rotary_modules_without_a_table_are_refused(cuda):
    bare = SimpleNamespace(head_size=64, rotary_dim=64, is_neox_style=True)
    _, k, v, positions = _inputs(cuda, 3, 1, 2, 64, torch.bfloat16, 15)
    pages, slots = torch.zeros(2, 4, 16, 2, 64, dtype=torch.bfloat16, device=cuda), torch.arange(3, device=cuda)
    with pytest.raises(NotImplementedError, match="cos_sin_cache"):
        append_paged_kv(bare, positions, k, v, pages, slots, 16)
    with pytest.raises(NotImplementedError, match="cos_sin_cache"):
        append_paged_kv4(bare, positions, k, v, PagedKV4.allocate(4, 16, 2, 64, cuda), slots)
    assert int((pages != 0).sum()) == 0
