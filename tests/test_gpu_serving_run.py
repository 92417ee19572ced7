"""The operators together, as a serving loop makes them: two prompts of different length are
rotated, appended to 16-bit and 4-bit pages and attended packed; then decode steps append one
token per sequence and attend over the 4-bit pages.  Each output is compared with attention in
64 bits over what the pages hold, and the 4-bit pages with the 16-bit ones."""

from __future__ import annotations

import math
from types import SimpleNamespace

import pytest
import torch

from cacheblend_b200 import (PagedKV4, append_paged_kv, append_paged_kv4, gather_paged_kv, gather_paged_kv4,
                             paged_attention4, prompt_attention)

pytestmark = pytest.mark.gpu

HEADS, KV_HEADS, HEAD, BLOCK = 16, 4, 128, 16


def _attend(q, k, v, scale):
    """q [n, heads, head] over k, v [keys, kv_heads, head], the queries last; 64 bits."""
    n, keys = q.shape[0], k.shape[0]
    hidden = torch.arange(keys, device=q.device)[None] > (torch.arange(n, device=q.device) + keys - n)[:, None]
    k, v = (x.double().repeat_interleave(HEADS // KV_HEADS, 1) for x in (k, v))
    w = torch.einsum("qhd,khd->hqk", q.double(), k) * scale
    p = torch.softmax(w.masked_fill(hidden, -math.inf), -1)
    return torch.einsum("hqk,khd->qhd", p, v), torch.einsum("hqk,khd->qhd", p, v.abs())


def _close(got, want, mass):
    """bf16 keeps 8 bits: a rounding is off by at most half a step, finfo.eps / 2 = 2^-8 relative.
    One for each probability (prompt; the 4-bit decode rounds its factors to fp16, which is less)
    and one for the result, half as much again for fp32 sums and exp2."""
    half_step = torch.finfo(torch.bfloat16).eps / 2
    worst = float(((got.double() - want).abs() / (half_step * (1.5 * mass + want.abs()) + 1e-6)).max())
    assert worst <= 1, worst


@pytest.mark.parametrize("captured", [False, True], ids=["eager", "graph"])
def test_prompts_then_decode(cuda, captured):
    gen = torch.Generator(device=cuda).manual_seed(30)
    inverse = 1.0 / (1e6 ** (torch.arange(0, HEAD, 2, dtype=torch.float64) / HEAD))
    angles = torch.arange(512, dtype=torch.float64)[:, None] * inverse
    rope = SimpleNamespace(head_size=HEAD, rotary_dim=HEAD, is_neox_style=True,
                           cos_sin_cache=torch.cat((angles.cos(), angles.sin()), -1).float().to(cuda))
    scale = HEAD ** -0.5
    lengths = [130, 37]
    pages = torch.zeros(2, 16, BLOCK, KV_HEADS, HEAD, dtype=torch.bfloat16, device=cuda)
    cache = PagedKV4.allocate(16, BLOCK, KV_HEADS, HEAD, cuda)
    table = torch.tensor([[4, 9, 1, 0, 15, 7, 8, 2, 3], [10, 5, 12, 6, 11, 13, 14, 0, 0]], dtype=torch.int32, device=cuda)

    def slots_of(seq, positions):
        return table[seq].long()[positions // BLOCK] * BLOCK + positions % BLOCK

    def projected(n):
        fused = torch.randn(n, (HEADS + 2 * KV_HEADS) * HEAD, generator=gen, device=cuda).to(torch.bfloat16)
        q, k, v = fused.split([HEADS * HEAD, KV_HEADS * HEAD, KV_HEADS * HEAD], -1)
        return q.unflatten(-1, (HEADS, HEAD)), k.unflatten(-1, (KV_HEADS, HEAD)), v.unflatten(-1, (KV_HEADS, HEAD))

    # the prompts: one padded batch, eight rows of padding behind
    total = sum(lengths) + 8
    q, k, v = projected(total)
    positions = torch.cat([*(torch.arange(n, device=cuda) for n in lengths), torch.zeros(8, dtype=torch.long, device=cuda)])
    slots = torch.cat([*(slots_of(i, torch.arange(n, device=cuda)) for i, n in enumerate(lengths)),
                       torch.full((8,), -1, device=cuda)])
    start = torch.tensor([0, lengths[0], sum(lengths)], dtype=torch.int32, device=cuda)
    turned = append_paged_kv(rope, positions, k, v, pages, slots, BLOCK, query=q)
    turned4 = append_paged_kv4(rope, positions, k, v, cache, slots, query=q)
    assert torch.equal(turned, turned4)
    written = slots[:sum(lengths)]
    rows = gather_paged_kv(pages, written, BLOCK)
    held = gather_paged_kv4(cache, written, torch.float32)
    # a code is off by half a step at most, a step is a fifteenth of its group's range; the pair's
    # fp16 rounding and its fp32 sum come on top
    spread = rows.float().unflatten(-1, (2, 64))
    step = (spread.amax(-1) - spread.amin(-1)) / 15
    off = (held - rows.float()).abs().unflatten(-1, (2, 64)).amax(-1)
    assert bool((off <= 0.51 * step + 2.0 ** -11 * (spread.abs().amax(-1) + 15 * step)).all())
    out = prompt_attention(turned, rows[0].contiguous(), rows[1].contiguous(), start, scale,
                           out=torch.full_like(turned, 3.0), key_start=start)
    assert (out[sum(lengths):] == 3).all()
    for i, n in enumerate(lengths):
        part = slice(int(start[i]), int(start[i]) + n)
        _close(out[part], *_attend(turned[part], rows[0][part], rows[1][part], scale))

    # decode steps over the 4-bit pages; captured: one graph, replayed with each step's inputs
    lens = torch.tensor(lengths, dtype=torch.int32, device=cuda)
    step_q, step_k, step_v = projected(2)
    step_position, step_slot = torch.zeros(2, dtype=torch.long, device=cuda), torch.zeros(2, dtype=torch.long, device=cuda)

    def decode():
        query = append_paged_kv4(rope, step_position, step_k, step_v, cache, step_slot, query=step_q)
        return query, paged_attention4(query, cache, table, lens, scale)

    def next_inputs():
        for have, new in zip((step_q, step_k, step_v), projected(2)):
            have.copy_(new)
        step_position.copy_(lens)
        step_slot.copy_(torch.stack([slots_of(i, step_position[i]) for i in range(2)]))
        lens.add_(1)

    graph = None
    for step_index in range(5):
        next_inputs()
        if captured:
            if graph is None:
                graph = torch.cuda.CUDAGraph()
                with torch.cuda.graph(graph):
                    query, got = decode()
            graph.replay()
        else:
            query, got = decode()
        torch.cuda.synchronize()
        for i in range(2):
            seen = slots_of(i, torch.arange(int(lens[i]), device=cuda))
            keys, values = gather_paged_kv4(cache, seen, torch.float32)
            _close(got[i:i + 1], *_attend(query[i:i + 1], keys, values, scale))
