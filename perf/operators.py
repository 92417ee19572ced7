"""What the serving operators around the blended cache are measured on.

Four operators, each in a plain torch form (``own`` false) and through the
package's entry points (``own`` true):

* ``append``  -- rotate fresh keys (and queries) and write K / V into 16-bit pages;
* ``append4`` -- the same into pages that hold 4 bits per value, then the written
  rows read back as values;
* ``decode4`` -- attention of single tokens (or a few) over 4-bit pages;
* ``prompt``  -- causal attention of a packed batch of prompts.

Head counts are those of the package's benchmark configurations (32 query heads
on 8 KV heads, 64 on 8, 32 on 4) and their tensor-parallel shards; lengths go
from one token to the benchmark's 98,304-token context.
"""

from __future__ import annotations

import math
import sys
from pathlib import Path
from types import SimpleNamespace

import torch

own = False

PACKAGE = str(Path(__file__).resolve().parents[1] / "pic-kvcache_b200")  # where the package lies, unless it is installed
DEVICE = "cuda"
GROUP = 64  # values of a 4-bit row that share a scale and a lowest value
TYPES = {"bf16": torch.bfloat16, "fp16": torch.float16}


def listed():
    return [
        # one decode step of 64 running requests
        dict(name="append decode", op="append", tokens=64, heads=32, kv_heads=8, head=128, rotary=128, neox=True,
             block=16, padded=0, dtype="bf16"),
        # a padded batch of fp16 prompts: pairs side by side, half of each head rotated, pages of 24 rows
        dict(name="append padded fp16", op="append", tokens=2731, heads=16, kv_heads=4, head=64, rotary=32, neox=False,
             block=24, padded=77, dtype="fp16"),
        # the whole of a long prompt
        dict(name="append prompt", op="append", tokens=16384, heads=32, kv_heads=8, head=128, rotary=128, neox=True,
             block=16, padded=0, dtype="bf16"),
        # one decode step of 200 requests into the 4-bit cache
        dict(name="append4 decode", op="append4", tokens=200, kv_heads=8, head=128, rotary=128, neox=True, block=16,
             dtype="bf16"),
        # a long prompt into the 4-bit cache
        dict(name="append4 prompt", op="append4", tokens=20011, kv_heads=8, head=128, rotary=128, neox=True, block=16,
             dtype="bf16"),
        # one request on one tensor-parallel shard: latency counts
        dict(name="decode4 single", op="decode4", seqs=1, keys=1000, tokens=1, heads=8, kv_heads=2, head=128, block=16,
             dtype="bf16"),
        # a batch of running requests of very different lengths
        dict(name="decode4 batch", op="decode4", seqs=64, keys=8192, tokens=1, heads=32, kv_heads=8, head=128, block=16,
             dtype="bf16"),
        # a few long contexts
        dict(name="decode4 long", op="decode4", seqs=6, keys=98304, tokens=1, heads=32, kv_heads=4, head=128, block=32,
             dtype="bf16"),
        # drafted tokens checked together, small heads, odd pages
        dict(name="decode4 several fp16", op="decode4", seqs=23, keys=5003, tokens=4, heads=16, kv_heads=4, head=64,
             block=24, dtype="fp16"),
        # one short prompt: latency counts
        dict(name="prompt short", op="prompt", seqs=1, tokens=301, prefix=0, heads=32, kv_heads=8, head=128, dtype="bf16"),
        # several prompts of different lengths, some behind a cached prefix
        dict(name="prompt packed fp16", op="prompt", seqs=9, tokens=8500, prefix=500, heads=32, kv_heads=4, head=128,
             dtype="fp16"),
        # one long prompt
        dict(name="prompt long", op="prompt", seqs=1, tokens=16384, prefix=0, heads=32, kv_heads=8, head=128, dtype="bf16"),
    ]


def _between(rng, low, high):
    return min(high, int(math.exp(rng.uniform(math.log(low), math.log(high + 1)))))


def draw(rng):
    op = rng.choice(("append", "append4", "decode4", "prompt"))
    dtype = rng.choice(("bf16", "fp16"))
    block = rng.choice((8, 16, 16, 24, 32, 64, 128))
    head = rng.choice((64, 128, 128))
    kv_heads = rng.choice((1, 2, 4, 8))
    heads = kv_heads * rng.choice((1, 2, 3, 4, 5, 7, 8))
    if op == "append":
        return dict(op=op, tokens=_between(rng, 1, 16000), heads=min(heads, 32) // kv_heads * kv_heads, kv_heads=kv_heads,
                    head=head, rotary=rng.choice((head, head, head // 2)), neox=rng.random() < 0.7, block=block,
                    padded=rng.choice((0, 0, 5, 61)), dtype=dtype)
    if op == "append4":
        return dict(op=op, tokens=_between(rng, 1, 20000), kv_heads=kv_heads, head=head,
                    rotary=rng.choice((head, head, head // 2)), neox=rng.random() < 0.7, block=block, dtype=dtype)
    if op == "decode4":
        seqs = _between(rng, 1, 128)
        tokens = rng.choice((1, 1, 1, 2, 5))
        keys = _between(rng, tokens, min(98304, 2000000 // (seqs * kv_heads)))
        return dict(op=op, seqs=seqs, keys=keys, tokens=tokens, heads=heads, kv_heads=kv_heads,
                    head=head, block=block, dtype=dtype)
    tokens = _between(rng, 16, 8000)
    seqs = _between(rng, 1, min(40, tokens))
    return dict(op=op, seqs=seqs, tokens=tokens, prefix=rng.choice((0, 0, 100, 700 if seqs <= 10 else 60)),
                heads=heads, kv_heads=kv_heads, head=head, dtype=dtype)


# ------------------------------------------------------------------ inputs
def _table(rotary, positions):
    """cos in the first half of a row, sin in the second, as a rotary module keeps them."""
    inverse = 1.0 / (1e6 ** (torch.arange(0, rotary, 2, dtype=torch.float64, device=DEVICE) / rotary))
    angles = torch.arange(positions, dtype=torch.float64, device=DEVICE)[:, None] * inverse[None, :]
    return torch.cat((angles.cos(), angles.sin()), dim=-1).float()


def _lengths(gen, count, total, least):
    """``count`` lengths of very different size that sum to ``total``."""
    weight = torch.rand(count, generator=gen) ** 2 + 0.02
    spread = (weight / weight.sum() * (total - least * count)).long() + least
    spread[0] += total - int(spread.sum())
    return spread


def _starts(lengths):
    return torch.cat((torch.zeros(1, dtype=torch.long), lengths.cumsum(0))).to(torch.int32).to(DEVICE)


def _padding(case):
    return min(case.get("padded", 0), case["tokens"] - 1)


def prepare(case, seed):
    gen = torch.Generator(device=DEVICE).manual_seed(seed)
    host = torch.Generator().manual_seed(seed)
    dtype = TYPES[case["dtype"]]
    head, kv_heads = case["head"], case["kv_heads"]

    def normal(*shape):
        return torch.randn(*shape, generator=gen, device=DEVICE, dtype=dtype)

    if case["op"] in ("append", "append4"):
        tokens, block = case["tokens"], case["block"]
        blocks = (tokens + tokens // 4) // block + 2
        heads = case.get("heads", 0)
        fused = normal(tokens, (heads + 2 * kv_heads) * head)  # one projection's output, cut into q, k, v
        q, k, v = fused.split([heads * head, kv_heads * head, kv_heads * head], dim=-1)
        slots = torch.randperm(blocks * block, generator=gen, device=DEVICE)[:tokens]
        padded = _padding(case)
        if padded:
            slots[tokens - padded:] = -1
        state = SimpleNamespace(
            op=case["op"], block=block, slots=slots, dtype=dtype,
            positions=torch.randint(0, 40000, (tokens,), generator=gen, device=DEVICE),
            key=k.unflatten(-1, (kv_heads, head)), value=v.unflatten(-1, (kv_heads, head)),
            query=q.unflatten(-1, (heads, head)) if heads else None,
            rope=SimpleNamespace(head_size=head, rotary_dim=case["rotary"], is_neox_style=case["neox"],
                                 cos_sin_cache=_table(case["rotary"], 40960)))
        if case["op"] == "append":
            state.pages = normal(2, blocks, block, kv_heads, head)
        else:
            state.codes = torch.zeros(2, blocks, kv_heads, block, head // 2, dtype=torch.uint8, device=DEVICE)
            state.scales = torch.zeros(2, blocks, kv_heads, block, head // GROUP, 2, dtype=torch.float16, device=DEVICE)
        return state
    if case["op"] == "decode4":
        seqs, block = case["seqs"], case["block"]
        lens = (torch.rand(seqs, generator=host) ** 2 * case["keys"]).long().clamp_(min=case["tokens"])
        lens[0] = case["keys"]
        width = -(-case["keys"] // block)
        blocks = int((-(-lens // block)).sum()) + 3
        order = torch.randperm(blocks, generator=host).to(torch.int32)
        table = torch.zeros(seqs, width, dtype=torch.int32)
        used = 0
        for i, n in enumerate((-(-lens // block)).tolist()):
            table[i, :n] = order[used:used + n]
            used += n
        counts = torch.full((seqs,), case["tokens"])
        if case["tokens"] > 1:
            counts = (case["tokens"] - torch.arange(seqs) % case["tokens"])[torch.randperm(seqs, generator=host)]
        scales = torch.rand(2, blocks, kv_heads, block, head // GROUP, 2, generator=gen, device=DEVICE)
        scales[..., 0] = scales[..., 0] * 0.2 + 0.15
        scales[..., 1] = scales[..., 1] * -1.5 - 1.2
        return SimpleNamespace(
            op="decode4", block=block, most=case["tokens"], scale=head ** -0.5, scales=scales.half(),
            codes=torch.randint(0, 256, (2, blocks, kv_heads, block, head // 2), generator=gen, device=DEVICE,
                                dtype=torch.uint8),
            table=table.to(DEVICE), lens=lens.to(torch.int32).to(DEVICE),
            start=_starts(counts) if case["tokens"] > 1 else None, query=normal(int(counts.sum()), case["heads"], head))
    seqs, tokens = case["seqs"], case["tokens"]
    lengths = _lengths(host, seqs, tokens, 1)
    prefix = torch.randint(0, case["prefix"] + 1, (seqs,), generator=host) if case["prefix"] else torch.zeros(seqs, dtype=torch.long)
    keys = int((lengths + prefix).sum())
    return SimpleNamespace(
        op="prompt", scale=head ** -0.5, query=normal(tokens, case["heads"], head), key=normal(keys, kv_heads, head),
        value=normal(keys, kv_heads, head), start=_starts(lengths),
        key_start=_starts(lengths + prefix) if case["prefix"] else None)


# ------------------------------------------------------------------ the plain forms
def _rotated(x, positions, rope):
    table = rope.cos_sin_cache[positions].float()[:, None, :]
    width = rope.rotary_dim
    cos, sin = table[..., :width // 2], table[..., width // 2:]
    x = x.float()
    turn, rest = x[..., :width], x[..., width:]
    if rope.is_neox_style:
        a, b = turn[..., :width // 2], turn[..., width // 2:]
        turn = torch.cat((a * cos - b * sin, b * cos + a * sin), dim=-1)
    else:
        a, b = turn[..., ::2], turn[..., 1::2]
        turn = torch.stack((a * cos - b * sin, b * cos + a * sin), dim=-1).flatten(-2)
    return torch.cat((turn, rest), dim=-1)


def _append(s):
    k = _rotated(s.key, s.positions, s.rope).to(s.dtype)
    kept = s.slots >= 0
    where = s.slots[kept]
    s.pages[0][where // s.block, where % s.block] = k[kept]
    s.pages[1][where // s.block, where % s.block] = s.value[kept]
    return {"pages": s.pages, "query": _rotated(s.query, s.positions, s.rope).to(s.dtype)}


def _held(x):
    """The values that 4 bits hold of ``x``: per group of 64 a lowest value and a step in fp16, codes 0 to 15."""
    groups = x.float().unflatten(-1, (-1, GROUP))
    low = groups.amin(-1, keepdim=True)
    step = ((groups.amax(-1, keepdim=True) - low) / 15).half().float()
    low = low.half().float()
    codes = ((groups - low) * torch.where(step > 0, 1 / step, 0)).round().clamp(0, 15)
    return (low + step * codes).flatten(-2)


def _append4(s):
    k = _rotated(s.key, s.positions, s.rope).to(s.dtype)
    return torch.stack((_held(k), _held(s.value))).to(s.dtype)


def _values(codes, scales, real):
    codes = torch.stack((codes & 15, codes >> 4), dim=-1).flatten(-2).to(real)
    scales = scales.to(real)
    return (codes.unflatten(-1, (-1, GROUP)) * scales[..., :1] + scales[..., 1:]).flatten(-2)


def _decode4(s):
    seqs, width = s.table.shape
    at = torch.arange(width * s.block, device=DEVICE)
    pages, rows = s.table[:, at // s.block].long(), (at % s.block).expand(seqs, -1)
    k = _values(s.codes[0][pages, :, rows], s.scales[0][pages, :, rows], torch.float32)  # [seq, key, head, value]
    kv_heads, head = k.shape[2:]
    start = s.start.long() if s.start is not None else torch.arange(seqs + 1, device=DEVICE)
    counts = start[1:] - start[:-1]
    step = torch.arange(s.most, device=DEVICE)
    token = (start[:-1, None] + step).clamp(max=s.query.shape[0] - 1)
    q = s.query.float()[token].unflatten(2, (kv_heads, -1))  # [seq, token, kv head, group, value]
    last = (s.lens - counts)[:, None] + step  # the last key that a token sees
    seen = (at <= last[..., None])[:, None, None]  # [seq, 1, 1, token, key]
    w = torch.einsum("bthgd,blhd->bhgtl", q, k).mul_(s.scale).masked_fill_(~seen, -torch.inf)
    p = (w - w.amax(-1, keepdim=True)).exp()
    p = p / p.sum(-1, keepdim=True)
    v = _values(s.codes[1][pages, :, rows], s.scales[1][pages, :, rows], torch.float32)
    out = torch.einsum("bhgtl,blhd->bthgd", p, v).flatten(2, 3)
    return out[step < counts[:, None]].to(s.query.dtype)


def _prompt(s):
    key_start = s.key_start if s.key_start is not None else s.start
    tokens, keys = s.query.shape[0], s.key.shape[0]
    at_q, at_k = torch.arange(tokens, device=DEVICE), torch.arange(keys, device=DEVICE)
    seq_q = torch.searchsorted(s.start[1:].long(), at_q, right=True)
    seq_k = torch.searchsorted(key_start[1:].long(), at_k, right=True)
    last = at_q - s.start[seq_q + 1] + key_start[seq_q + 1]  # the last key that a token sees
    seen = (seq_q[:, None] == seq_k) & (at_k <= last[:, None])
    kv_heads = s.key.shape[1]
    q = s.query.float().unflatten(1, (kv_heads, -1))
    out = torch.empty_like(s.query).unflatten(1, (kv_heads, -1))
    for h in range(kv_heads):
        w = torch.einsum("qgd,kd->gqk", q[:, h], s.key[:, h].float()).mul_(s.scale).masked_fill_(~seen, -torch.inf)
        p = (w - w.amax(-1, keepdim=True)).exp_()
        p /= p.sum(-1, keepdim=True)
        out[:, h] = torch.einsum("gqk,kd->qgd", p, s.value[:, h].float())
    return out.flatten(1, 2)


def _own(s):
    if PACKAGE not in sys.path:
        sys.path.insert(0, PACKAGE)
    if s.op == "append":
        from cacheblend_b200 import append_paged_kv

        query = append_paged_kv(s.rope, s.positions, s.key, s.value, s.pages, s.slots, s.block, query=s.query)
        return {"pages": s.pages, "query": query}
    if s.op == "append4":
        from cacheblend_b200 import PagedKV4, append_paged_kv4, gather_paged_kv4

        cache = PagedKV4(s.codes, s.scales)
        append_paged_kv4(s.rope, s.positions, s.key, s.value, cache, s.slots)
        return gather_paged_kv4(cache, s.slots, s.dtype)
    if s.op == "decode4":
        from cacheblend_b200 import PagedKV4, paged_attention4

        return paged_attention4(s.query, PagedKV4(s.codes, s.scales), s.table, s.lens, s.scale, query_start=s.start)
    from cacheblend_b200 import prompt_attention

    return prompt_attention(s.query, s.key, s.value, s.start, s.scale, key_start=s.key_start)


def run(state):
    if own:
        return _own(state)
    return {"append": _append, "append4": _append4, "decode4": _decode4, "prompt": _prompt}[state.op](state)


# ------------------------------------------------------------------ what a pass cannot do without
def _seen(case):
    """Keys that a decode case reads on average (lengths are squares of even draws, the first one whole)."""
    return case["keys"] + (case["seqs"] - 1) * (case["keys"] / 3 + 0.5)


def work(case):
    head, kv_heads = case["head"], case["kv_heads"]
    if case["op"] == "append":
        rows, turned = case["tokens"] - _padding(case), case["heads"] + kv_heads
        return {"bytes": (case["tokens"] * case["heads"] + rows * 2 * kv_heads) * head * 4 + case["tokens"] * (16 + 4 * case["rotary"]),
                "flops": 3 * case["tokens"] * turned * case["rotary"]}
    if case["op"] == "append4":
        values = 2 * case["tokens"] * kv_heads * head
        # values in, held, read back, values out
        return {"bytes": values * (2 + 2 * (0.5 + 4 / GROUP) + 2) + case["tokens"] * (16 + 4 * case["rotary"]), "flops": 8 * values}
    if case["op"] == "decode4":
        keys, tokens = _seen(case), case["seqs"] * (1 + case["tokens"]) / 2
        return {"bytes": 2 * keys * kv_heads * head * (0.5 + 4 / GROUP) + 4 * tokens * case["heads"] * head,
                "flops": 4 * keys * (1 + case["tokens"]) / 2 * case["heads"] * head}
    # pairs of a token and a key that it sees, from the same lengths that seed 0 draws
    gen = torch.Generator().manual_seed(0)
    lengths = _lengths(gen, case["seqs"], case["tokens"], 1).double()
    pairs = float((lengths * (lengths + 1) / 2 + lengths * case["prefix"] / 2).sum())
    keys = case["tokens"] + case["seqs"] * case["prefix"] / 2
    return {"bytes": 4 * head * (case["tokens"] * case["heads"] + keys * kv_heads), "flops": 4 * head * case["heads"] * pairs}


# ------------------------------------------------------------------ in 64 bits
def _turned64(x, positions, rope):
    """Rotation as a product of complex numbers."""
    width = rope.rotary_dim
    row = rope.cos_sin_cache.double()[positions]
    turn = torch.complex(row[:, :width // 2], row[:, width // 2:])[:, None, :]
    x = x.double()
    out = x.clone()
    first, second = (slice(0, width // 2), slice(width // 2, width)) if rope.is_neox_style else (slice(0, width, 2), slice(1, width, 2))
    z = torch.complex(x[..., first], x[..., second]) * turn
    out[..., first], out[..., second] = z.real, z.imag
    return out


def _attend64(q, k, v, scale, last):
    """q [token, head, value] over k, v [key, kv head, value]; token t sees the keys 0 to last[t]."""
    kv_heads = k.shape[1]
    q = q.double().unflatten(1, (kv_heads, -1))
    out = torch.zeros_like(q)
    hidden = torch.arange(k.shape[0], device=k.device)[None, :] > last[:, None]
    for h in range(kv_heads):
        for g in range(q.shape[2]):
            w = (q[:, h, g] @ k[:, h].double().T) * scale
            w[hidden] = -math.inf
            out[:, h, g] = torch.softmax(w, dim=-1) @ v[:, h].double()
    return out.flatten(1, 2)


def exact(case, seed):
    s = prepare(case, seed)
    if s.op == "append":
        pages = s.pages.double()
        flat = pages.view(2, -1, *pages.shape[3:])
        real = (s.slots >= 0).nonzero().flatten()
        flat[0].index_copy_(0, s.slots[real], _turned64(s.key, s.positions, s.rope)[real])
        flat[1].index_copy_(0, s.slots[real], s.value.double()[real])
        return {"pages": pages, "query": _turned64(s.query, s.positions, s.rope)}
    if s.op == "append4":
        held = []
        for x in (_turned64(s.key, s.positions, s.rope).to(s.dtype), s.value):
            x = x.double().reshape(*x.shape[:2], -1, GROUP)
            low, high = x.min(-1).values, x.max(-1).values
            step, low = ((high - low) / 15).half().double()[..., None], low.half().double()[..., None]
            codes = torch.where(step > 0, (x - low) / step, torch.zeros_like(x)).round().clamp(0, 15)
            held.append((codes * step + low).flatten(-2))
        return torch.stack(held)
    if s.op == "decode4":
        starts = s.start.tolist() if s.start is not None else list(range(len(s.lens) + 1))
        out = []
        for i, n in enumerate(s.lens.tolist()):
            pages = s.table[i, :-(-n // s.block)].long()
            k, v = (_values(s.codes[x][pages], s.scales[x][pages], torch.float64).transpose(1, 2).flatten(0, 1)[:n] for x in (0, 1))
            count = starts[i + 1] - starts[i]
            last = torch.arange(n - count, n, device=DEVICE)
            out.append(_attend64(s.query[starts[i]:starts[i + 1]], k, v, s.scale, last))
        return torch.cat(out)
    starts = s.start.tolist()
    key_starts = s.key_start.tolist() if s.key_start is not None else starts
    out = []
    for a, b, c, d in zip(starts, starts[1:], key_starts, key_starts[1:]):
        last = torch.arange(d - c - (b - a), d - c, device=DEVICE)
        out.append(_attend64(s.query[a:b], s.key[c:d], s.value[c:d], s.scale, last))
    return torch.cat(out)
