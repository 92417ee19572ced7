"""Fresh keys and values into the paged cache, rotated on the way, and 4-bit pages.

``append_paged_kv`` writes a step's or a prompt's K and V into the same paged
layouts that ``scatter_paged_kv`` takes, with K (and, if given, the queries)
rotated at their positions in the same launch: what a serving program does
between the projections and the attention, and what the side executor does with
a rotary module, a reshape and two copies.  ``append_paged_kv4`` does the same
into ``PagedKV4`` pages, which hold 4 bits per value; ``gather_paged_kv4`` reads
rows back as values, and ``paged_attention4`` attends to them in place.

No counterpart in cacheblend_vllm, which leaves these steps to vLLM.
CUDA tensors only.
"""

from __future__ import annotations

import contextlib
from dataclasses import dataclass

import torch

from . import _native
from .kv_layout import KVLayer, describe_paged

GROUP = 64  # values of a 4-bit row that share a step and a lowest value


@dataclass(frozen=True)
class PagedKV4:
    """One layer's paged K and V in 4 bits.

    ``codes``: uint8 ``[2, num_blocks, num_heads, block_size, head_size // 2]``, dimension 2i
    of a row in the low nibble of byte i, 2i + 1 in the high one.  ``scales``: float16
    ``[2, num_blocks, num_heads, block_size, head_size // 64, 2]``, each group's step and
    lowest value: a value is ``lowest + step * code``.  Plane 0 is K, plane 1 V.  The rows
    of both are contiguous; the other strides are free (a view of a larger pool will do).
    Head sizes 64 and 128.  Steps and lowest values are finite, but for groups that are not: their
    step is NaN, and whatever sees such a group of V has NaN in its 64 dimensions, of K in all.
    """

    codes: torch.Tensor
    scales: torch.Tensor

    def __post_init__(self) -> None:
        codes, scales = self.codes, self.scales
        shape = codes.shape
        if len(shape) != 5 or shape[0] != 2 or codes.dtype != torch.uint8:
            raise ValueError("codes must be uint8 [2, blocks, heads, block_size, head_size // 2]")
        _, blocks, heads, rows, half = shape
        if half not in (32, 64):
            raise NotImplementedError(f"4-bit pages hold heads of 64 or 128 values, not {2 * half}")
        if scales.dtype != torch.float16 or scales.shape != (2, blocks, heads, rows, half // 32, 2):
            raise ValueError("scales must be float16 [2, blocks, heads, block_size, head_size // 64, 2]")
        if codes.device != scales.device:
            raise ValueError("codes and scales must live on one device")
        if heads == 0 or rows == 0:
            raise ValueError("4-bit pages need at least one head and one row")
        *_, group, pair = scales.stride()
        if codes.stride(4) != 1 or pair != 1 or (half == 64 and group != 2):
            raise ValueError("the rows of 4-bit pages must be contiguous")

    @classmethod
    def allocate(cls, num_blocks: int, block_size: int, num_heads: int, head_size: int,
                 device: torch.device | str = "cuda") -> "PagedKV4":
        """Zeroed pages (every value reads as 0)."""
        if head_size not in (64, 128):
            raise NotImplementedError(f"4-bit pages hold heads of 64 or 128 values, not {head_size}")
        shape = (2, num_blocks, num_heads, block_size)
        return cls(torch.zeros(*shape, head_size // 2, dtype=torch.uint8, device=device),
                   torch.zeros(*shape, head_size // GROUP, 2, dtype=torch.float16, device=device))

    @property
    def num_blocks(self) -> int:
        return int(self.codes.shape[1])

    @property
    def num_heads(self) -> int:
        return int(self.codes.shape[2])

    @property
    def block_size(self) -> int:
        return int(self.codes.shape[3])

    @property
    def head_size(self) -> int:
        return 2 * int(self.codes.shape[4])

    @property
    def device(self) -> torch.device:
        return self.codes.device

    def _pages(self) -> tuple:
        """The pages as the C ABI takes them: pointers and byte strides (block, row, head)."""
        plane, block, head, row, _ = self.codes.stride()
        s_plane, s_block, s_head, s_row, _, _ = self.scales.stride()
        codes, scales = self.codes.data_ptr(), self.scales.data_ptr()
        return (codes, codes + plane, block, row, head, scales, scales + 2 * s_plane, 2 * s_block, 2 * s_row, 2 * s_head)


_HERE = contextlib.nullcontext()
# No Stream object is built (2 us of a decode call).  None on a torch without CUDA bindings, where every
# call refuses its tensors before it needs a stream.
_raw_stream = getattr(torch._C, "_cuda_getCurrentRawStream", None)


def on_device(device: int, stream: torch.cuda.Stream | None):
    """Context in which a call allocates and launches: ``stream``, or the device's current stream."""
    if stream is not None:
        if stream.device.index != device:
            raise ValueError(f"the stream belongs to {stream.device}, the tensors to cuda:{device}")
        return torch.cuda.stream(stream)
    return _HERE if device == torch.cuda.current_device() else torch.cuda.device(device)


def _contiguous_empty(like: torch.Tensor) -> torch.Tensor:
    """A contiguous tensor of ``like``'s shape, type and device."""
    return torch.empty_like(like) if like.is_contiguous() else torch.empty_like(like, memory_format=torch.contiguous_format)


def _index(name: str, index: torch.Tensor, count: int, device: int, low: int | None, high: int) -> torch.Tensor:
    """One int64 per token on ``device``; host values are range-checked first."""
    if index.ndim != 1 or index.numel() != count:
        raise ValueError(f"{name} must hold one entry per token ({count}), got shape {tuple(index.shape)}")
    where = index.get_device()
    if where == device and index.dtype is torch.long and index.is_contiguous():
        return index
    if index.is_floating_point() or index.dtype == torch.bool:
        raise ValueError(f"{name} must be whole numbers, not {index.dtype}")
    if index.device.type == "cpu":
        if count and ((low is not None and int(index.min()) < low) or int(index.max()) >= high):
            raise IndexError(f"{name} out of range: [{int(index.min())}, {int(index.max())}] for {high}")
    elif where != device:
        raise ValueError(f"{name} must live on the host or on cuda:{device}")
    return index.to(device=torch.device("cuda", device), dtype=torch.long).contiguous()


def _check_rows(key: torch.Tensor, value: torch.Tensor, query: torch.Tensor | None) -> tuple:
    """(shape, dtype, device index, strides of key, of value, of query) of rows that go together."""
    shape, dtype, device = key.shape, key.dtype, key.get_device()
    if len(shape) != 3:
        raise ValueError(f"key must be [tokens, heads, head_size], got {tuple(shape)}")
    if value.shape != shape:
        raise ValueError(f"key and value must have the same shape, not {tuple(shape)} and {tuple(value.shape)}")
    if value.dtype is not dtype or value.get_device() != device:
        raise ValueError("value must share the keys' dtype and device")
    of_key, of_value, of_query = key.stride(), value.stride(), (0, 0, 1)
    if query is not None:
        q = query.shape
        if len(q) != 3 or q[0] != shape[0] or q[2] != shape[2]:
            raise ValueError(f"query {tuple(q)} does not match the keys {tuple(shape)}")
        if query.dtype is not dtype or query.get_device() != device:
            raise ValueError("query must share the keys' dtype and device")
        of_query = query.stride()
    if shape[2] > 1 and not (of_key[2] == of_value[2] == of_query[2] == 1):
        raise ValueError("the values of a head must be contiguous in key, value and query")
    if dtype not in _native.DTYPE_CODES:
        _native.dtype_code(dtype)
    return shape, dtype, device, of_key, of_value, of_query


def _page_planes(kv_layer: KVLayer, block_size: int) -> tuple:
    """(K address, V address, shape, strides, dtype, device index) of 16/32-bit pages [blocks, rows, heads, head_size].

    The merged layouts are taken apart by arithmetic: describe_paged's views are most of a
    decode step's call.  Whatever is unusual goes through it."""
    if isinstance(kv_layer, torch.Tensor) and kv_layer.ndim == 5:
        shape, strides = kv_layer.shape, kv_layer.stride()
        key = kv_layer.data_ptr()
        if shape[0] == 2 and 0 < block_size <= shape[2]:
            return (key, key + strides[0] * kv_layer.element_size(), shape[1:], strides[1:], kv_layer.dtype,
                    kv_layer.get_device())
        if shape[1] == 2 and shape[0] != 2 and 0 < block_size <= shape[2]:
            return (key, key + strides[1] * kv_layer.element_size(), (shape[0], *shape[2:]), (strides[0], *strides[2:]),
                    kv_layer.dtype, kv_layer.get_device())
    paged = describe_paged(kv_layer, block_size)
    return (paged.key.data_ptr(), paged.value.data_ptr(), paged.key.shape, paged.key.stride(), paged.dtype,
            paged.key.get_device())


def _rotation(rotary_emb, head_size: int, dtype: torch.dtype, device: int) -> tuple:
    """(table or None, table dtype code, positions it holds, rotary_dim, neox)."""
    if rotary_emb is None:
        return None, _native.DTYPE_CODES[torch.float32], 0, 0, 1
    table = getattr(rotary_emb, "cos_sin_cache", None)
    if table is None:
        raise NotImplementedError("the append needs a rotary module with cos_sin_cache")
    rotary_dim = int(getattr(rotary_emb, "rotary_dim", head_size))
    if rotary_emb.head_size != head_size:
        raise ValueError(f"the rotation is made for heads of {rotary_emb.head_size} values, not {head_size}")
    if table.ndim != 2 or table.shape[1] != rotary_dim or rotary_dim <= 0 or rotary_dim % 2:
        raise ValueError("RoPE cache width does not match rotary_dim")
    if table.get_device() != device:
        raise ValueError("the RoPE cache must live on the keys' device")
    if table.dtype is not torch.float32 and table.dtype is not dtype:
        raise NotImplementedError(f"the RoPE cache must be float32 or {dtype}, not {table.dtype}")
    if not table.is_contiguous():
        table = table.contiguous()
    return table, _native.DTYPE_CODES[table.dtype], table.shape[0], rotary_dim, 1 if rotary_emb.is_neox_style else 0


def _append(entry: str, rotary_emb, positions, key, value, query, rows: tuple, slot_mapping, num_blocks: int,
            block_size: int, pages: tuple, stream) -> torch.Tensor | None:
    (tokens, heads, head_size), dtype, device, of_key, of_value, of_query = rows
    with on_device(device, stream):
        table, table_code, max_position, rotary_dim, neox = _rotation(rotary_emb, head_size, dtype, device)
        slots = _index("slot_mapping", slot_mapping, tokens, device, None, num_blocks * block_size)
        where = 0
        if rotary_dim:
            if positions is None:
                raise ValueError("a rotation needs one position per token")
            positions = _index("positions", positions, tokens, device, 0, max_position)
            where = positions.data_ptr()
        turned, q_heads, q, out = None, 0, 0, 0
        size = key.element_size()
        if query is not None:
            turned = _contiguous_empty(query)
            q_heads, q, out = query.shape[1], query.data_ptr(), turned.data_ptr()
        if tokens == 0:
            return turned
        _native.call_packed(
            entry, device, key.data_ptr(), of_key[0] * size, of_key[1] * size, value.data_ptr(), of_value[0] * size,
            of_value[1] * size, q, of_query[0] * size, of_query[1] * size, out, q_heads * head_size * size,
            head_size * size, tokens, q_heads, heads, head_size, _native.DTYPE_CODES[dtype], where,
            0 if table is None else table.data_ptr(), table_code, max_position, rotary_dim, neox, *pages, num_blocks,
            block_size, slots.data_ptr(), _raw_stream(device))
        return turned


def append_paged_kv(
    rotary_emb,
    positions: torch.Tensor | None,
    key: torch.Tensor,
    value: torch.Tensor,
    kv_layer: KVLayer,
    slot_mapping: torch.Tensor,
    block_size: int,
    query: torch.Tensor | None = None,
    stream: torch.cuda.Stream | None = None,
) -> torch.Tensor | None:
    """Rotate ``key`` at ``positions`` and write it with ``value`` into the pages.

    ``key``, ``value``: ``[tokens, kv_heads, head_size]`` of the cache's type, any token and
    head strides (slices of one projection's output will do).  ``kv_layer``: one of the paged
    layouts of ``scatter_paged_kv`` with rows of ``[kv_heads, head_size]``.  ``slot_mapping``:
    the slot of each token; a NEGATIVE slot marks padding, whose row is not written (unlike
    ``scatter_paged_kv``, where it wraps).  The slots of one call must be distinct, and the rows
    must not lie in the pages themselves.
    ``rotary_emb``: what carries ``cos_sin_cache`` (float32 or the keys' type), ``head_size``,
    ``rotary_dim`` and ``is_neox_style``; None writes the keys as they are.  Returns
    ``query`` ``[tokens, q_heads, head_size]`` rotated at the same positions, in a new tensor,
    or None without one.

    The products and their sum are rounded to fp32 each, and once to the element type; a float32
    table is used as it is (``relocate_key`` rounds it, and each product, to the keys' type).
    Slots and positions on the host are range-checked (IndexError); on the device a slot
    outside the cache, or a position outside the table, leaves the pages as they were (and
    gives a zero query row).
    """
    checked = _check_rows(key, value, query)
    (_, heads, head_size), dtype, device, _, _, _ = checked
    k_pages, v_pages, shape, strides, cache_dtype, cache_device = _page_planes(kv_layer, block_size)
    if device < 0 or cache_device < 0:
        _native.require_cuda(key, *(kv_layer if not isinstance(kv_layer, torch.Tensor) else (kv_layer,)))
    if dtype is not cache_dtype or device != cache_device:
        raise ValueError("keys must match the KV cache dtype and device")
    if len(shape) != 4 or shape[2] != heads or shape[3] != head_size:
        raise ValueError(f"pages {tuple(shape)} do not hold rows of {(heads, head_size)}")
    if strides[3] != 1 and head_size > 1:
        raise ValueError("the values of a head must be contiguous in the pages")
    size = key.element_size()
    return _append("cb_append_paged_kv", rotary_emb, positions, key, value, query, checked, slot_mapping, shape[0],
                   block_size, (k_pages, v_pages, strides[0] * size, strides[1] * size, strides[2] * size), stream)


def append_paged_kv4(
    rotary_emb,
    positions: torch.Tensor | None,
    key: torch.Tensor,
    value: torch.Tensor,
    cache: PagedKV4,
    slot_mapping: torch.Tensor,
    query: torch.Tensor | None = None,
    stream: torch.cuda.Stream | None = None,
) -> torch.Tensor | None:
    """``append_paged_kv`` into 4-bit pages (bf16, fp16 or fp32 keys and values).

    Each row is first rounded to its own type, as 16-bit pages would hold it.  Per group of 64
    values: lowest value and step = (highest - lowest) / 15 in float16, codes rounded to the
    nearest.  Values beyond +-65504 are held at that; a group with a NaN or an infinity reads
    as NaN.
    """
    checked = _check_rows(key, value, query)
    (_, heads, head_size), _, device, _, _, _ = checked
    if device < 0 or not cache.codes.is_cuda:
        _native.require_cuda(cache.codes, key)
    if device != cache.codes.get_device():
        raise ValueError("keys must live on the cache's device")
    _, num_blocks, cache_heads, rows, half = cache.codes.shape
    if heads != cache_heads or head_size != 2 * half:
        raise ValueError(f"the cache holds rows of {(cache_heads, 2 * half)}, not {(heads, head_size)}")
    return _append("cb_append_paged_kv4", rotary_emb, positions, key, value, query, checked, slot_mapping, num_blocks, rows,
                   cache._pages(), stream)


def gather_paged_kv4(
    cache: PagedKV4,
    slot_mapping: torch.Tensor,
    dtype: torch.dtype = torch.bfloat16,
    out: torch.Tensor | None = None,
    stream: torch.cuda.Stream | None = None,
) -> torch.Tensor:
    """The values of 4-bit rows as ``[2, tokens, heads, head_size]`` of ``dtype``.

    A negative slot (padding) reads as zeros; so does, on the device, one outside the cache
    (IndexError for host slots).  A finite value past fp16's end (a step is rounded, so a group's highest
    code may stand for up to 65,536) reads as +-65504 in fp16.
    """
    codes = cache.codes
    device = codes.get_device()
    if device < 0:
        _native.require_cuda(codes)
    _, num_blocks, heads, rows, half = codes.shape
    tokens = slot_mapping.numel()
    shape = (2, tokens, heads, 2 * half)
    if dtype not in _native.DTYPE_CODES:
        _native.dtype_code(dtype)
    if out is not None:
        if out.shape != shape:
            raise ValueError(f"gather output has shape {tuple(out.shape)}, expected {shape}")
        if out.dtype is not dtype or out.get_device() != device:
            raise ValueError("gather output must match the dtype and the cache's device")
        if out.stride(3) != 1:
            raise ValueError("the values of a head must be contiguous in the output")
    with on_device(device, stream):
        slots = _index("slot_mapping", slot_mapping, tokens, device, None, num_blocks * rows)
        result = out if out is not None else torch.empty(shape, dtype=dtype, device=codes.device)
        if tokens == 0:
            return result
        size = result.element_size()
        plane, token, head, _ = result.stride()
        _native.call_packed(
            "cb_gather_paged_kv4", device, *cache._pages(), num_blocks, rows, heads, 2 * half, slots.data_ptr(), tokens,
            result.data_ptr(), plane * size, token * size, head * size, _native.DTYPE_CODES[dtype], _raw_stream(device))
        return result
