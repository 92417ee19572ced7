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
    Head sizes 64 and 128.
    """

    codes: torch.Tensor
    scales: torch.Tensor

    def __post_init__(self) -> None:
        codes, scales = self.codes, self.scales
        if codes.ndim != 5 or codes.shape[0] != 2 or codes.dtype != torch.uint8:
            raise ValueError("codes must be uint8 [2, blocks, heads, block_size, head_size // 2]")
        if codes.shape[4] not in (32, 64):
            raise NotImplementedError(f"4-bit pages hold heads of 64 or 128 values, not {2 * codes.shape[4]}")
        if scales.dtype != torch.float16 or tuple(scales.shape) != (*codes.shape[:4], codes.shape[4] * 2 // GROUP, 2):
            raise ValueError("scales must be float16 [2, blocks, heads, block_size, head_size // 64, 2]")
        if codes.device != scales.device:
            raise ValueError("codes and scales must live on one device")
        if codes.shape[2] == 0 or codes.shape[3] == 0:
            raise ValueError("4-bit pages need at least one head and one row")
        if codes.stride(4) != 1 or scales.stride(5) != 1 or (scales.shape[4] > 1 and scales.stride(4) != 2):
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


def on_device(device: torch.device, stream: torch.cuda.Stream | None):
    """Context in which a call allocates and launches: ``stream``, or the device's current stream."""
    if stream is not None:
        if stream.device != device:
            raise ValueError(f"the stream belongs to {stream.device}, the tensors to {device}")
        return torch.cuda.stream(stream)
    return _HERE if device.index == torch.cuda.current_device() else torch.cuda.device(device)


def current_handle() -> int:
    """The current device's current stream, without building a Stream object (2 us of a decode call)."""
    return torch._C._cuda_getCurrentRawStream(torch.cuda.current_device())


def _index(name: str, index: torch.Tensor, count: int, device: torch.device, low: int | None, high: int) -> torch.Tensor:
    """One int64 per token on ``device``; host values are range-checked first."""
    if index.ndim != 1 or index.numel() != count:
        raise ValueError(f"{name} must hold one entry per token ({count}), got shape {tuple(index.shape)}")
    if index.is_floating_point() or index.dtype == torch.bool:
        raise ValueError(f"{name} must be whole numbers, not {index.dtype}")
    if index.device.type == "cpu" and count:
        if (low is not None and int(index.min()) < low) or int(index.max()) >= high:
            raise IndexError(f"{name} out of range: [{int(index.min())}, {int(index.max())}] for {high}")
    elif index.device.type != "cpu" and index.device != device:
        raise ValueError(f"{name} must live on the host or on {device}")
    if index.dtype != torch.long or index.device != device:
        index = index.to(device=device, dtype=torch.long)
    return index.contiguous()


def _rows(name: str, tensor: torch.Tensor, like: torch.Tensor) -> None:
    if tensor.ndim != 3:
        raise ValueError(f"{name} must be [tokens, heads, head_size], got {tuple(tensor.shape)}")
    if tensor.shape[0] != like.shape[0] or tensor.shape[2] != like.shape[2]:
        raise ValueError(f"{name} {tuple(tensor.shape)} does not match the keys {tuple(like.shape)}")
    if tensor.dtype != like.dtype or tensor.device != like.device:
        raise ValueError(f"{name} must share the keys' dtype and device")
    if tensor.shape[2] > 1 and tensor.stride(2) != 1:
        raise ValueError(f"the values of a head of {name} must be contiguous")


def _rotation(rotary_emb, head_size: int, key: torch.Tensor) -> tuple:
    """(table or None, table dtype code, positions it holds, rotary_dim, neox)."""
    if rotary_emb is None:
        return None, _native.DTYPE_CODES[torch.float32], 0, 0, 1
    table = rotary_emb.cos_sin_cache
    rotary_dim = int(getattr(rotary_emb, "rotary_dim", head_size))
    if int(rotary_emb.head_size) != head_size:
        raise ValueError(f"the rotation is made for heads of {rotary_emb.head_size} values, not {head_size}")
    if table.ndim != 2 or table.shape[1] != rotary_dim or rotary_dim <= 0 or rotary_dim % 2:
        raise ValueError("RoPE cache width does not match rotary_dim")
    if table.device != key.device:
        raise ValueError("the RoPE cache must live on the keys' device")
    if table.dtype not in (torch.float32, key.dtype):
        raise NotImplementedError(f"the RoPE cache must be float32 or {key.dtype}, not {table.dtype}")
    return table.contiguous(), _native.dtype_code(table.dtype), int(table.shape[0]), rotary_dim, \
        int(bool(rotary_emb.is_neox_style))


def _append(entry: str, rotary_emb, positions, key, value, query, slot_mapping, num_slots: int, block_size: int,
            num_blocks: int, pages: tuple, stream) -> torch.Tensor | None:
    tokens, heads, head_size = key.shape
    table, table_code, max_position, rotary_dim, neox = _rotation(rotary_emb, head_size, key)
    with on_device(key.device, stream):
        slots = _index("slot_mapping", slot_mapping, tokens, key.device, None, num_slots)
        where = None
        if rotary_dim:
            if positions is None:
                raise ValueError("a rotation needs one position per token")
            where = _index("positions", positions, tokens, key.device, 0, max_position)
        turned = None if query is None else torch.empty(query.shape, dtype=query.dtype, device=query.device)
        if tokens == 0:
            return turned
        size = key.element_size()
        strides = [s * size for t in (key, value) for s in t.stride()[:2]]
        q = (0, 0, 0, 0, 0, 0) if query is None else (
            query.data_ptr(), query.stride(0) * size, query.stride(1) * size,
            turned.data_ptr(), turned.stride(0) * size, turned.stride(1) * size)
        _native.call(entry, key.data_ptr(), strides[0], strides[1], value.data_ptr(), strides[2], strides[3], *q, tokens,
                     0 if query is None else query.shape[1], heads, head_size, _native.dtype_code(key.dtype),
                     0 if where is None else where.data_ptr(), 0 if table is None else table.data_ptr(), table_code,
                     max_position, rotary_dim, neox, *pages, num_blocks, block_size, slots.data_ptr(),
                     current_handle())
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
    ``scatter_paged_kv``, where it wraps).  The slots of one call must be distinct.
    ``rotary_emb``: what carries ``cos_sin_cache`` (float32 or the keys' type), ``head_size``,
    ``rotary_dim`` and ``is_neox_style``; None writes the keys as they are.  Returns
    ``query`` ``[tokens, q_heads, head_size]`` rotated at the same positions, in a new tensor,
    or None without one.

    The products and their sum are rounded to fp32 each, and once to the element type.
    Slots and positions on the host are range-checked (IndexError); on the device a slot
    outside the cache, or a position outside the table, leaves the pages as they were (and
    gives a zero query row).
    """
    _rows("key", key, key)
    _rows("value", value, key)
    if value.shape != key.shape:
        raise ValueError("key and value must have the same shape")
    if query is not None:
        _rows("query", query, key)
    paged = describe_paged(kv_layer, block_size)
    _native.require_cuda(paged.key, key)
    _native.dtype_code(key.dtype)
    if key.dtype != paged.dtype or key.device != paged.device:
        raise ValueError("keys must match the KV cache dtype and device")
    if paged.key.ndim != 4 or tuple(paged.key.shape[2:]) != tuple(key.shape[1:]):
        raise ValueError(f"pages {tuple(paged.key.shape)} do not hold rows of {tuple(key.shape[1:])}")
    if paged.key.shape[3] > 1 and paged.key.stride(3) != 1:
        raise ValueError("the values of a head must be contiguous in the pages")
    pages = (paged.key.data_ptr(), paged.value.data_ptr(), paged.block_stride, paged.slot_stride,
             paged.key.stride(2) * key.element_size())
    return _append("cb_append_paged_kv", rotary_emb, positions, key, value, query, slot_mapping,
                   paged.num_blocks * paged.block_size, paged.block_size, paged.num_blocks, pages, stream)


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
    _rows("key", key, key)
    _rows("value", value, key)
    if value.shape != key.shape:
        raise ValueError("key and value must have the same shape")
    if query is not None:
        _rows("query", query, key)
    _native.require_cuda(cache.codes, key)
    _native.dtype_code(key.dtype)
    if key.device != cache.device:
        raise ValueError("keys must live on the cache's device")
    if tuple(key.shape[1:]) != (cache.num_heads, cache.head_size):
        raise ValueError(f"the cache holds rows of {(cache.num_heads, cache.head_size)}, not {tuple(key.shape[1:])}")
    return _append("cb_append_paged_kv4", rotary_emb, positions, key, value, query, slot_mapping,
                   cache.num_blocks * cache.block_size, cache.block_size, cache.num_blocks, cache._pages(), stream)


def gather_paged_kv4(
    cache: PagedKV4,
    slot_mapping: torch.Tensor,
    dtype: torch.dtype = torch.bfloat16,
    out: torch.Tensor | None = None,
    stream: torch.cuda.Stream | None = None,
) -> torch.Tensor:
    """The values of 4-bit rows as ``[2, tokens, heads, head_size]`` of ``dtype``.

    A negative slot (padding) reads as zeros; so does, on the device, one outside the cache
    (IndexError for host slots).
    """
    _native.require_cuda(cache.codes)
    tokens = int(slot_mapping.numel())
    shape = (2, tokens, cache.num_heads, cache.head_size)
    code = _native.dtype_code(dtype)
    if out is not None:
        if tuple(out.shape) != shape:
            raise ValueError(f"gather output has shape {tuple(out.shape)}, expected {shape}")
        if out.dtype != dtype or out.device != cache.device:
            raise ValueError("gather output must match the dtype and the cache's device")
        if out.stride(3) != 1:
            raise ValueError("the values of a head must be contiguous in the output")
    with on_device(cache.device, stream):
        slots = _index("slot_mapping", slot_mapping, tokens, cache.device, None, cache.num_blocks * cache.block_size)
        result = out if out is not None else torch.empty(shape, dtype=dtype, device=cache.device)
        if tokens == 0:
            return result
        size = result.element_size()
        codes_k, codes_v, block_stride, slot_stride, head_stride, *scales = cache._pages()
        _native.call("cb_gather_paged_kv4", codes_k, codes_v, block_stride, slot_stride, head_stride, *scales,
                     cache.num_blocks, cache.block_size, cache.num_heads, cache.head_size, slots.data_ptr(), tokens,
                     result.data_ptr(), result.stride(0) * size, result.stride(1) * size, result.stride(2) * size, code,
                     current_handle())
        return result
