"""Attention: of a blend request's staging, of packed prompts, and of decode steps over 4-bit pages.

Blend attention on the tensor cores (cb_blend_attention): the side executor's
attention of the computed, possibly pruned, queries over the whole staging
context: Qwen3BlendExecutor._attention (cacheblend_vllm/ascend.py:798-846).  Queries sit at absolute positions and
attend every staging row at or before their position; grouped query heads
share their KV head.  ``prompt_attention`` and ``paged_attention4``: at the end of the file.
"""

from __future__ import annotations

import ctypes
import functools
import math

import torch

from . import _native
from .append import PagedKV4, _contiguous_empty, _raw_stream, on_device


# exact_rounding argument -> the C ABI's mode code
_MODES = {True: 1, "reference": 1, "flash": 2, False: 0, "fused": 0}


def attention_supported(query: torch.Tensor, key: torch.Tensor) -> bool:
    """Shapes cb_blend_attention takes: head size 128, bf16 / fp16, query heads
    a multiple of KV heads with the group count dividing 128."""
    if query.ndim != 3 or key.ndim != 3 or query.shape[2] != 128 or key.shape[2] != 128:
        return False
    if query.dtype not in (torch.bfloat16, torch.float16) or key.dtype != query.dtype:
        return False
    hq, hkv = query.shape[1], key.shape[1]
    return hkv > 0 and hq % hkv == 0 and 128 % (hq // hkv) == 0


def attention_workspace_bytes(num_queries: int, num_keys: int, num_q_heads: int, num_kv_heads: int,
                              head_size: int, dtype: torch.dtype) -> int:
    out = ctypes.c_int64(0)
    _native.call("cb_blend_attention_workspace_size", num_queries, num_keys, num_q_heads,
                 num_kv_heads, head_size, _native.dtype_code(dtype), ctypes.addressof(out))
    return int(out.value)


def blend_attention(
    query: torch.Tensor,
    key: torch.Tensor,
    value: torch.Tensor,
    query_positions: torch.Tensor,
    scale: float,
    workspace: torch.Tensor | None = None,
    device_error: torch.Tensor | None = None,
    stream: torch.cuda.Stream | None = None,
    exact_rounding: bool | str = True,
) -> torch.Tensor:
    """out [Nq, Hq, D] for query [Nq, Hq, D] at ``query_positions`` (each in [0, Nk)),
    key / value [Nk, Hkv, D] (rows = positions).

    ``exact_rounding``:

    * True / ``"reference"`` -- the einsum path's roundings in its order (element-type
      logits, element-type logit * scale, the normalized probabilities rounded to the
      element type before P V): a row log2-sum-exp launch, then the products.
    * ``"flash"`` -- the same logit roundings in one launch with the unnormalized
      probabilities rounded and the row sum divided at the end (within one element-type
      ulp per probability of the reference).
    * False / ``"fused"`` -- fp32 logits * scale like the reference's fused attention
      kernel (ascend.py:814-830) and flash attention, in one launch."""
    mode = _MODES.get(exact_rounding if isinstance(exact_rounding, str) else bool(exact_rounding))
    if mode is None:
        raise ValueError(f"exact_rounding must be True, False, 'reference', 'flash' or 'fused', "
                         f"not {exact_rounding!r}")
    _native.require_cuda(query, key, value)
    if query.ndim != 3 or key.ndim != 3 or value.shape != key.shape:
        raise ValueError("query must be [tokens, q_heads, head]; key and value [keys, kv_heads, head]")
    if not (query.dtype == key.dtype == value.dtype):
        raise ValueError("query, key and value must share a dtype")
    for name, t in (("query", query), ("key", key), ("value", value)):
        if t.stride(2) != 1 or t.stride(1) != t.shape[2]:
            raise ValueError(f"{name} heads must be contiguous within a row")
    num_queries, num_q_heads, head_size = query.shape
    num_keys, num_kv_heads, _ = key.shape
    positions = query_positions.to(device=query.device, dtype=torch.long).contiguous()
    if positions.numel() != num_queries:
        raise ValueError("one position per query row is required")
    out = torch.empty_like(query, memory_format=torch.contiguous_format)
    if num_queries == 0:
        return out
    need = attention_workspace_bytes(num_queries, num_keys, num_q_heads, num_kv_heads, head_size,
                                     query.dtype)
    if workspace is None or workspace.numel() < need:
        workspace = torch.empty(need, dtype=torch.uint8, device=query.device)
    esize = query.element_size()
    _native.call(
        "cb_blend_attention", query.data_ptr(), query.stride(0) * esize, key.data_ptr(),
        key.stride(0) * esize, value.data_ptr(), value.stride(0) * esize, num_keys, num_q_heads,
        num_kv_heads, head_size, _native.dtype_code(query.dtype), positions.data_ptr(), num_queries,
        float(scale), mode, out.data_ptr(), out.stride(0) * esize,
        workspace.data_ptr(), workspace.numel(),
        0 if device_error is None else device_error.data_ptr(), _native.stream_handle(stream),
    )
    return out


_HALVES = (torch.bfloat16, torch.float16)
_MOST = torch.finfo(torch.float32).max * math.log(2)  # a scale goes to fp32, and there to powers of two


def _int32(name: str, tensor: torch.Tensor, device: int, ndim: int) -> None:
    if tensor.dtype is not torch.int32 or tensor.get_device() != device or tensor.ndim != ndim:
        raise ValueError(f"{name} must be a {ndim}-dimensional int32 tensor on the query's device")
    if not tensor.is_contiguous() and tensor.stride(-1) != 1 and tensor.shape[-1] > 1:
        raise ValueError(f"{name} must be contiguous")


def _attention_out(query: torch.Tensor, out: torch.Tensor | None) -> torch.Tensor:
    if out is None:
        return _contiguous_empty(query)
    if out.shape != query.shape or out.dtype != query.dtype or out.device != query.device:
        raise ValueError("out must match the query's shape, dtype and device")
    if out.stride(2) != 1:
        raise ValueError("out heads must be contiguous")
    return out


def _scratch(workspace: torch.Tensor | None, need, device: torch.device) -> torch.Tensor:
    """The caller's workspace, or one of ``need()`` bytes."""
    if workspace is None:
        return torch.empty(need(), dtype=torch.uint8, device=device)
    if workspace.dtype != torch.uint8 or workspace.device != device or not workspace.is_contiguous():
        raise ValueError("workspace must be contiguous uint8 on the query's device")
    return workspace


def paged_attention4_workspace_bytes(num_tokens: int, num_seqs: int, num_q_heads: int, num_kv_heads: int,
                                     head_size: int) -> int:
    size = ctypes.c_int64(0)
    _native.call("cb_paged_attention4_workspace_size", num_tokens, num_seqs, num_q_heads, num_kv_heads, head_size,
                 ctypes.addressof(size))
    return int(size.value)


_decode_bytes = functools.lru_cache(paged_attention4_workspace_bytes)  # a size depends on sizes alone


def paged_attention4(
    query: torch.Tensor,
    cache: PagedKV4,
    block_table: torch.Tensor,
    seq_lens: torch.Tensor,
    scale: float,
    query_start: torch.Tensor | None = None,
    out: torch.Tensor | None = None,
    workspace: torch.Tensor | None = None,
    stream: torch.cuda.Stream | None = None,
) -> torch.Tensor:
    """Causal attention of each sequence's newest tokens over its 4-bit pages: ``[tokens, q_heads, head]``.

    ``query``: ``[tokens, q_heads, head_size]`` bf16 or fp16; query head h attends KV head
    ``h // (q_heads // kv_heads)``.  ``block_table``: int32 ``[seqs, pages]``, the pages of each
    sequence in order; ``seq_lens``: int32 ``[seqs]``, its keys, those of the query tokens
    included (append them first).  One token per sequence, or ``query_start``: int32
    ``[seqs + 1]``, where each sequence's rows begin; token j of n sees the keys at or before
    ``seq_lens - n + j``.

    A row that sees no key (an empty sequence) is zeros; rows behind the last sequence are left
    as ``out`` held them.  Pages outside the cache and keys past the table's width are left out;
    a cache of no pages is refused.  Logits are fp32: a row whose logits it does not hold or tell
    apart (beyond 2^30 or so) need not come out finite.  ``scale`` must be finite.
    ``workspace``: ``paged_attention4_workspace_bytes`` of uint8, for callers that keep one
    (two calls that may overlap need two); otherwise allocated per call.
    """
    if query.ndim != 3:
        raise ValueError("query must be [tokens, q_heads, head_size]")
    dtype, device = query.dtype, query.get_device()
    if dtype not in _HALVES:
        raise NotImplementedError(f"queries must be bfloat16 or float16, not {dtype}")
    tokens, heads, head_size = query.shape
    _, num_blocks, kv_heads, rows, half = cache.codes.shape
    if head_size != 2 * half or heads == 0 or heads % kv_heads:
        raise ValueError(f"query {tuple(query.shape)} does not fit {kv_heads} KV heads of {2 * half}")
    token, head, value = query.stride()
    if value != 1:
        raise ValueError("query heads must be contiguous")
    if cache.codes.get_device() != device:
        raise ValueError("query and cache must live on one device")
    _int32("block_table", block_table, device, 2)
    _int32("seq_lens", seq_lens, device, 1)
    seqs, width = block_table.shape
    if seq_lens.numel() != seqs:
        raise ValueError("block_table must hold one row per sequence")
    start = 0
    if query_start is not None:
        _int32("query_start", query_start, device, 1)
        if query_start.numel() != seqs + 1:
            raise ValueError("query_start must hold one entry per sequence and one more")
        start = query_start.data_ptr()
    elif tokens != seqs:
        raise ValueError(f"{tokens} query tokens for {seqs} sequences need query_start")
    if not -_MOST < scale < _MOST:
        raise ValueError(f"the scale must be finite, not {scale}")
    if device < 0:
        _native.require_cuda(query)
    with on_device(device, stream):
        result = _attention_out(query, out)
        if tokens == 0 or seqs == 0:
            return result
        workspace = _scratch(
            workspace, lambda: _decode_bytes(tokens, seqs, heads, kv_heads, head_size), query.device)
        out_token, out_head, _ = result.stride()
        _native.call_packed(
            "cb_paged_attention4", device, query.data_ptr(), 2 * token, 2 * head, tokens, heads,
            _native.DTYPE_CODES[dtype], start, *cache._pages(), num_blocks, rows, kv_heads, head_size, block_table.data_ptr(), block_table.stride(0), width,
            seq_lens.data_ptr(), seqs, float(scale), result.data_ptr(), 2 * out_token, 2 * out_head, workspace.data_ptr(),
            workspace.numel(), _raw_stream(device))
        return result


def prompt_attention_workspace_bytes(num_queries: int, num_seqs: int, num_q_heads: int, num_kv_heads: int,
                                     head_size: int) -> int:
    size = ctypes.c_int64(0)
    _native.call("cb_prompt_attention_workspace_size", num_queries, num_seqs, num_q_heads, num_kv_heads, head_size,
                 ctypes.addressof(size))
    return int(size.value)


_prompt_bytes = functools.lru_cache(prompt_attention_workspace_bytes)


def prompt_attention(
    query: torch.Tensor,
    key: torch.Tensor,
    value: torch.Tensor,
    query_start: torch.Tensor,
    scale: float,
    key_start: torch.Tensor | None = None,
    out: torch.Tensor | None = None,
    workspace: torch.Tensor | None = None,
    device_error: torch.Tensor | None = None,
    stream: torch.cuda.Stream | None = None,
) -> torch.Tensor:
    """Causal attention of a packed batch of prompts: ``[tokens, q_heads, head_size]``.

    ``query``: ``[tokens, q_heads, head_size]``, ``key`` and ``value``: ``[keys, kv_heads, head_size]``,
    bf16 or fp16, heads of 64 or 128 values, rows 16-byte aligned (slices of one projection's
    output will do); query head h attends KV head ``h // (q_heads // kv_heads)``.
    ``query_start``: int32 ``[seqs + 1]`` on the device, where each sequence's rows begin,
    ascending; ``key_start`` the same for its keys, if it has more of them than queries (a
    cached prefix): its n queries are then the last n of its k keys, and query j sees the keys
    at or before ``k - n + j``.

    A query that sees no key gives zeros; rows of no sequence are left as ``out`` held them, and
    nothing that a masked place or another sequence holds reaches an output.  A row whose seen
    logits are all -inf is NaN, as of any softmax of them.  Probabilities are rounded to the
    element type before they meet the values.  ``scale`` must be positive and finite.
    ``device_error``: int32, set to a code if a wait inside the kernel ran out of its 2 seconds
    (rows are then missing); without it that goes unreported.
    ``workspace``: ``prompt_attention_workspace_bytes`` of uint8, for callers that keep
    one (two calls that may overlap need two); otherwise allocated per call.
    """
    shape, key_shape = query.shape, key.shape
    if len(shape) != 3 or len(key_shape) != 3 or value.shape != key_shape:
        raise ValueError("query must be [tokens, q_heads, head_size]; key and value [keys, kv_heads, head_size]")
    dtype, device = query.dtype, query.get_device()
    if dtype not in _HALVES:
        raise NotImplementedError(f"prompt attention needs bfloat16 or float16, not {dtype}")
    if key.dtype is not dtype or value.dtype is not dtype:
        raise ValueError("query, key and value must share a dtype")
    tokens, heads, head_size = shape
    keys, kv_heads, key_size = key_shape
    if key_size != head_size or kv_heads == 0 or heads == 0 or heads % kv_heads:
        raise ValueError(f"query {tuple(shape)} does not fit keys {tuple(key_shape)}")
    if key.get_device() != device or value.get_device() != device:
        raise ValueError("query, key and value must live on one device")
    strides = query.stride(), key.stride(), value.stride()
    if not (strides[0][2] == strides[1][2] == strides[2][2] == 1):
        raise ValueError("the heads of query, key and value must be contiguous")
    _int32("query_start", query_start, device, 1)
    seqs = query_start.numel() - 1
    if seqs < 0:
        raise ValueError("query_start must hold one entry per sequence and one more")
    if key_start is None:
        if keys != tokens:
            raise ValueError(f"{keys} keys for {tokens} queries need key_start")
        key_start = query_start
    else:
        _int32("key_start", key_start, device, 1)
        if key_start.numel() != seqs + 1:
            raise ValueError("key_start must hold as many entries as query_start")
    if not 0 < scale < _MOST:
        raise ValueError(f"the scale must be positive and finite, not {scale}")
    if device_error is not None and (device_error.dtype != torch.int32 or device_error.get_device() != device):
        raise ValueError("device_error must be int32 on the query's device")
    if device < 0:
        _native.require_cuda(query)
    with on_device(device, stream):
        result = _attention_out(query, out)
        if tokens == 0 or seqs == 0:
            return result
        workspace = _scratch(
            workspace, lambda: _prompt_bytes(tokens, seqs, heads, kv_heads, head_size), query.device)
        strides = (*strides, result.stride())
        if tokens == 1 or keys == 1 or heads == 1 or kv_heads == 1:  # dimensions of one may carry any stride
            strides = [(t if n > 1 else h * (r if h > 1 else head_size), r if h > 1 else head_size)
                       for (n, h, _), (t, r, _) in zip((shape, key_shape, key_shape, shape), strides)]
        (q_token, q_head, *_), (k_token, k_head, *_), (v_token, v_head, *_), (out_token, out_head, *_) = strides
        _native.call_packed(
            "cb_prompt_attention", device, query.data_ptr(), 2 * q_token, 2 * q_head, key.data_ptr(), 2 * k_token,
            2 * k_head, value.data_ptr(), 2 * v_token, 2 * v_head, tokens, keys, heads, kv_heads, head_size,
            _native.DTYPE_CODES[dtype], query_start.data_ptr(), key_start.data_ptr(), seqs, float(scale),
            result.data_ptr(), 2 * out_token, 2 * out_head, workspace.data_ptr(), workspace.numel(),
            0 if device_error is None else device_error.data_ptr(), _raw_stream(device))
        return result
