"""Refusals of paged_attention4 and prompt_attention, without a GPU."""

from __future__ import annotations

import ctypes

import pytest
import torch

from cacheblend_b200 import PagedKV4, _native, paged_attention4, prompt_attention

CACHE = PagedKV4.allocate(4, 16, 2, 64, "cpu")
Q = torch.zeros(3, 4, 64, dtype=torch.bfloat16)
TABLE = torch.zeros(3, 2, dtype=torch.int32)
LENS = torch.ones(3, dtype=torch.int32)
START = torch.tensor([0, 1, 3], dtype=torch.int32)
K = torch.zeros(3, 2, 64, dtype=torch.bfloat16)


@pytest.mark.parametrize("query,table,lens,start,error", [
    (Q[0], TABLE, LENS, None, ValueError),
    (Q.float(), TABLE, LENS, None, NotImplementedError),
    (Q[..., :32], TABLE, LENS, None, ValueError),          # another head size
    (Q[:, :3], TABLE, LENS, None, ValueError),             # 3 heads on 2
    (Q.transpose(1, 2).contiguous().transpose(1, 2), TABLE, LENS, None, ValueError),
    (Q, TABLE.long(), LENS, None, ValueError),
    (Q, TABLE[0], LENS, None, ValueError),
    (Q, TABLE[:2], LENS, None, ValueError),
    (Q, TABLE, LENS.long(), None, ValueError),
    (Q[:2], TABLE, LENS, None, ValueError),                # no query_start
    (Q, TABLE, LENS, START, ValueError),                   # one entry short
    (Q, TABLE.repeat(1, 2)[:, ::2], LENS, None, ValueError),
    (Q, TABLE, LENS, None, RuntimeError),                  # all fits: no CPU fallback
])
def test_paged_attention4_refuses(query, table, lens, start, error):
    with pytest.raises(error):
        paged_attention4(query, CACHE, table, lens, 0.1, query_start=start)


@pytest.mark.parametrize("query,key,value,start,scale,key_start,error", [
    (Q[0], K, K, START, 0.1, None, ValueError),
    (Q, K, K[:2], START, 0.1, None, ValueError),
    (Q.float(), K, K, START, 0.1, None, NotImplementedError),
    (Q, K.half(), K.half(), START, 0.1, None, ValueError),
    (Q[:, :3], K, K, START, 0.1, None, ValueError),
    (Q, K[..., :32], K[..., :32], START, 0.1, None, ValueError),
    (Q, K.transpose(1, 2).contiguous().transpose(1, 2), K, START, 0.1, None, ValueError),
    (Q, K, K, START.long(), 0.1, None, ValueError),
    (Q, K, K, START[:0], 0.1, None, ValueError),
    (Q[:2], K, K, START, 0.1, None, ValueError),           # more keys than queries: key_start
    (Q, K, K, START, 0.1, START[:2], ValueError),
    (Q, K, K, START, 0.0, None, ValueError),
    (Q, K, K, START, float("nan"), None, ValueError),
    (Q, K, K, START, 0.1, None, RuntimeError),             # all fits: no CPU fallback
])
def test_prompt_attention_refuses(query, key, value, start, scale, key_start, error):
    with pytest.raises(error):
        prompt_attention(query, key, value, start, scale, key_start=key_start)


def test_workspace_sizes_without_a_gpu():
    lib = _native.load_library()
    size = ctypes.c_int64(-1)
    assert lib.cb_paged_attention4_workspace_size(0, 0, 8, 2, 128, ctypes.byref(size)) == 0 and size.value == 0
    assert lib.cb_paged_attention4_workspace_size(5, 3, 8, 2, 128, ctypes.byref(size)) == 0 and size.value > 0
    assert lib.cb_paged_attention4_workspace_size(5, 3, 8, 3, 128, ctypes.byref(size)) == _native.CB_ERR_INVALID
    assert lib.cb_paged_attention4_workspace_size(5, 3, 8, 2, 96, ctypes.byref(size)) == _native.CB_ERR_UNSUPPORTED
    assert lib.cb_paged_attention4_workspace_size(5, 0, 8, 2, 128, ctypes.byref(size)) == _native.CB_ERR_INVALID
    assert lib.cb_paged_attention4_workspace_size(5, 3, 8, 2, 128, None) == _native.CB_ERR_INVALID
    # one 16-byte record per pair of query tiles: 64 queries of 4 heads to a KV head
    assert lib.cb_prompt_attention_workspace_size(1000, 3, 32, 8, 128, ctypes.byref(size)) == 0
    assert size.value == 256 + (1000 // 64 + 3) * 16
    assert lib.cb_prompt_attention_workspace_size(1000, 3, 129, 1, 128, ctypes.byref(size)) == _native.CB_ERR_UNSUPPORTED
    assert lib.cb_prompt_attention_workspace_size(1000, 3, 8, 2, 256, ctypes.byref(size)) == _native.CB_ERR_UNSUPPORTED
    assert lib.cb_prompt_attention_workspace_size(-1, 3, 8, 2, 128, ctypes.byref(size)) == _native.CB_ERR_INVALID


def test_c_entries_refuse_before_any_device_work():
    lib = _native.load_library()
    # no stream and no output address: argument checks only
    def decode(tokens=2, heads=8, dtype=0, head=128, seqs=2, kv=2, blocks=4, block=16):
        return lib.cb_paged_attention4(None, 0, 0, tokens, heads, dtype, None, None, None, 0, 0, 0, None, None, 0, 0, 0, blocks,
                                       block, kv, head, None, 0, 0, None, seqs, 0.1, None, 0, 0, None, 0, None)
    assert decode(tokens=0, seqs=0) == 0
    assert decode() == _native.CB_ERR_INVALID and b"null" in lib.cb_last_error()
    assert decode(dtype=2) == _native.CB_ERR_UNSUPPORTED
    assert decode(head=96) == _native.CB_ERR_UNSUPPORTED
    assert decode(kv=3) == _native.CB_ERR_INVALID
    assert decode(tokens=3) == _native.CB_ERR_INVALID and b"query_start" in lib.cb_last_error()
    assert decode(block=0) == _native.CB_ERR_INVALID

    def prompt(queries=2, keys=2, heads=8, kv=2, head=128, dtype=0, seqs=1, scale=0.1):
        return lib.cb_prompt_attention(None, 0, 0, None, 0, 0, None, 0, 0, queries, keys, heads, kv, head, dtype, None, None,
                                       seqs, scale, None, 0, 0, None, 0, None, None)
    assert prompt(queries=0) == 0
    assert prompt() == _native.CB_ERR_INVALID
    assert prompt(scale=0.0) == _native.CB_ERR_INVALID
    assert prompt(dtype=2) == _native.CB_ERR_UNSUPPORTED
    assert prompt(head=32) == _native.CB_ERR_UNSUPPORTED
    assert prompt(keys=-1) == _native.CB_ERR_INVALID


def test_packed_calls_refuse_alike():
    """cb_call_packed: the entries' own refusals, and those of words that fit no entry."""
    lib = _native.load_library()
    assert [code for code, _, _ in _native.PACKED.values()] == list(range(5))
    for name, (code, pack, count) in _native.PACKED.items():
        words = pack(*[0] * count)
        assert len(words) == 8 * count
        direct = getattr(lib, name)(*[0] * count)
        message = lib.cb_last_error()
        packed = lib.cb_call_packed(code, 0, words, count)
        if packed != _native.CB_ERR_CUDA:  # (no device here: it cannot be made current)
            assert packed == direct and lib.cb_last_error() == message
        assert lib.cb_call_packed(code, 0, words, count - 1) == _native.CB_ERR_INVALID
        assert b"words" in lib.cb_last_error()
        assert lib.cb_call_packed(code, -1, words, count) == _native.CB_ERR_INVALID
        assert lib.cb_call_packed(code, 0, None, count) == _native.CB_ERR_INVALID
    assert lib.cb_call_packed(5, 0, b"\0" * 64, 8) == _native.CB_ERR_INVALID
    code, pack, count = _native.PACKED["cb_prompt_attention"]
    values = [0] * count
    values[14] = 1 << 32  # the element type's code is an int
    assert lib.cb_call_packed(code, 0, pack(*values), count) == _native.CB_ERR_INVALID
    assert b"fit" in lib.cb_last_error()


@pytest.mark.parametrize("scale", [float("nan"), float("inf"), -float("inf"), 1e39])
def test_scales_that_are_not_finite(scale):
    """A scale that fp32 does not hold is refused, not taken for another."""
    with pytest.raises(ValueError, match="scale"):
        paged_attention4(Q, CACHE, TABLE, LENS, scale)
    with pytest.raises(ValueError, match="scale"):
        prompt_attention(Q, K, K, START, scale)
    lib = _native.load_library()
    assert lib.cb_paged_attention4(None, 0, 0, 2, 8, 0, None, None, None, 0, 0, 0, None, None, 0, 0, 0, 4, 16, 2, 128, None, 0, 0,
                                   None, 2, scale, None, 0, 0, None, 0, None) == _native.CB_ERR_INVALID
    assert b"scale" in lib.cb_last_error()
    assert lib.cb_prompt_attention(None, 0, 0, None, 0, 0, None, 0, 0, 2, 2, 8, 2, 128, 0, None, None, 1, scale, None, 0, 0, None,
                                   0, None, None) == _native.CB_ERR_INVALID
    assert b"scale" in lib.cb_last_error()
