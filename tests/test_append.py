"""Refusals of the paged append and of the 4-bit pages, without a GPU."""

from __future__ import annotations

import ctypes
from types import SimpleNamespace

import pytest
import torch

from cacheblend_b200 import PagedKV4, _native, append_paged_kv, append_paged_kv4, gather_paged_kv4

ROPE = SimpleNamespace(head_size=64, rotary_dim=64, is_neox_style=True, cos_sin_cache=torch.zeros(8, 64))
K = torch.zeros(3, 2, 64, dtype=torch.bfloat16)
PAGES = torch.zeros(2, 4, 16, 2, 64, dtype=torch.bfloat16)
SLOTS = torch.arange(3)


@pytest.mark.parametrize("key,value,query", [
    (K[0], K[0], None),                      # not three dimensions
    (K, K[:2], None),                        # another token count
    (K, K[:, :1], None),                     # another head count
    (K, K.float(), None),                    # another type
    (K.transpose(1, 2).contiguous().transpose(1, 2), K, None),  # values of a head apart
    (K, K, K[..., :32]),
    (K, K, K.float()),
])
def test_append_refuses_rows(key, value, query):
    with pytest.raises(ValueError):
        append_paged_kv(ROPE, SLOTS, key, value, PAGES, SLOTS, 16, query=query)
    with pytest.raises(ValueError):
        append_paged_kv4(ROPE, SLOTS, key, value, PagedKV4.allocate(2, 16, 2, 64, "cpu"), SLOTS, query=query)


def test_append_needs_cuda_and_known_layouts():
    with pytest.raises(RuntimeError, match="CUDA tensors only"):
        append_paged_kv(ROPE, SLOTS, K, K, PAGES, SLOTS, 16)
    with pytest.raises(RuntimeError, match="CUDA tensors only"):
        append_paged_kv4(ROPE, SLOTS, K, K, PagedKV4.allocate(2, 16, 2, 64, "cpu"), SLOTS)
    with pytest.raises(RuntimeError, match="CUDA tensors only"):
        gather_paged_kv4(PagedKV4.allocate(2, 16, 2, 64, "cpu"), SLOTS)
    with pytest.raises(ValueError):
        append_paged_kv(ROPE, SLOTS, K, K, torch.zeros(3, 3, 16, 2, 64, dtype=torch.bfloat16), SLOTS, 16)
    with pytest.raises(ValueError, match="block_size"):
        append_paged_kv(ROPE, SLOTS, K, K, PAGES, SLOTS, 17)


@pytest.mark.parametrize("codes,scales,error", [
    ((2, 4, 2, 16, 32), (2, 4, 2, 16, 2, 2), ValueError),
    ((2, 4, 2, 16, 48), (2, 4, 2, 16, 1, 2), NotImplementedError),
    ((3, 4, 2, 16, 32), (3, 4, 2, 16, 1, 2), ValueError),
    ((2, 4, 0, 16, 32), (2, 4, 0, 16, 1, 2), ValueError),
])
def test_pages_refuse_shapes(codes, scales, error):
    with pytest.raises(error):
        PagedKV4(torch.zeros(codes, dtype=torch.uint8), torch.zeros(scales, dtype=torch.float16))


def test_pages_refuse_types_and_strides():
    codes, scales = torch.zeros(2, 4, 2, 16, 32, dtype=torch.uint8), torch.zeros(2, 4, 2, 16, 1, 2, dtype=torch.float16)
    with pytest.raises(ValueError):
        PagedKV4(codes.int(), scales)
    with pytest.raises(ValueError):
        PagedKV4(codes, scales.float())
    with pytest.raises(ValueError, match="contiguous"):
        PagedKV4(torch.zeros(2, 4, 2, 16, 64, dtype=torch.uint8)[..., ::2], scales)
    cache = PagedKV4(codes, scales)
    assert (cache.num_blocks, cache.num_heads, cache.block_size, cache.head_size) == (4, 2, 16, 64)


def _c_append(**changed):
    """cb_append_paged_kv with made-up aligned addresses: refused before any device work."""
    a = dict(key=256, kts=256, khs=128, value=256, vts=256, vhs=128, q=0, qts=0, qhs=0, qo=0, qots=0, qohs=0, tokens=3, heads=0,
             kv_heads=2, head=64, dtype=0, positions=256, table=256, table_dtype=2, most=8, rotary=64, neox=1, kc=256, vc=256,
             bs=4096, ss=256, hs=128, blocks=4, block=16, slots=256)
    a.update(changed)
    # no stream and no page pointer to ask the device of: argument checks only
    return _native.load_library().cb_append_paged_kv(*[None if v is None else v for v in a.values()], None)


@pytest.mark.parametrize("changed,status", [
    (dict(kc=None, tokens=-1), -1), (dict(kc=None, kv_heads=0), -1), (dict(kc=None, block=0), -1), (dict(kc=None, rotary=65), -1),
    (dict(kc=None, rotary=66), -1), (dict(kc=None, dtype=7), -2), (dict(kc=None, table_dtype=1), -2), (dict(kc=None), -1),
    (dict(kc=None, blocks=1 << 50), -1), (dict(kc=None, tokens=0), 0),
])
def test_c_entry_refuses(changed, status):
    assert _c_append(**changed) == status
    if status:
        assert _native.load_library().cb_last_error()


def test_c_entry_4_bit_refuses():
    lib = _native.load_library()
    base = [None, 0, 0, None, 0, 0, None, 0, 0, None, 0, 0, 0, 0, 2, 64, 0, None, None, 2, 0, 64, 1, None, None, 0, 0, 0,
            None, None, 0, 0, 0, 4, 16, None, None]
    assert lib.cb_append_paged_kv4(*base) == 0  # no tokens
    base[12] = 1
    assert lib.cb_append_paged_kv4(*base) == _native.CB_ERR_INVALID
    assert b"null" in lib.cb_last_error()
    assert lib.cb_gather_paged_kv4(*[None, None, 0, 0, 0, None, None, 0, 0, 0, 4, 16, 2, 64, None, 1, None, 0, 0, 0, 0, None]) == \
        _native.CB_ERR_INVALID
    assert isinstance(lib.cb_gather_paged_kv4, ctypes._CFuncPtr)


def test_import_without_cuda_bindings():
    """The package imports, and refuses CPU tensors as ever, on a torch that has no CUDA bindings."""
    import subprocess
    import sys
    from pathlib import Path

    code = """
import torch
for name in [n for n in dir(torch._C) if n.startswith("_cuda_")]:
    delattr(torch._C, name)
from cacheblend_b200 import CacheBlendConfig, append_paged_kv, paged_attention4
key, pages = torch.zeros(3, 2, 64), torch.zeros(2, 4, 16, 2, 64)
try:
    append_paged_kv(None, None, key, key, pages, torch.arange(3), 16)
except RuntimeError as error:
    print(error)
"""
    run = subprocess.run([sys.executable, "-c", code], capture_output=True, text=True,
                         cwd=Path(__file__).resolve().parents[1] / "pic-kvcache_b200")
    assert run.returncode == 0 and "CUDA tensors only" in run.stdout, run.stderr
