"""Sizes beyond what the cache's attention takes are refused before any GPU call."""
import pytest
import torch

from pasa_amd import _lib
from pasa_amd.kv_cache import MAX_KEYS, KVCache8, cached_attention

from test_kv_cache_host import attn, kv8, status


def test_too_many_keys():
    cache = KVCache8.empty(3, 2, 64, page_size=128, device="cpu")
    q, lens = torch.zeros(1, 2, 64, dtype=torch.bfloat16), torch.zeros(1, dtype=torch.int32)
    wide = torch.zeros(1, MAX_KEYS // 128 + 1, dtype=torch.int32)  # 64 MB
    with pytest.raises(ValueError, match="at most"):
        cached_attention(q, cache, wide, lens)
    with pytest.raises(ValueError, match="no CPU path"):
        cached_attention(q, cache, wide, lens, max_kv_len=MAX_KEYS)


def test_c_too_many_keys():
    lib = _lib.load()
    status(lib, lib.pasa_kv8_attn(kv8(), attn(max_kv=MAX_KEYS + 1), 0x1000, 1 << 30, None), -6, "max_kv")
    status(lib, lib.pasa_kv8_attn(kv8(), attn(max_kv=MAX_KEYS, q=None), 0x1000, 1 << 30, None), -1, "NULL")
    assert lib.pasa_kv8_attn_workspace_bytes(2, 2, 2, 2, 128, MAX_KEYS + 1) == 0
