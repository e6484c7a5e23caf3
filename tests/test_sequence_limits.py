"""Sizes at the ends of what the calls on sequences take.  No GPU is asked before an argument is."""
import ctypes

import pytest

import fyusenet_amd as fa
from fyusenet_amd import capi


@pytest.mark.parametrize("pages,page_tokens", [(2048, 1024), (2049, 1024), (1 << 18, 8), ((1 << 18) + 1, 8), (1 << 20, 1024)])
def test_cache_refuses_sizes_beyond_64_bits(pages, page_tokens):
    """Pages of 2^53 or 2^46 bytes, so many of them that the product is 2^64 (zero in 64 bits) or a little more."""
    d = capi.CacheDesc(ctypes.sizeof(capi.CacheDesc), capi.STORAGE_F32, 65536, 65536, 65536, 256, page_tokens, pages, 1, 8)
    h = ctypes.c_void_p()
    with pytest.raises(fa.FynException) as e:
        capi.check(capi.lib().fyn_cache_create(0, ctypes.byref(d), ctypes.byref(h)))
    assert e.value.code == capi.ERR_INVALID and "addressed" in str(e.value) and not h.value


def test_attention_refuses_more_tokens_than_can_be_counted():
    """Positions are 32 bits, with room for the end of the last tile: beyond that nothing is computed, and not silently."""
    for batch, tokens in ((1, 2 ** 31 - 1), (1, 2 ** 31 - 100), (3, 715827882)):
        d = capi.AttentionDesc()
        d.struct_size, d.storage, d.batch, d.tokens, d.heads, d.kv_heads, d.head_dim = ctypes.sizeof(d), capi.STORAGE_F16, batch, tokens, 1, 1, 8
        with pytest.raises(fa.FynException) as e:
            capi.check(capi.lib().fyn_attention(ctypes.byref(d), None))
        assert e.value.code == capi.ERR_INVALID and "%d sequences of %d tokens" % (batch, tokens) in str(e.value)
