"""A K/V cache of 8-bit codes in pages (no reference counterpart: tensorax has no cache)."""
from __future__ import annotations

from ... import functional as F
from ...tensor import Tensor


class QuantizedKVCache:
    """Device memory for the keys and values of many sequences, in pages of ``page_size`` tokens.

    A row (one token of one K/V head) is ``head_dim`` one-byte codes that share a float32 scale: ``"e4m3"`` (scale a power of
    two, four significant bits an element) or ``"int8"`` (127 steps to the row's largest element).  Which page holds which
    tokens is the caller's: every call takes a page table [batch, pages of a sequence], as a list or array or, uploaded once,
    as ``cache.indices(table)``.  What no write has reached holds whatever the memory held.
    """

    def __init__(self, num_pages: int, num_kv_heads: int, head_dim: int, page_size: int = 64, dtype: str = "e4m3"):
        from ... import _C
        self._impl = _C.KvCacheImpl(num_pages, num_kv_heads, page_size, head_dim, dtype)

    num_pages = property(lambda self: self._impl.pages)
    num_kv_heads = property(lambda self: self._impl.kv_heads)
    page_size = property(lambda self: self._impl.page_size)
    head_dim = property(lambda self: self._impl.d)
    dtype = property(lambda self: self._impl.format)

    @staticmethod
    def indices(array, words: bool = False):
        """Page tables, lengths, positions, row lists (or, with ``words``, a tree's words) on the device, for use in many calls."""
        import numpy as np

        from ... import _C
        return _C.IndexImpl(array, np.uint64 if words else np.int32)

    def write(self, key: Tensor, value: Tensor, page_table, start=None, counts=None, rows=None, sync: bool = True) -> None:
        """``F.kv_cache_write`` into this cache."""
        F.kv_cache_write(self, key, value, page_table, start, counts, rows, sync)

    def read(self, page_table, tokens: int, start=None, counts=None, dtype: str = "float16", sync: bool = True):
        """``F.kv_cache_read`` of this cache: (K, V)."""
        return F.kv_cache_read(self, page_table, tokens, start, counts, dtype, sync)

    def attend(self, query: Tensor, page_table, kv_lens, q_lens=None, tree=None, window=None, sinks: int = 0,
               out_dtype: str = "float32", sync: bool = True) -> Tensor:
        """``F.kv_cache_attention`` over this cache."""
        return F.kv_cache_attention(query, self, page_table, kv_lens, q_lens, tree, window, sinks, out_dtype, sync)

    def __repr__(self) -> str:
        return (f"QuantizedKVCache(num_pages={self.num_pages}, num_kv_heads={self.num_kv_heads}, head_dim={self.head_dim}, "
                f"page_size={self.page_size}, dtype={self.dtype!r})")
