"""Streaming caches (reference cortex/cache): the paged LRU embedding cache, the
device event-page cache that streaming decode windows are assembled from, and the
paged K/V cache that attention reads in place."""

from cortex.cache.paged import KVBatch, PagedKVCache
from cortex.cache.streaming import EventWindowCache, PageMeta, StreamingKVCache

__all__ = ["EventWindowCache", "KVBatch", "PageMeta", "PagedKVCache", "StreamingKVCache"]
