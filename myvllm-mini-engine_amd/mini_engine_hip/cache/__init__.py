"""Paged KV-cache storage and page ownership."""

from .kv_cache import KVCachePool, KVCachePoolFP4, KVCacheShape
from .page_pool import PagePool

__all__ = ["KVCachePool", "KVCachePoolFP4", "KVCacheShape", "PagePool"]
