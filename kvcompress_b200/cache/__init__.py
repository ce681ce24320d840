"""Compressed KV cache containers."""

from kvcompress_b200.cache.compress import CompressedKVCache, LayerEntry, normalize_kv, payload_to_meta
from kvcompress_b200.cache.manager import CacheManager
from kvcompress_b200.cache.metadata import CompressionMetadata, LayerCompression
from kvcompress_b200.cache.paged import CacheStep, PagedKVCache

__all__ = ["CacheManager", "CacheStep", "CompressedKVCache", "CompressionMetadata", "LayerCompression", "LayerEntry",
           "PagedKVCache", "normalize_kv", "payload_to_meta"]
