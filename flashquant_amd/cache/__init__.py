"""Pre-allocated compressed KV storage for the fused attention path
(counterpart of src/flashquant/cache/buffer_pool.py), and paged storage driven
from the GPU, packed, at 8 or at 16 bits."""
from flashquant_amd.cache.buffer_pool import CompressedBuffer, CompressedKVLayer
from flashquant_amd.cache.paged import PagedKV8Layer, PagedKVLayer, PagedStep, PagedTQ4Layer, PageTable

__all__ = ["CompressedBuffer", "CompressedKVLayer", "PageTable", "PagedStep", "PagedKVLayer", "PagedKV8Layer", "PagedTQ4Layer"]
