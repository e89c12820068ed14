"""Pre-allocated compressed KV storage for the fused attention path
(counterpart of src/flashquant/cache/buffer_pool.py), and paged storage driven
from the GPU, packed or at 16 bits."""
from flashquant_amd.cache.buffer_pool import CompressedBuffer, CompressedKVLayer
from flashquant_amd.cache.paged import PagedKVLayer, PagedStep, PagedTQ4Layer, PageTable

__all__ = ["CompressedBuffer", "CompressedKVLayer", "PageTable", "PagedStep", "PagedKVLayer", "PagedTQ4Layer"]
