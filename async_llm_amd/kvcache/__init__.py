from .mha_pool import MHAKVCache
from .page_allocator import PageAllocator
from .quantized_pool import QuantizedKVCache

__all__ = ["MHAKVCache", "PageAllocator", "QuantizedKVCache"]
