"""MI355X-native drop-in for the `flash_attention_sm75` package.

Public surface of reference src/flash_attention_sm75/__init__.py:1-4, and what
this package adds to it.
"""
from .ops import (flash_attention, flash_attention_backward, flash_attention_forward,
                  flash_attention_forward_ex, flash_attention_forward_lse)
from .paged import (flash_attention_paged, flash_attention_paged_prefix, paged_attention_weights,
                    paged_cache_evict, paged_cache_read, paged_cache_write)

__version__ = "0.1.0"
__all__ = ["flash_attention_forward", "flash_attention_forward_ex", "flash_attention_forward_lse",
           "flash_attention", "flash_attention_backward",
           "flash_attention_paged", "flash_attention_paged_prefix", "paged_attention_weights",
           "paged_cache_evict", "paged_cache_read", "paged_cache_write"]
