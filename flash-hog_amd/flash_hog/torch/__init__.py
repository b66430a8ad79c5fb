"""PyTorch front-end: flash_hog.torch.attention.dot_product_attention, and the paged cache's
operators (flash_hog.torch.paged)."""

from flash_hog.torch.attention import dot_product_attention
from flash_hog.torch.paged import paged_attention, paged_cache_read, paged_cache_write

__all__ = ["dot_product_attention", "paged_attention", "paged_cache_read", "paged_cache_write"]
