"""PyTorch front-end: flash_hog.torch.attention.dot_product_attention, what stands before it
(flash_hog.torch.rotary), and the paged cache's operators (flash_hog.torch.paged)."""

from flash_hog.torch.attention import dot_product_attention
from flash_hog.torch.paged import (paged_attention, paged_block_attention, paged_block_select, paged_cache_compact,
                                   paged_cache_extend, paged_cache_read, paged_cache_write, paged_key_means)
from flash_hog.torch.rotary import qk_norm_rotary

__all__ = ["dot_product_attention", "paged_attention", "paged_block_attention", "paged_block_select",
           "paged_cache_compact", "paged_cache_extend", "paged_cache_read", "paged_cache_write", "paged_key_means",
           "qk_norm_rotary"]
