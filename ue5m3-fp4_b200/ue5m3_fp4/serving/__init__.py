"""Token-by-token use of a frozen packed model: products with packed weights, attention over a paged
key/value cache, sampling."""

from ue5m3_fp4.serving.cache import PagedKVCache
from ue5m3_fp4.serving.operators import packed_matvec, paged_attention, sample_tokens

__all__ = ["PagedKVCache", "packed_matvec", "paged_attention", "sample_tokens"]
