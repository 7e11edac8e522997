from radeon_kernels.ops.paged_cache_8bit.api import paged_attention_decode_8bit, paged_cache_append_8bit

__all__ = ["paged_attention_decode_8bit", "paged_cache_append_8bit"]
