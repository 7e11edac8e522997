from radeon_kernels.ops.rotary.api import rotary_embedding, rotary_frequencies

__all__ = ["rotary_embedding", "rotary_frequencies"]
