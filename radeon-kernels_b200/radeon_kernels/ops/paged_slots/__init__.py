from radeon_kernels.ops.paged_slots.api import paged_slots

__all__ = ["paged_slots"]
