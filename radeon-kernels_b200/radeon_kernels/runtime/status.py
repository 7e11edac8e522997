"""``rk.device_status()``: what the kernels of this process could not tell the host at launch.

Kernels that meet an index out of range in device memory skip it, and kernels whose bounded
wait runs out give up; both set a bit in a status word of their library on that device.
Every loaded library has a word of its own -- the built-in one and each kernel pack -- so
this reads them all.
"""

from __future__ import annotations

from typing import Any, Iterable

from radeon_kernels import _native


def _modules() -> Iterable[Any]:
    from radeon_kernels.ops._runtime import loaded_modules

    yield _native.extension()
    yield from loaded_modules()


def device_status() -> int:
    """Reads and clears the status of the current device, after synchronising its current stream.

    0: nothing to report; 1 (``RK_ERR_INVALID_ARGUMENT``): a kernel launched since the last
    call met an index out of range and skipped it; 4 (``RK_ERR_TIMEOUT``): a bounded wait
    ran out.  Not for use while a stream is being captured."""

    return max((int(module.device_status()) for module in _modules()), default=0)


__all__ = ["device_status"]
