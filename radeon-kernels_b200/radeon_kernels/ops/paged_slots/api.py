"""Public slot maps: ``rk.paged_slots(block_tables, context_lengths, new_lengths, free_blocks,
*, num_tokens, block_size)``.

Where the new tokens of a step go in a paged K/V cache, computed on the GPU from the requests'
lengths: request ``b`` holds ``context_lengths[b]`` tokens and gets ``new_lengths[b]`` more (0:
none).  Its row of ``block_tables [batch, max_blocks]`` is extended in place by the blocks that
it now needs, taken from ``free_blocks`` in request order (no other entry is written), and a
new ``(slot_mapping, positions, lengths, blocks_used)`` is returned:

* ``slot_mapping [num_tokens]`` int64: ``block * block_size + offset`` of every new token, the
  requests' tokens one after the other, ``-1`` behind the last -- what
  ``rk.paged_cache_append_8bit`` takes;
* ``positions [num_tokens]``: the token's position in its request (0 behind the last) -- what
  ``rk.rotary_embedding`` takes;
* ``lengths [batch]``: ``context_lengths + new_lengths``, at most ``max_blocks * block_size`` --
  what the decode attention takes after the append;
* ``blocks_used [1]``: entries of ``free_blocks`` that the step needs; more than
  ``len(free_blocks)`` means that the list was too short.

Index tensors share int32 or int64.  ``num_tokens`` is the size of the step's token buffer, at
least ``new_lengths.sum()``; the host never reads a length back, so a step can be captured in
a CUDA graph.  Tokens without a block get slot -1, and that, a negative length (taken as 0) or
a buffer that is too short makes the next device status check report an invalid argument.

The reference has no such operator; operator ``"paged_slots"`` (semantic version 1.0).
"""

from __future__ import annotations

from typing import Any

from radeon_kernels.ops._common import device_index_of, torch_runtime
from radeon_kernels.ops._frontend import Args, dispatch, quick_call, remember_call
from radeon_kernels.ops._runtime import OperatorRuntime, default_operator_runtime
from radeon_kernels.providers import cuda_builtin

MAXIMUM_TOKENS = 2**31 - 1


def _execute(block_tables: Any, context_lengths: Any, new_lengths: Any, free_blocks: Any, num_tokens: int,
             block_size: int, *, torch_module: Any, runtime: OperatorRuntime, key_of_call: Any = None) -> Any:
    args = Args("paged_slots", torch_module, block_tables=block_tables, context_lengths=context_lengths,
                new_lengths=new_lengths, free_blocks=free_blocks)
    args.indices(block_tables=2, context_lengths=1, new_lengths=1, free_blocks=1)
    args.alike("block_tables", "context_lengths", "new_lengths", "free_blocks")
    for name, value in (("num_tokens", num_tokens), ("block_size", block_size)):
        args.expect(not isinstance(value, bool) and isinstance(value, int), f"{name} must be an int", TypeError)
    batch, max_blocks = args.dims("block_tables")
    args.expect(batch > 0 and max_blocks > 0, "block_tables dimensions must be positive")
    args.expect(args.dims("context_lengths") == (batch,) and args.dims("new_lengths") == (batch,),
                "lengths must contain one length per row of block_tables")
    args.expect(block_size > 0, "block_size must be positive")
    args.expect(max_blocks * block_size < 2**31, "max_blocks * block_size must be below 2**31")
    args.expect(0 <= num_tokens <= MAXIMUM_TOKENS, "num_tokens must be in [0, 2**31 - 1]")
    args.expect(all(t.is_contiguous() for t in args.values.values()), "inputs must be contiguous")
    device_index = device_index_of(torch_module, block_tables)
    signature = {"index_dtype": args.index_dtype("block_tables"), "block_size": block_size, "contiguous": True}
    result = dispatch(
        args, runtime, semantic_version="1.0", signature=signature, device_index=device_index,
        native_arguments=(block_tables, context_lengths, new_lengths, free_blocks, num_tokens, block_size),
        fallback=cuda_builtin.paged_slots, fallback_selected=cuda_builtin.SELECTED_PAGED_SLOTS,
    )
    remember_call(runtime, key_of_call, "paged_slots", device_index, signature)
    return tuple(result)


def paged_slots(block_tables: Any, context_lengths: Any, new_lengths: Any, free_blocks: Any, *, num_tokens: int,
                block_size: int) -> tuple[Any, Any, Any, Any]:
    """Extend the block tables by a step's new blocks and map its tokens to cache slots."""

    runtime, call = default_operator_runtime(), None
    if type(num_tokens) is int and type(block_size) is int:
        try:
            call = ("paged_slots", block_tables.dtype, block_tables.device, block_size)
            result = quick_call(runtime, call, (block_tables, context_lengths, new_lengths, free_blocks, num_tokens,
                                                block_size))
            if result is not None:
                return tuple(result)
        except AttributeError:
            call = None  # no tensor: the checks say so
    return _execute(block_tables, context_lengths, new_lengths, free_blocks, num_tokens, block_size,
                    torch_module=torch_runtime("paged_slots"), runtime=runtime, key_of_call=call)
