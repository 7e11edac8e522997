"""Public operators of a paged K/V cache in 8 bits: ``rk.paged_cache_append_8bit(key, value,
key_cache, value_cache, key_scales, value_scales, slot_mapping)`` and
``rk.paged_attention_decode_8bit(query, key_cache, value_cache, key_scales, value_scales,
block_tables, context_lengths, scale=None)``.

``key_cache`` / ``value_cache`` ``[num_blocks, block_size, kv_heads, head_dim]`` (layout
``block_slot_head_dim``, as the 16-bit cache of ``rk.paged_attention_decode``) hold
``torch.float8_e4m3fn`` or ``torch.int8``; ``key_scales`` / ``value_scales`` ``[num_blocks,
kv_heads]`` float32 hold one scale per block and head, and a stored value stands for itself
times its scale.  head_dim 64, 128 or 256; inference only: inputs that require gradients or carry
forward-mode tangents are refused.

The append stores ``key`` / ``value`` ``[tokens, kv_heads, head_dim]`` (fp16/bf16, slices of a
projection are read in place) at ``slot_mapping [tokens]`` (int32/int64, ``block * block_size +
offset``, negative: skip), updates caches and scales in place and returns them.  A block's
scale is the least power of two that its rows fit in: it starts anew when the block's first
slot is written and otherwise only grows, re-rounding the rows that stay.  The tokens of one
block are adjacent in ``slot_mapping`` and their slots ascend, as ``rk.paged_slots`` lays them
out; a second run of tokens for a block, and slots past the cache, are skipped and reported by
the next device status check.

The attention has the semantics of ``rk.paged_attention_decode`` (same shapes, index types,
NaN for an empty sequence, skipped and reported block-table entries out of range) for any
number of query heads per KV head and any block size.

The reference has no 8-bit cache; operators ``"paged_cache_append_8bit"`` and
``"paged_attention_decode_8bit"`` (semantic version 1.0).  Sizes that change from step to step
are not part of their dispatch signatures.
"""

from __future__ import annotations

from typing import Any

from radeon_kernels.ops._common import torch_runtime
from radeon_kernels.ops._frontend import Args, dispatch, quick_call, remember_call
from radeon_kernels.ops._runtime import OperatorRuntime, default_operator_runtime
from radeon_kernels.providers import cuda_builtin

HEAD_DIMS = (64, 128, 256)
MAXIMUM_BLOCK_SIZE = 1024
MAXIMUM_TOKENS = 2**30 - 1


def _check_cache(args: Args) -> tuple[str, tuple[int, ...]]:
    """(cache dtype name, cache dimensions) of the caches and scales in ``args``, checked."""

    torch = args.torch
    names = {torch.float8_e4m3fn: "e4m3", torch.int8: "int8"}
    for name, rank in (("key_cache", 4), ("value_cache", 4), ("key_scales", 2), ("value_scales", 2)):
        tensor = args[name]
        args.expect(isinstance(tensor, torch.Tensor), f"{name} must be a PyTorch tensor", TypeError)
        args.expect(tensor.dim() == rank, f"{name} must be rank {rank}")
        args.expect(tensor.is_cuda, f"{name} must be on a visible CUDA GPU")
        if rank == 4:
            args.expect(tensor.dtype in names, f"{name} must use torch.float8_e4m3fn or torch.int8", TypeError)
        else:
            args.expect(tensor.dtype == torch.float32, f"{name} must use torch.float32", TypeError)
    args.alike("key_cache", "value_cache").alike("key_scales", "value_scales")
    args.expect(args["key_scales"].device == args["key_cache"].device, "scales must use the same device as the caches")
    dims = args.dims("key_cache")
    args.expect(args.dims("value_cache") == dims, "key_cache and value_cache must have the same shape")
    args.expect(min(dims) > 0, "cache dimensions must be positive")
    args.expect(args.dims("key_scales") == (dims[0], dims[2]) and args.dims("value_scales") == (dims[0], dims[2]),
                "scales must have shape [num_blocks, kv_heads]")
    return names[args["key_cache"].dtype], dims


def _execute_append(key: Any, value: Any, key_cache: Any, value_cache: Any, key_scales: Any, value_scales: Any,
                    slot_mapping: Any, *, torch_module: Any, runtime: OperatorRuntime, key_of_call: Any = None) -> Any:
    args = Args("paged_cache_append_8bit", torch_module, key=key, value=value, key_cache=key_cache,
                value_cache=value_cache, key_scales=key_scales, value_scales=value_scales, slot_mapping=slot_mapping)
    args.tensors(key=3, value=3).alike("key", "value")
    cache_dtype, (num_blocks, block_size, kv_heads, head_dim) = _check_cache(args)
    args.indices(slot_mapping=1)
    args.expect(key_cache.device == key.device and slot_mapping.device == key.device,
                "caches and slot_mapping must use the same device as key")
    tokens = args.dims("key")[0]
    args.expect(args.dims("value") == args.dims("key"), "key and value must have the same shape")
    args.expect(args.dims("key") == (tokens, kv_heads, head_dim) and head_dim in HEAD_DIMS,
                "heads and head_dim must match the cache and head_dim be one of 64, 128, 256")
    args.expect(block_size <= MAXIMUM_BLOCK_SIZE, f"block_size must be at most {MAXIMUM_BLOCK_SIZE}")
    args.expect(tokens <= MAXIMUM_TOKENS, "tokens must be below 2**30")
    args.expect(args.dims("slot_mapping") == (tokens,), "slot_mapping must contain one slot per token")
    args.expect(all(args[n].is_contiguous() for n in ("key_cache", "value_cache", "key_scales", "value_scales",
                                                      "slot_mapping")), "caches, scales and slot_mapping must be contiguous")
    args.expect(key_cache.data_ptr() != value_cache.data_ptr() and key_scales.data_ptr() != value_scales.data_ptr(),
                "keys and values must have caches and scales of their own")
    context = args.context(*args.values)
    args.expect(not context.requires_grad, "is inference-only and does not support autograd")
    signature = {
        "dtype": context.dtype, "cache_dtype": cache_dtype, "kv_heads": kv_heads, "head_dim": head_dim,
        "block_size": block_size, "index_dtype": args.index_dtype("slot_mapping"),
        "cache_layout": "block_slot_head_dim", "requires_grad": False,
    }
    result = dispatch(
        args, runtime, semantic_version="1.0", signature=signature, device_index=context.device_index,
        native_arguments=(key, value, key_cache, value_cache, key_scales, value_scales, slot_mapping),
        fallback=cuda_builtin.paged_cache_append_8bit, fallback_selected=cuda_builtin.SELECTED_PAGED_APPEND_8BIT,
    )
    remember_call(runtime, key_of_call, "paged_cache_append_8bit", context.device_index, signature)
    return tuple(result)


def _execute_attention(query: Any, key_cache: Any, value_cache: Any, key_scales: Any, value_scales: Any,
                       block_tables: Any, context_lengths: Any, scale: float | None = None, *, torch_module: Any,
                       runtime: OperatorRuntime, key_of_call: Any = None) -> Any:
    args = Args("paged_attention_decode_8bit", torch_module, query=query, key_cache=key_cache, value_cache=value_cache,
                key_scales=key_scales, value_scales=value_scales, block_tables=block_tables,
                context_lengths=context_lengths)
    args.tensors(query=3)
    cache_dtype, (num_blocks, block_size, kv_heads, cache_head_dim) = _check_cache(args)
    args.indices(block_tables=2, context_lengths=1)
    args.expect(key_cache.device == query.device and block_tables.device == query.device
                and context_lengths.device == query.device, "caches and index tensors must use the same device as query")
    args.expect(block_tables.dtype == context_lengths.dtype, "block_tables and context_lengths must use the same dtype",
                TypeError)
    batch, query_heads, head_dim = args.dims("query")
    table_rows, max_blocks = args.dims("block_tables")
    args.expect(min(batch, query_heads) > 0, "tensor dimensions must be positive")
    args.expect(cache_head_dim == head_dim and head_dim in HEAD_DIMS,
                "head_dim must match cache and be one of 64, 128, 256")
    args.expect(query_heads % kv_heads == 0, "query_heads must be divisible by kv_heads")
    args.expect(table_rows == batch and max_blocks > 0, "block_tables must have shape [batch, max_blocks]")
    args.expect(max_blocks * block_size < 2**31 - 64, "max_blocks * block_size must be below 2**31 - 64")
    args.expect(args.dims("context_lengths") == (batch,), "context_lengths must contain one length per sequence")
    context = args.inference_only(*args.values)
    scale_value, scale_mode = args.scale(scale, head_dim)
    signature = {
        "dtype": context.dtype, "cache_dtype": cache_dtype, "query_heads": query_heads, "kv_heads": kv_heads,
        "head_dim": head_dim, "block_size": block_size, "index_dtype": args.index_dtype("block_tables"),
        "cache_layout": "block_slot_head_dim", "scale_mode": scale_mode, "contiguous": True, "requires_grad": False,
    }
    result = dispatch(
        args, runtime, semantic_version="1.0", signature=signature, device_index=context.device_index,
        native_arguments=(query, key_cache, value_cache, key_scales, value_scales, block_tables, context_lengths,
                          scale_value),
        fallback=cuda_builtin.paged_attention_decode_8bit,
        fallback_selected=cuda_builtin.SELECTED_PAGED_ATTENTION_8BIT,
    )
    remember_call(runtime, key_of_call, "paged_attention_decode_8bit", context.device_index, signature)
    return result


def paged_cache_append_8bit(key: Any, value: Any, key_cache: Any, value_cache: Any, key_scales: Any,
                            value_scales: Any, slot_mapping: Any) -> tuple[Any, Any, Any, Any]:
    """Store new keys and values in an 8-bit paged cache, in place; returns caches and scales."""

    runtime, call = default_operator_runtime(), None
    try:
        call = ("paged_cache_append_8bit", key.dtype, key.device, key_cache.dtype, key_cache.shape[1:], slot_mapping.dtype)
        result = quick_call(runtime, call, (key, value, key_cache, value_cache, key_scales, value_scales, slot_mapping))
        if result is not None:
            return tuple(result)
    except AttributeError:
        call = None  # no tensors: the checks say so
    return _execute_append(key, value, key_cache, value_cache, key_scales, value_scales, slot_mapping,
                           torch_module=torch_runtime("paged_cache_append_8bit"), runtime=runtime, key_of_call=call)


def paged_attention_decode_8bit(query: Any, key_cache: Any, value_cache: Any, key_scales: Any, value_scales: Any,
                                block_tables: Any, context_lengths: Any, scale: float | None = None) -> Any:
    """Attend one query token per sequence over an 8-bit paged K/V cache."""

    runtime, call = default_operator_runtime(), None
    if scale is None or type(scale) is float:
        try:
            shape = query.shape
            call = ("paged_attention_decode_8bit", query.dtype, query.device, shape[1:], key_cache.dtype, key_cache.shape[1:],
                    block_tables.dtype, scale is None)
            result = quick_call(runtime, call, (query, key_cache, value_cache, key_scales, value_scales, block_tables,
                                                context_lengths, shape[2] ** -0.5 if scale is None else scale))
            if result is not None:
                return result
        except (AttributeError, IndexError):
            call = None  # no tensors of the right ranks: the checks say so
    return _execute_attention(query, key_cache, value_cache, key_scales, value_scales, block_tables, context_lengths,
                              scale, torch_module=torch_runtime("paged_attention_decode_8bit"), runtime=runtime,
                              key_of_call=call)
