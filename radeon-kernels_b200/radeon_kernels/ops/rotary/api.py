"""Public rotary positions: ``rk.rotary_embedding(query, key, positions, frequencies, *,
interleaved=False, amplitude=1.0)`` and ``rk.rotary_frequencies(...)``.

``query [tokens, query_heads, head_dim]`` and ``key [tokens, kv_heads, head_dim]`` (CUDA
fp16/bf16) are turned by their ``positions [tokens]`` (int32/int64): the first ``2 *
len(frequencies)`` elements of each head are pairs ``(i, i + n)``, or ``(2i, 2i + 1)`` when
``interleaved``, and pair ``i`` at position ``p`` becomes ``amplitude * (a cos - b sin, b cos +
a sin)`` at the angle ``p * frequencies[i]``; the rest of the head is copied.  The result is a
new dense pair ``(query, key)``.  Queries and keys that are slices of one projection are read
in place (any stride between tokens and heads); inputs that require gradients get the inverse
rotation of theirs.  Forward-mode tangents are refused.

``frequencies`` (float64, radians per position) is computed once by
:func:`rotary_frequencies`, which also knows the usual rules for stretching a model's context.
Angles are formed in float64 in the kernel, so far positions keep their precision.

The reference has no such operator; names, checks and dispatch are those of its neighbours.
Operator ``"rotary_embedding"`` (semantic version 1.0); the token count is not part of the
dispatch signature, so steps of every size share one decision.
"""

from __future__ import annotations

import math
from typing import Any

from radeon_kernels.ops._common import torch_runtime
from radeon_kernels.ops._frontend import Args, dispatch, quick_call, remember_call
from radeon_kernels.ops._runtime import OperatorRuntime, default_operator_runtime
from radeon_kernels.providers import cuda_builtin

MAXIMUM_HEAD_DIM = 1024
MAXIMUM_HEADS = 32767
SCALINGS = ("none", "linear", "ntk", "yarn")


def _execute(query: Any, key: Any, positions: Any, frequencies: Any, interleaved: bool = False,
             amplitude: float = 1.0, *, torch_module: Any, runtime: OperatorRuntime, key_of_call: Any = None) -> Any:
    args = Args("rotary_embedding", torch_module, query=query, key=key, positions=positions, frequencies=frequencies)
    args.tensors(query=3, key=3).alike("query", "key").indices(positions=1)
    args.expect(isinstance(frequencies, torch_module.Tensor), "frequencies must be a PyTorch tensor", TypeError)
    args.expect(frequencies.dim() == 1, "frequencies must be rank 1")
    args.expect(frequencies.dtype == torch_module.float64, "frequencies must use torch.float64", TypeError)
    args.expect(positions.device == query.device and frequencies.device == query.device,
                "positions and frequencies must use the same device as query")
    args.expect(isinstance(interleaved, bool), "interleaved must be bool", TypeError)
    args.expect(not isinstance(amplitude, bool) and isinstance(amplitude, (int, float)), "amplitude must be a number",
                TypeError)
    args.expect(math.isfinite(amplitude), "amplitude must be finite")
    tokens, query_heads, head_dim = args.dims("query")
    key_tokens, kv_heads, key_head_dim = args.dims("key")
    (pairs,) = args.dims("frequencies")
    args.expect(key_tokens == tokens and key_head_dim == head_dim, "query and key must share tokens and head_dim")
    args.expect(args.dims("positions") == (tokens,), "positions must hold one position per token")
    args.expect(0 < query_heads <= MAXIMUM_HEADS and 0 < kv_heads <= MAXIMUM_HEADS,
                f"head counts must be in [1, {MAXIMUM_HEADS}]")
    args.expect(head_dim <= MAXIMUM_HEAD_DIM, f"head_dim must be at most {MAXIMUM_HEAD_DIM}")
    args.expect(1 <= pairs and 2 * pairs <= head_dim, "frequencies must hold 1 to head_dim // 2 pairs")
    args.expect(not frequencies.requires_grad, "frequencies must not require gradients")
    context = args.context("query", "key")
    signature = {
        "dtype": context.dtype, "query_heads": query_heads, "kv_heads": kv_heads, "head_dim": head_dim,
        "rotary_dim": 2 * pairs, "pairing": "interleaved" if interleaved else "halves",
        "index_dtype": args.index_dtype("positions"), "requires_grad": context.requires_grad,
    }
    result = dispatch(
        args, runtime, semantic_version="1.0", signature=signature, device_index=context.device_index,
        native_arguments=(query, key, positions, frequencies, interleaved, float(amplitude)),
        fallback=cuda_builtin.rotary_embedding, fallback_selected=cuda_builtin.SELECTED_ROTARY,
    )
    remember_call(runtime, key_of_call, "rotary_embedding", context.device_index, signature)
    return tuple(result)


def rotary_embedding(query: Any, key: Any, positions: Any, frequencies: Any, *, interleaved: bool = False,
                     amplitude: float = 1.0) -> tuple[Any, Any]:
    """Rotate queries and keys by their positions; returns new ``(query, key)``."""

    runtime, call = default_operator_runtime(), None
    if type(amplitude) is float and type(interleaved) is bool:
        try:
            call = ("rotary_embedding", query.dtype, query.device, query.shape[1:], key.shape[1], positions.dtype,
                    frequencies.shape, interleaved, query.requires_grad or key.requires_grad)
            result = quick_call(runtime, call, (query, key, positions, frequencies, interleaved, amplitude))
            if result is not None:
                return tuple(result)
        except (AttributeError, IndexError):
            call = None  # no tensors of the right ranks: the checks say so
    return _execute(query, key, positions, frequencies, interleaved, amplitude,
                    torch_module=torch_runtime("rotary_embedding"), runtime=runtime, key_of_call=call)


def rotary_frequencies(rotary_dim: int, *, base: float = 10000.0, scaling: str = "none", factor: float = 1.0,
                       original_length: int | None = None, fast_turns: float = 32.0, slow_turns: float = 1.0,
                       device: Any = "cuda") -> Any:
    """Radians per position of each of the ``rotary_dim // 2`` pairs, as a float64 tensor.

    Pair ``i`` turns by ``base ** (-2 i / rotary_dim)`` per position.  ``scaling`` stretches a
    model trained on shorter contexts by ``factor``:

    * ``"linear"``: every frequency is divided by ``factor`` (position interpolation);
    * ``"ntk"``: the base grows by ``factor ** (rotary_dim / (rotary_dim - 2))``, which leaves
      the fastest pair alone and divides the slowest by ``factor``;
    * ``"yarn"``: pairs that turn more than ``fast_turns`` times within ``original_length``
      positions stay, those that turn less than ``slow_turns`` times are divided by
      ``factor``, and the ones between are blended linearly by their index.  Such models
      are run with an ``amplitude`` of ``0.1 * ln(factor) + 1``.
    """

    import torch

    for name, value in (("rotary_dim", rotary_dim), ("base", base), ("factor", factor), ("fast_turns", fast_turns),
                        ("slow_turns", slow_turns)):
        if isinstance(value, bool) or not isinstance(value, int if name == "rotary_dim" else (int, float)):
            raise TypeError(f"rotary_frequencies {name} must be {'an int' if name == 'rotary_dim' else 'a number'}")
    if rotary_dim < 2 or rotary_dim % 2:
        raise ValueError("rotary_frequencies rotary_dim must be even and positive")
    if not (math.isfinite(base) and base > 1.0):
        raise ValueError("rotary_frequencies base must be finite and above 1")
    if scaling not in SCALINGS:
        raise ValueError(f"rotary_frequencies scaling must be one of {', '.join(SCALINGS)}")
    if not (math.isfinite(factor) and factor >= 1.0):
        raise ValueError("rotary_frequencies factor must be finite and at least 1")
    if scaling == "ntk":
        if rotary_dim < 4:
            raise ValueError("rotary_frequencies scaling 'ntk' needs rotary_dim of at least 4")
        base = base * factor ** (rotary_dim / (rotary_dim - 2))
    frequencies = [base ** (-2.0 * i / rotary_dim) for i in range(rotary_dim // 2)]
    if scaling == "linear":
        frequencies = [f / factor for f in frequencies]
    elif scaling == "yarn":
        if isinstance(original_length, bool) or not isinstance(original_length, int) or original_length < 1:
            raise ValueError("rotary_frequencies scaling 'yarn' needs original_length, the trained context length")
        if not (math.isfinite(fast_turns) and math.isfinite(slow_turns) and fast_turns > slow_turns > 0.0):
            raise ValueError("rotary_frequencies turns must satisfy fast_turns > slow_turns > 0")

        def index_of(turns: float) -> float:
            # The (fractional) pair that turns `turns` times within original_length positions.
            return rotary_dim * math.log(original_length / (turns * 2.0 * math.pi)) / (2.0 * math.log(base))

        low = max(math.floor(index_of(fast_turns)), 0)
        high = min(math.ceil(index_of(slow_turns)), rotary_dim - 1)
        shares = [min(max((i - low) / max(high - low, 1e-3), 0.0), 1.0) for i in range(rotary_dim // 2)]
        frequencies = [f / factor * s + f * (1.0 - s) for f, s in zip(frequencies, shares)]
    return torch.tensor(frequencies, dtype=torch.float64, device=device)
