"""rk.rotary_embedding on the GPU against the 64-bit rotation: pairings, partial heads, odd
sizes, strides, far and negative positions, gradients, streams and graphs."""

from __future__ import annotations

import numpy as np
import pytest

import paged8_reference as ref

pytestmark = pytest.mark.gpu


def _dtype(name):
    import torch

    return {"bf16": torch.bfloat16, "fp16": torch.float16}[name]


def _check(out, x, positions, frequencies, interleaved, amplitude, dtype, inverse=False):
    want, slack = ref.rotary(x.detach().double().cpu().numpy(), positions.cpu().numpy(), frequencies.cpu().numpy(),
                             interleaved, amplitude, inverse)
    got = out.detach().double().cpu().numpy()
    bound = slack * (1 + ref.HALF_STEP[dtype]) + ref.rounding(want, dtype)
    assert out.is_contiguous() and got.shape == want.shape
    worst = np.max(np.abs(got - want) - bound, initial=-1.0)
    assert worst <= 0, worst


def _inputs(tokens, query_heads, kv_heads, dim, dtype, seed=0):
    import torch

    gen = torch.Generator().manual_seed(seed)
    return tuple(torch.randn((tokens, h, dim), generator=gen).to(_dtype(dtype)).cuda() for h in (query_heads, kv_heads))


CASES = [
    # tokens, query heads, kv heads, head_dim, rotary_dim
    (1, 32, 8, 128, 128),
    (5, 4, 1, 64, 64),
    (3, 5, 3, 80, 20),   # pairs that are no whole vectors
    (2, 1, 1, 2, 2),     # the smallest head
    (7, 3, 2, 6, 4),
    (4, 2, 2, 96, 24),
    (9, 28, 4, 256, 64),
    (2, 2, 1, 1024, 1024),
    (2500, 3, 2, 128, 64),  # several tokens to a CTA, the last CTA ragged
    (2501, 2, 1, 10, 10),
]


@pytest.mark.parametrize("interleaved", [False, True], ids=["halves", "interleaved"])
@pytest.mark.parametrize("dtype", ["bf16", "fp16"])
@pytest.mark.parametrize("tokens, query_heads, kv_heads, dim, rotary_dim", CASES)
def test_matches_the_rotation(tokens, query_heads, kv_heads, dim, rotary_dim, dtype, interleaved):
    import torch

    import radeon_kernels as rk

    query, key = _inputs(tokens, query_heads, kv_heads, dim, dtype)
    index = torch.int32 if tokens % 2 else torch.int64
    positions = (torch.arange(tokens, device="cuda") * 37 + 5).to(index)
    frequencies = rk.rotary_frequencies(rotary_dim)
    amplitude = 1.0 if dtype == "bf16" else 1.2079
    out_q, out_k = rk.rotary_embedding(query, key, positions, frequencies, interleaved=interleaved, amplitude=amplitude)
    _check(out_q, query, positions, frequencies, interleaved, amplitude, dtype)
    _check(out_k, key, positions, frequencies, interleaved, amplitude, dtype)
    assert rk.get_last_dispatch()["selected"] == "native/rotary_embedding"


@pytest.mark.parametrize("interleaved", [False, True], ids=["halves", "interleaved"])
@pytest.mark.parametrize("offset", [1, 2, 4, 8])
@pytest.mark.parametrize("tokens, heads, dim, rotary_dim", [(3, 3, 96, 24), (700, 2, 80, 20), (2500, 1, 72, 40), (5000, 3, 12, 4)])
def test_vectors_of_every_width(tokens, heads, dim, rotary_dim, offset, interleaved):
    """Rows that start 2, 4, 8 and 16 bytes off, with sizes that allow 2, 4, 8 and 16 bytes at a time; many tokens of few heads."""
    import torch

    import radeon_kernels as rk

    gen = torch.Generator().manual_seed(tokens)
    flat = torch.randn(offset + tokens * (heads + 1) * dim, generator=gen).half().cuda()[offset:].view(tokens, heads + 1, dim)
    query, key = flat[:, :heads], flat[:, heads:]
    positions = torch.arange(tokens, dtype=torch.int32, device="cuda") * 11
    frequencies = rk.rotary_frequencies(rotary_dim)
    out_q, out_k = rk.rotary_embedding(query, key, positions, frequencies, interleaved=interleaved)
    _check(out_q, query, positions, frequencies, interleaved, 1.0, "fp16")
    _check(out_k, key, positions, frequencies, interleaved, 1.0, "fp16")


@pytest.mark.parametrize("positions", [[0], [2**30 + 7, -3], [131071, 1048575, -(2**31)], [2**40, -(2**40) + 1]])
def test_far_and_negative_positions(positions):
    import torch

    import radeon_kernels as rk

    query, key = _inputs(len(positions), 2, 1, 64, "fp16", seed=3)
    at = torch.tensor(positions, dtype=torch.int64, device="cuda")
    for scaling in ("none", "linear", "ntk", "yarn"):
        frequencies = rk.rotary_frequencies(64, scaling=scaling, factor=8.0, original_length=4096)
        out_q, out_k = rk.rotary_embedding(query, key, at, frequencies)
        _check(out_q, query, at, frequencies, False, 1.0, "fp16")
        _check(out_k, key, at, frequencies, False, 1.0, "fp16")


@pytest.mark.parametrize("interleaved", [False, True], ids=["halves", "interleaved"])
@pytest.mark.parametrize("layout", ["joint", "offset", "heads-first", "last-strided", "broadcast"])
def test_strided_inputs(layout, interleaved):
    import torch

    import radeon_kernels as rk

    tokens, hq, hk, dim = 6, 4, 2, 64
    gen = torch.Generator().manual_seed(8)
    if layout == "joint":
        joint = torch.randn((tokens, hq + 2 * hk, dim), generator=gen).bfloat16().cuda()
        query, key = joint[:, :hq], joint[:, hq : hq + hk]
    elif layout == "offset":  # rows that start on an odd element: no 16-byte vectors
        flat = torch.randn(tokens * (hq + hk) * dim + 1, generator=gen).bfloat16().cuda()
        query = flat[1 : 1 + tokens * hq * dim].view(tokens, hq, dim)
        key = flat[1 + tokens * hq * dim :].view(tokens, hk, dim)
    elif layout == "heads-first":
        query = torch.randn((hq, tokens, dim), generator=gen).bfloat16().cuda().transpose(0, 1)
        key = torch.randn((hk, tokens, dim), generator=gen).bfloat16().cuda().transpose(0, 1)
    elif layout == "last-strided":
        query = torch.randn((tokens, hq, 2 * dim), generator=gen).bfloat16().cuda()[..., ::2]
        key = torch.randn((tokens, dim, hk), generator=gen).bfloat16().cuda().transpose(1, 2)
    else:
        query = torch.randn((1, hq, dim), generator=gen).bfloat16().cuda().expand(tokens, hq, dim)
        key = torch.randn((tokens, 1, dim), generator=gen).bfloat16().cuda().expand(tokens, hk, dim)
    positions = torch.arange(2 * tokens, dtype=torch.int32, device="cuda")[::2]
    frequencies = rk.rotary_frequencies(32)
    out_q, out_k = rk.rotary_embedding(query, key, positions, frequencies, interleaved=interleaved)
    _check(out_q, query, positions, frequencies, interleaved, 1.0, "bf16")
    _check(out_k, key, positions, frequencies, interleaved, 1.0, "bf16")


def test_no_tokens():
    import torch

    import radeon_kernels as rk

    query, key = _inputs(0, 4, 2, 64, "bf16")
    empty = torch.empty(0, dtype=torch.int32, device="cuda")
    out_q, out_k = rk.rotary_embedding(query, key, empty, rk.rotary_frequencies(64))
    assert out_q.shape == (0, 4, 64) and out_k.shape == (0, 2, 64)


def test_non_finite_values_stay_in_their_pairs():
    import torch

    import radeon_kernels as rk

    query, key = _inputs(1, 1, 1, 64, "fp16")
    query[0, 0, 3], query[0, 0, 60] = float("inf"), float("nan")
    positions = torch.tensor([9], device="cuda")
    out, _ = rk.rotary_embedding(query, key, positions, rk.rotary_frequencies(32))
    out = out[0, 0].cpu()
    touched = [3, 19]  # pair (3, 3 + 16); element 60 is behind the rotated part
    assert not torch.isfinite(out[touched]).any() and torch.isnan(out[60])
    rest = [i for i in range(64) if i not in touched + [60]]
    assert torch.isfinite(out[rest]).all()


@pytest.mark.parametrize("interleaved", [False, True], ids=["halves", "interleaved"])
@pytest.mark.parametrize("dtype", ["bf16", "fp16"])
@pytest.mark.parametrize("dim, rotary_dim", [(128, 128), (80, 20), (10, 6)])
def test_gradients_are_the_inverse_rotation(dim, rotary_dim, dtype, interleaved):
    import torch

    import radeon_kernels as rk

    tokens = 11
    query, key = _inputs(tokens, 3, 2, dim, dtype, seed=1)
    grad_q, grad_k = _inputs(tokens, 3, 2, dim, dtype, seed=2)
    query.requires_grad_(True)
    key.requires_grad_(True)
    positions = torch.arange(tokens, device="cuda") * 1000
    frequencies = rk.rotary_frequencies(rotary_dim)
    out = rk.rotary_embedding(query, key, positions, frequencies, interleaved=interleaved, amplitude=1.5)
    got_q, got_k = torch.autograd.grad(out, (query, key), (grad_q, grad_k))
    _check(out[0], query, positions, frequencies, interleaved, 1.5, dtype)
    _check(got_q, grad_q, positions, frequencies, interleaved, 1.5, dtype, inverse=True)
    _check(got_k, grad_k, positions, frequencies, interleaved, 1.5, dtype, inverse=True)


def test_gradients_against_differences():
    """The operator is linear: a difference along e is its value at e, exactly, up to roundings.

    <g, R e> and <R^T g, e> differ by the roundings of both results: each output is off by
    half a step of its value and the fp32 slack, so the products by their sums."""
    import torch

    import radeon_kernels as rk

    tokens, dim = 4, 64
    query, key = _inputs(tokens, 2, 2, dim, "fp16", seed=5)
    (direction, grad), _ = _inputs(tokens, 2, 2, dim, "fp16", seed=6), None
    positions, frequencies = torch.tensor([0, 3, 77, 5000], device="cuda"), rk.rotary_frequencies(dim)
    query.requires_grad_(True)
    out, _ = rk.rotary_embedding(query, key, positions, frequencies)
    (back,) = torch.autograd.grad(out, query, grad)
    with torch.no_grad():
        at, _ = rk.rotary_embedding(query + direction, key, positions, frequencies)
        there, _ = rk.rotary_embedding(query, key, positions, frequencies)
        moved = (query + direction).double() - query.double()  # the step that was taken
    forward = (grad.double() * (at.double() - there.double())).sum().item()
    backward = (back.double() * moved).sum().item()
    half = 2.0**-11 + 2.0**-19
    bound = (grad.double().abs() * (at.double().abs() + there.double().abs() + 2.0**-6)).sum() * half
    bound += (back.double().abs() * moved.abs()).sum() * half + moved.abs().sum() * 2.0**-6 * half
    assert abs(forward - backward) <= bound.item()


def test_gradients_of_shared_and_single_inputs():
    import torch

    import radeon_kernels as rk

    tokens, dim = 5, 64
    positions, frequencies = torch.arange(tokens, device="cuda"), rk.rotary_frequencies(dim)
    # One key head expanded to four: its gradient is the sum of theirs.
    single = torch.randn(tokens, 1, dim, device="cuda", dtype=torch.float32).half().requires_grad_(True)
    query, _ = _inputs(tokens, 4, 1, dim, "fp16")
    grad = torch.randn(tokens, 4, dim, device="cuda").half()
    _, out = rk.rotary_embedding(query, single.expand(tokens, 4, dim), positions, frequencies)
    (got,) = torch.autograd.grad(out, single, grad)
    rotated, _ = rk.rotary_embedding(grad, grad, -positions, frequencies)
    want = rotated.double().sum(1, keepdim=True)
    # autograd adds the four rounded gradients in fp16 or wider: at most 4 more roundings.
    assert ((got.double() - want).abs() <= 4 * 2.0**-11 * rotated.double().abs().sum(1, keepdim=True) + 2.0**-24).all()
    # The same tensor as query and key, and only one output used.
    both = torch.randn(tokens, 2, dim, device="cuda").half().requires_grad_(True)
    out_q, out_k = rk.rotary_embedding(both, both, positions, frequencies)
    assert torch.equal(out_q, out_k)
    g = torch.randn_like(out_q)
    (one,) = torch.autograd.grad(out_q, both, g, retain_graph=True)
    (two,) = torch.autograd.grad((out_q, out_k), both, (g, g))
    assert torch.equal(two, one + one)


def test_second_derivative_is_the_rotation_again():
    import torch

    import radeon_kernels as rk

    query, key = _inputs(3, 2, 1, 64, "fp16", seed=4)
    positions, frequencies = torch.arange(3, device="cuda") + 10, rk.rotary_frequencies(64)
    query.requires_grad_(True)
    out, _ = rk.rotary_embedding(query, key, positions, frequencies)
    weight = torch.randn_like(out).requires_grad_(True)
    (grad,) = torch.autograd.grad(out, query, weight, create_graph=True)
    along = torch.randn_like(grad)
    (again,) = torch.autograd.grad(grad, weight, along)
    _check(again, along, positions, frequencies, False, 1.0, "fp16")


def test_in_a_graph_forward_and_backward():
    import torch

    import radeon_kernels as rk

    tokens, dim = 33, 128
    query, key = _inputs(tokens, 4, 2, dim, "bf16")
    grad_q, grad_k = _inputs(tokens, 4, 2, dim, "bf16", seed=9)
    positions, frequencies = torch.arange(tokens, device="cuda"), rk.rotary_frequencies(dim)
    query.requires_grad_(True)
    key.requires_grad_(True)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        for _ in range(2):
            out = rk.rotary_embedding(query, key, positions, frequencies)
            torch.autograd.grad(out, (query, key), (grad_q, grad_k))
        del out  # no eager graph of these leaves lives during the capture
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = rk.rotary_embedding(query, key, positions, frequencies)
        grads = torch.autograd.grad(out, (query, key), (grad_q, grad_k))
    for shift in (0, 517):
        with torch.no_grad():
            query.copy_(torch.roll(query, 1, 0))
            positions.add_(shift)
        graph.replay()
        torch.cuda.synchronize()
        _check(out[0], query, positions, frequencies, False, 1.0, "bf16")
        _check(grads[1], grad_k, positions, frequencies, False, 1.0, "bf16", inverse=True)


def test_on_a_side_stream():
    import torch

    import radeon_kernels as rk

    query, key = _inputs(600, 8, 2, 128, "bf16")
    positions, frequencies = torch.arange(600, device="cuda"), rk.rotary_frequencies(128)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        out, _ = rk.rotary_embedding(query, key, positions, frequencies)
    torch.cuda.current_stream().wait_stream(side)
    torch.cuda.synchronize()
    _check(out, query, positions, frequencies, False, 1.0, "bf16")


@pytest.mark.parametrize("requires_grad", [False, True])
def test_forward_mode_tangents_are_refused(requires_grad):
    """Refused by first calls and by calls of a kind that has been served."""
    import torch
    from torch.autograd import forward_ad

    import radeon_kernels as rk

    rows = torch.randn((3, 2, 64), device="cuda").bfloat16()
    frequencies, positions = rk.rotary_frequencies(64), torch.arange(3, device="cuda")
    caches = [torch.zeros((1, 16, 2, 64), dtype=torch.int8, device="cuda") for _ in range(2)]
    scales = [torch.ones((1, 2), device="cuda") for _ in range(2)]
    tables = torch.zeros((3, 1), dtype=torch.int64, device="cuda")
    for served in (False, True):
        if served:
            rk.rotary_embedding(rows, rows, positions, frequencies)
            rk.paged_cache_append_8bit(rows, rows, *caches, *scales, positions)
            rk.paged_attention_decode_8bit(rows, *caches, *scales, tables, positions)
        with forward_ad.dual_level():
            dual = forward_ad.make_dual(rows.clone().requires_grad_(requires_grad), torch.ones_like(rows))
            for query, key in ((dual, rows), (rows, dual)):
                with pytest.raises(RuntimeError, match="forward-mode"):
                    rk.rotary_embedding(query, key, positions, frequencies)
            if requires_grad:
                continue  # the others refuse that in any case
            for key, value in ((dual, rows), (rows, dual)):
                with pytest.raises(RuntimeError, match="forward-mode"):
                    rk.paged_cache_append_8bit(key, value, *caches, *scales, positions)
            with pytest.raises(RuntimeError, match="forward-mode"):
                rk.paged_attention_decode_8bit(dual, *caches, *scales, tables, positions)
            assert not caches[0].any() or served
