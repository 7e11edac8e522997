"""rk.paged_slots on the GPU against a loop over the requests: every output exactly."""

from __future__ import annotations

import numpy as np
import pytest

import paged8_reference as ref
from radeon_kernels import _native, device_status

pytestmark = pytest.mark.gpu


def _run(tables, has, gets, free, num_tokens, block_size, index):
    import torch

    import radeon_kernels as rk

    dtype = {"int32": torch.int32, "int64": torch.int64}[index]
    device_tables = torch.tensor(tables).to(dtype).cuda()
    assert device_status() == _native.RK_OK
    out = rk.paged_slots(device_tables, torch.tensor(has).to(dtype).cuda(), torch.tensor(gets).to(dtype).cuda(),
                         torch.tensor(free, dtype=torch.int64).to(dtype).cuda(), num_tokens=num_tokens,
                         block_size=block_size)
    assert [t.dtype for t in out] == [torch.int64, dtype, dtype, dtype]
    status = device_status()
    want = ref.slots(np.array(tables), np.array(has), np.array(gets), list(free), num_tokens, block_size)
    for got, expected in zip((*out, device_tables), want[:3] + (np.array([want[3]]), want[4])):
        np.testing.assert_array_equal(got.cpu().numpy(), expected)
    assert status == (_native.RK_OK if want[5] else _native.RK_ERR_INVALID_ARGUMENT)
    assert rk.get_last_dispatch()["selected"] == "native/paged_slots"
    return out


def _case(seed, batch, longest, most, block_size, extra=0):
    rng = np.random.default_rng(seed)
    has, gets = rng.integers(0, longest + 1, batch), rng.integers(0, most + 1, batch)
    width = max(1, -(-int((has + gets).max()) // block_size)) + extra
    blocks = rng.permutation(batch * width + 8)
    tables = np.full((batch, width), -7)  # entries beyond a request's blocks: left as they are
    at = 0
    for b in range(batch):
        n = -(-int(has[b]) // block_size)
        tables[b, :n] = blocks[at : at + n]
        at += n
    return tables, has, gets, blocks[at:].tolist()


@pytest.mark.parametrize("index", ["int32", "int64"])
@pytest.mark.parametrize(
    "batch, longest, most, block_size, padding",
    [
        (1, 0, 1, 16, 0),
        (1, 5, 1, 1, 0),
        (3, 17, 9, 7, 4),
        (64, 300, 1, 16, 0),
        (33, 100, 700, 24, 1000),   # several CTAs of tokens, padding across a CTA's edge
        (255, 50, 2, 8, 3),
        (256, 50, 3, 8, 0),
        (257, 50, 3, 8, 0),         # larger CTAs
        (700, 20, 5, 4, 129),
        (2, 0, 40000, 64, 1),
        (1024, 9, 30, 5, 0),
        (1025, 40, 1, 16, 7),       # a second round of requests
        (2500, 3, 4, 2, 5000),
    ],
)
def test_matches_a_loop(batch, longest, most, block_size, padding, index):
    tables, has, gets, free = _case(batch, batch, longest, most, block_size, extra=batch % 3)
    _run(tables, has, gets, free, int(gets.sum()) + padding, block_size, index)


def test_nothing_to_place():
    tables, has, _, free = _case(1, 4, 30, 0, 8)
    out = _run(tables, has, np.zeros(4, int), free, 0, 8, "int32")
    assert out[0].numel() == 0
    _run(tables, has, np.zeros(4, int), [], 5, 8, "int64")  # only padding, no free block


def test_free_list_too_short():
    """Entries and slots that miss a block are -1; the count says how many were needed."""
    tables, has, gets, free = _case(2, 9, 20, 40, 8)
    needed = int((-(-(has + gets) // 8) - -(-has // 8)).sum())
    out = _run(tables, has, gets, free[: needed - 3], int(gets.sum()), 8, "int32")
    assert int(out[3]) == needed


def test_tokens_past_the_table_and_the_buffer():
    tables = np.array([[4, -1], [9, 2], [-1, -1]])
    # Request 1 overruns its row by 4 tokens; the third gets the only free block that is left.
    _run(tables, [5, 14, 0], [3, 6, 8], [30, 31, 32], 17, 8, "int64")
    _run(tables, [5, 8, 0], [3, 8, 8], [30, 31, 32], 10, 8, "int32")  # buffer of 10 for 19 tokens


def test_negative_lengths_and_missing_blocks():
    _run(np.array([[1, 2], [3, 4]]), [-5, 3], [4, -2], [7, 8, 9], 6, 4, "int64")
    # A table entry that should be there and is not: its tokens have no slot.
    _run(np.array([[-1, 2]]), [2], [4], [7], 4, 4, "int32")


def test_large_numbers_of_blocks():
    """Slots past 2^31 with int32 tables."""
    out = _run(np.array([[2**30, -1]]), [3], [5], [2**30 + 1], 8, 4, "int32")
    assert int(out[0][0]) == 2**30 * 4 + 3


def test_huge_lengths_do_not_overflow():
    _run(np.array([[1, 2]]), [2**62], [2**62], [5], 3, 4, "int64")


def test_replayed_graph_follows_its_inputs():
    import torch

    import radeon_kernels as rk

    tables, has, gets, free = _case(5, 6, 30, 10, 8, extra=4)
    t = [torch.tensor(x).cuda() for x in (tables, has, gets)] + [torch.tensor(free).cuda()]
    tokens = 80
    rk.paged_slots(t[0].clone(), *t[1:], num_tokens=tokens, block_size=8)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = rk.paged_slots(*t, num_tokens=tokens, block_size=8)
    for seed in (6, 7):
        tables, has, gets, free2 = _case(seed, 6, 30, 10, 8)
        wide = np.full(t[0].shape, -1)
        wide[:, : tables.shape[1]] = tables[:, : wide.shape[1]]
        t[0].copy_(torch.tensor(wide))
        t[1].copy_(torch.tensor(has))
        t[2].copy_(torch.tensor(gets))
        graph.replay()
        want = ref.slots(wide, has, gets, free, tokens, 8)
        for got, expected in zip((*out, t[0]), want[:3] + (np.array([want[3]]), want[4])):
            np.testing.assert_array_equal(got.cpu().numpy(), expected)
    device_status()


@pytest.mark.parametrize("index", ["int32", "int64"])
@pytest.mark.parametrize("batch", [1, 5, 300, 1100])
def test_a_single_request_overruns_the_buffer(batch, index):
    """More tokens than the buffer holds are reported, whichever request has them all."""
    for at in {0, batch // 2, batch - 1}:
        gets = np.zeros(batch, int)
        gets[at] = 100
        tables = np.full((batch, 8), -1)
        for tokens in (99, 50, 1, 0):
            _run(tables, np.zeros(batch, int), gets, list(range(20)), tokens, 16, index)
        _run(tables, np.zeros(batch, int), gets, list(range(20)), 100, 16, index)  # just enough


def test_no_buffer_and_tokens_to_place():
    _run(np.full((3, 4), -1), [0, 5, 0], [1, 0, 2], [7, 8, 9], 0, 8, "int32")
    _run(np.full((2, 4), -1), [0, 0], [1, 1], [7, 8, 9], 0, 8, "int64")


@pytest.mark.parametrize("block_size", [2, 5, 16, 2**20])
def test_entries_whose_slots_exceed_64_bits(block_size):
    """They have no slot and are reported, in a table as in the free list; the largest that fit are mapped."""
    import torch

    import radeon_kernels as rk

    most = (2**63 - 1 - (block_size - 1)) // block_size
    for held, free, well in ((most, most - 1, True), (most, 2**63 - 1, False), (2**63 - 1, most, False), (2**62, 2**62, None)):
        fits = [b <= most for b in (held, free)]
        tables = torch.tensor([[held, -1]], device="cuda")
        slots, *_ = rk.paged_slots(tables, torch.tensor([1], device="cuda"), torch.tensor([block_size], device="cuda"),
                                   torch.tensor([free], device="cuda"), num_tokens=block_size, block_size=block_size)
        want = [held * block_size + i if fits[0] else -1 for i in range(1, block_size)]
        want.append(free * block_size if fits[1] else -1)
        assert slots.tolist() == want
        assert device_status() == (_native.RK_OK if all(fits) else _native.RK_ERR_INVALID_ARGUMENT)
        if well is not None:
            assert all(fits) == well
