"""rk.paged_cache_append_8bit and rk.paged_attention_decode_8bit on the GPU: the append bit by
bit against its 64-bit definition, the attention within the error of its roundings, and a
decode loop of all four operators."""

from __future__ import annotations

import numpy as np
import pytest

import paged8_reference as ref
from radeon_kernels import _native, device_status

pytestmark = pytest.mark.gpu


def _torch_dtype(name):
    import torch

    return {"bf16": torch.bfloat16, "fp16": torch.float16, "e4m3": torch.float8_e4m3fn, "int8": torch.int8}[name]


def _values(cache):
    """A cache's stored values as float64 on the host."""
    return cache.cpu().float().double().numpy()


def _random_cache(rng, shape, kind):
    import torch

    x = torch.from_numpy(rng.normal(size=shape).astype(np.float32)) * (ref.LARGEST[kind] / 4)
    x = x.clamp(-ref.LARGEST[kind], ref.LARGEST[kind])
    return (x.round().to(torch.int8) if kind == "int8" else x.to(torch.float8_e4m3fn)).cuda()


# ------------------------------------------------------------------------------ append
def _append(rng, rows, slots, kind, blocks, size, index="int64", scales=None, cache=None):
    """Runs one append of (key, value) rows and checks caches, scales and status."""
    import torch

    import radeon_kernels as rk

    key, value = rows
    heads, dim = key.shape[1], key.shape[2]
    shape = (blocks, size, heads, dim)
    caches = cache or [_random_cache(rng, shape, kind) for _ in range(2)]
    if scales is None:
        scales = [torch.from_numpy(2.0 ** rng.integers(-9, -3, (blocks, heads)).astype(np.float32)).cuda() for _ in range(2)]
    slot_mapping = torch.tensor(slots, dtype={"int32": torch.int32, "int64": torch.int64}[index]).cuda()
    before = [_values(c) for c in caches], [s.double().cpu().numpy() for s in scales]
    assert device_status() == _native.RK_OK
    out = rk.paged_cache_append_8bit(key, value, *caches, *scales, slot_mapping)
    assert rk.get_last_dispatch()["selected"] == "native/paged_cache_append_8bit"
    assert [o.data_ptr() for o in out] == [t.data_ptr() for t in (*caches, *scales)]
    well = True
    for i, x in enumerate((key, value)):
        want, want_scales, ok = ref.append(x.double().cpu().numpy(), before[0][i], before[1][i], np.array(slots, np.int64), kind)
        np.testing.assert_array_equal(scales[i].double().cpu().numpy(), want_scales)
        np.testing.assert_array_equal(_values(caches[i]), want)
        well = well and ok
    assert device_status() == (_native.RK_OK if well else _native.RK_ERR_INVALID_ARGUMENT)
    return caches, scales


def _rows(rng, tokens, heads, dim, dtype, spread=1.0):
    import torch

    size = np.exp(spread * rng.normal(size=(tokens, heads, 1)))
    return [torch.from_numpy((rng.normal(size=(tokens, heads, dim)) * size).astype(np.float32)).to(_torch_dtype(dtype)).cuda()
            for _ in range(2)]


def _prefill_slots(rng, blocks, size, lengths):
    """Slots of requests that start at random offsets, in shuffled blocks."""
    order, at, slots = rng.permutation(blocks), 0, []
    for n in lengths:
        start = int(rng.integers(0, size))
        need = -(-(start + n) // size)
        mine = order[at : at + need]
        at += need
        slots += [int(mine[(start + i) // size]) * size + (start + i) % size for i in range(n)]
    assert at <= blocks
    return slots


@pytest.mark.parametrize("kind", ["e4m3", "int8"])
@pytest.mark.parametrize("dtype", ["bf16", "fp16"])
@pytest.mark.parametrize(
    "dim, heads, size, lengths",
    [
        (64, 1, 16, [1]),
        (128, 8, 16, [1] * 40),
        (128, 3, 16, [5, 0, 16, 33, 1]),
        (256, 2, 8, [7, 25]),
        (64, 5, 24, [100, 3]),     # a block size that is no power of two
        (128, 1, 1, [9]),          # a token to a block
        (128, 9, 64, [70, 64]),    # more rows than a warp holds; more heads than warps
        (256, 1, 128, [300]),
        (64, 2, 1024, [1500]),
        (128, 2, 16, [1100, 1200]),  # enough tokens for claims
    ],
)
def test_append_matches_its_definition(dim, heads, size, lengths, dtype, kind):
    rng = np.random.default_rng(dim + size + heads)
    blocks = sum(-(-n // size) + 1 for n in lengths) + 2
    slots = _prefill_slots(rng, blocks, size, lengths)
    _append(rng, _rows(rng, len(slots), heads, dim, dtype), slots, kind, blocks, size, "int32" if size % 3 else "int64")


@pytest.mark.parametrize("tokens", [0, 2100], ids=["scan", "claims"])
@pytest.mark.parametrize("dim, heads, size", [(256, 2, 16), (256, 9, 64), (128, 5, 128), (64, 1, 1000), (256, 1, 1024), (128, 3, 24)])
def test_long_runs_of_large_blocks(dim, heads, size, tokens):
    """Runs that one warp does not hold: new blocks, blocks that go on with larger values, gaps, runs that come again."""
    rng = np.random.default_rng(dim + size)
    blocks = 6
    pad = lambda slots: slots + [-1] * max(0, tokens - len(slots))
    whole = lambda block, first, last, step=1: list(range(block * size + first, block * size + last, step))
    cache = scales = None
    for i, slots in enumerate((whole(0, 0, size - 2) + whole(3, 0, size // 2) + whole(1, 1, 9),
                               whole(3, size // 2, size) + whole(1, 9, size, 2) + whole(0, size - 2, size) + whole(4, 0, 1),
                               whole(2, 0, size - 5) + whole(5, 3, size) + whole(2, size - 5, size) + whole(4, 1, 14),
                               [-1] + whole(1, 10, size, 3) + [-1, -1] + whole(5, 0, size))):
        rows = [r * 2.0**i for r in _rows(rng, max(len(slots), tokens), heads, dim, "bf16")]
        cache, scales = _append(rng, rows, pad(slots), "int8" if size % 3 else "e4m3", blocks, size, scales=scales, cache=cache)


@pytest.mark.parametrize("kind", ["e4m3", "int8"])
def test_a_block_that_fills_token_by_token(kind):
    """Magnitudes grow and fall: the scale follows the largest, older rows are re-rounded."""
    rng = np.random.default_rng(1)
    blocks, size, heads, dim = 3, 8, 2, 64
    caches = scales = None
    for step in range(2 * size):
        rows = [r * 2.0 ** float(rng.integers(-6, 7)) for r in _rows(rng, 1, heads, dim, "bf16")]
        slot = [(1 if step < size else 2) * size + step % size]
        caches, scales = _append(rng, rows, slot, kind, blocks, size, scales=scales, cache=caches)


def test_a_new_block_forgets_its_last_owner():
    import torch

    rng = np.random.default_rng(2)
    scales = [torch.full((2, 1), 2.0**40).cuda() for _ in range(2)]
    _, scales = _append(rng, _rows(rng, 1, 1, 64, "bf16"), [16], "int8", 2, 16, scales=scales)
    assert scales[0][1].item() < 2.0**40 and scales[0][0].item() == 2.0**40


@pytest.mark.parametrize("bad", [0.0, -1.0, float("nan"), float("inf")])
def test_scales_that_are_no_scales_count_as_none(bad):
    import torch

    rng = np.random.default_rng(3)
    scales = [torch.full((2, 2), bad).cuda() for _ in range(2)]
    import radeon_kernels as rk

    caches = [_random_cache(rng, (2, 8, 2, 64), "e4m3") for _ in range(2)]
    rows = _rows(rng, 2, 2, 64, "fp16")
    rk.paged_cache_append_8bit(*rows, *caches, *scales, torch.tensor([3, 4], device="cuda"))
    for i in range(2):
        want, want_scales, _ = ref.append(rows[i].double().cpu().numpy(), np.zeros((2, 8, 2, 64)), np.zeros((2, 2)),
                                          np.array([3, 4]), "e4m3")
        np.testing.assert_array_equal(_values(caches[i])[0, :5], want[0, :5])  # kept rows stand for zeros
        np.testing.assert_array_equal(scales[i][0].double().cpu().numpy(), want_scales[0])


@pytest.mark.parametrize("tokens", [6, 2100], ids=["scan", "claims"])
def test_repeated_slots_and_blocks_are_refused(tokens):
    """The first run of a block is stored; the others are skipped and reported."""
    rng = np.random.default_rng(4)
    size, blocks = 16, 300
    tail = [-1] * (tokens - 6)
    for slots in ([5, 5, 6, 40, 41, -1], [5, 40, 6, 41, 7, 8], [3, 2, 1, 0, 17, 16], [20, -1, 21, 22, 4, 5],
                  [7, 8, 9, 10, 11, 7]):
        _append(rng, _rows(rng, tokens, 2, 64, "bf16"), slots + tail, "int8", blocks, size)


def test_many_runs_of_one_block():
    """Each of thousands of tokens starts a run of the same block; one comes back to it much later."""
    rng = np.random.default_rng(8)
    _append(rng, _rows(rng, 2400, 2, 64, "bf16"), [37] * 2400, "int8", 4, 16)
    _append(rng, _rows(rng, 2400, 2, 64, "bf16"), [37] + [-1] * 2380 + [38, 39] + [-1] * 16 + [5], "e4m3", 4, 16)


@pytest.mark.parametrize("tokens", [5, 2500], ids=["scan", "claims"])
def test_slots_outside_the_cache(tokens):
    rng = np.random.default_rng(5)
    slots = [-1, 2, 8 * 16, 17, 2**40] + [-3] * (tokens - 5)
    _append(rng, _rows(rng, tokens, 1, 128, "fp16"), slots, "e4m3", 8, 16)
    _append(rng, _rows(rng, tokens, 1, 128, "fp16"), [-1] * tokens, "e4m3", 8, 16)


def test_gaps_within_a_block():
    """Ascending slots with holes: rows between the new ones count as kept."""
    rng = np.random.default_rng(6)
    for slots in ([19, 22, 23, 29, 35], [16, 20, 31, 32], [18, 31, 33]):
        _append(rng, _rows(rng, len(slots), 2, 128, "bf16", spread=2.0), slots, "e4m3", 4, 16)


def test_append_of_nothing():
    import torch

    import radeon_kernels as rk

    caches = [torch.zeros((2, 8, 2, 64), dtype=torch.int8, device="cuda") for _ in range(2)]
    scales = [torch.zeros((2, 2), device="cuda") for _ in range(2)]
    rows = torch.empty((0, 2, 64), dtype=torch.float16, device="cuda")
    rk.paged_cache_append_8bit(rows, rows, *caches, *scales, torch.empty(0, dtype=torch.int64, device="cuda"))
    assert not caches[0].any() and not scales[0].any()


@pytest.mark.parametrize("kind", ["e4m3", "int8"])
@pytest.mark.parametrize("dtype", ["bf16", "fp16"])
def test_extreme_values(dtype, kind):
    """Zeros, subnormals, the largest values, infinities and NaN: only finite values set a scale."""
    import torch

    import radeon_kernels as rk

    finfo = torch.finfo(_torch_dtype(dtype))
    rows = torch.zeros((6, 1, 64), dtype=_torch_dtype(dtype))
    rows[1, 0, :4] = torch.tensor([finfo.smallest_normal, -finfo.smallest_normal, finfo.smallest_normal / 2, 0.0])
    rows[2, 0, :4] = torch.tensor([finfo.max, -finfo.max, 1.0, finfo.tiny])
    rows[3, 0, :4] = torch.tensor([float("inf"), -float("inf"), 3.0, float("nan")])
    rows[4, 0, :] = float("nan")
    rows[5, 0, :] = float("inf")
    rows = rows.cuda()
    for t in range(6):
        cache = [torch.zeros((1, 4, 1, 64), device="cuda").to(_torch_dtype(kind)) for _ in range(2)]
        scales = [torch.zeros((1, 1), device="cuda") for _ in range(2)]
        rk.paged_cache_append_8bit(rows[t : t + 1], rows[t : t + 1], *cache, *scales, torch.tensor([0], device="cuda"))
        want, want_scales, _ = ref.append(rows[t : t + 1].double().cpu().numpy(), np.zeros((1, 4, 1, 64)), np.zeros((1, 1)),
                                          np.array([0]), kind)
        np.testing.assert_array_equal(scales[0].double().cpu().numpy(), want_scales)
        np.testing.assert_array_equal(_values(cache[0]), want)


@pytest.mark.parametrize("layout", ["joint", "misaligned", "heads-first", "last-strided"])
def test_append_of_strided_rows(layout):
    import torch

    rng = np.random.default_rng(7)
    tokens, heads, dim = 9, 2, 64
    if layout == "joint":
        joint = torch.randn((tokens, 8, dim), device="cuda").bfloat16()
        rows = [joint[:, 4:6], joint[:, 6:]]
    elif layout == "misaligned":
        flat = torch.randn(2 * tokens * heads * dim + 3, device="cuda").bfloat16()
        n = tokens * heads * dim
        rows = [flat[1 : 1 + n].view(tokens, heads, dim), flat[3 + n :].view(tokens, heads, dim)]
    elif layout == "heads-first":
        rows = [torch.randn((heads, tokens, dim), device="cuda").bfloat16().transpose(0, 1) for _ in range(2)]
    else:
        rows = [torch.randn((tokens, heads, 2 * dim), device="cuda").bfloat16()[..., ::2] for _ in range(2)]
    _append(rng, rows, _prefill_slots(rng, 6, 8, [tokens]), "e4m3", 6, 8)


@pytest.mark.parametrize("tokens", [4, 2304], ids=["scan", "claims"])
def test_append_in_a_replayed_graph(tokens):
    import torch

    import radeon_kernels as rk

    rng = np.random.default_rng(8)
    size, blocks, heads, dim = 16, 200, 2, 64
    rows = _rows(rng, tokens, heads, dim, "bf16")
    caches = [_random_cache(rng, (blocks, size, heads, dim), "e4m3") for _ in range(2)]
    scales = [torch.full((blocks, heads), 2.0**-7).cuda() for _ in range(2)]
    slot_mapping = torch.full((tokens,), -1, dtype=torch.int64, device="cuda")
    rk.paged_cache_append_8bit(*rows, *caches, *scales, slot_mapping)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        rk.paged_cache_append_8bit(*rows, *caches, *scales, slot_mapping)
    for seed in (1, 2):
        slots = _prefill_slots(np.random.default_rng(seed), blocks, size, [tokens])
        slot_mapping.copy_(torch.tensor(slots))
        before = [_values(c) for c in caches], [s.double().cpu().numpy() for s in scales]
        graph.replay()
        for i in range(2):
            want, want_scales, _ = ref.append(rows[i].double().cpu().numpy(), before[0][i], before[1][i], np.array(slots), "e4m3")
            np.testing.assert_array_equal(scales[i].double().cpu().numpy(), want_scales)
            np.testing.assert_array_equal(_values(caches[i]), want)
    assert device_status() == _native.RK_OK


# --------------------------------------------------------------------------- attention
class Problem:
    def __init__(self, lengths, query_heads, kv_heads, dim, size, dtype="bf16", kind="e4m3", index="int32", seed=0,
                 spread=0.3, extra=1, query_scale=1.0):
        import torch

        rng = np.random.default_rng(seed)
        self.rng, self.dtype, self.kind, self.size = rng, dtype, kind, size
        batch = len(lengths)
        need = [-(-max(n, 0) // size) for n in lengths]
        width = max(1, max(need)) + extra
        pool = sum(need) + 3
        order = rng.permutation(pool)
        tables, at = np.full((batch, width), -1), 0
        for b, n in enumerate(need):
            tables[b, :n] = order[at : at + n]
            at += n
        self.index = {"int32": torch.int32, "int64": torch.int64}[index]
        self.tables = torch.tensor(tables).to(self.index).cuda()
        self.lengths = torch.tensor(lengths).to(self.index).cuda()
        self.query = torch.from_numpy(rng.normal(size=(batch, query_heads, dim)) * query_scale).to(_torch_dtype(dtype)).cuda()
        self.caches = [_random_cache(rng, (pool, size, kv_heads, dim), kind) for _ in range(2)]
        self.scales = [torch.from_numpy((np.exp(spread * rng.normal(size=(pool, kv_heads))) * 4 / ref.LARGEST[kind])
                                        .astype(np.float32)).cuda() for _ in range(2)]

    def run(self, scale=None):
        import radeon_kernels as rk

        return rk.paged_attention_decode_8bit(self.query, *self.caches, *self.scales, self.tables, self.lengths, scale)

    def check(self, out, scale=None):
        want, bound = ref.attention(
            self.query.double().cpu().numpy(), *[_values(c) for c in self.caches],
            *[s.double().cpu().numpy() for s in self.scales], self.tables.cpu().numpy(), self.lengths.cpu().numpy(),
            scale or ref.default_scale(self.query.shape[2]), self.dtype)
        got = out.double().cpu().numpy()
        np.testing.assert_array_equal(np.isnan(got), np.isnan(want))
        worst = np.nanmax(np.abs(got - want) - bound) if np.isfinite(want).any() else -1.0
        assert worst <= 0, worst


@pytest.mark.parametrize("kind", ["e4m3", "int8"])
@pytest.mark.parametrize("dtype", ["bf16", "fp16"])
@pytest.mark.parametrize(
    "lengths, query_heads, kv_heads, dim, size",
    [
        ([1], 1, 1, 64, 16),
        ([1, 2, 15, 16, 17, 63, 64, 65], 8, 2, 128, 16),
        ([1003], 32, 8, 128, 16),
        ([5, 0, 130], 4, 4, 64, 8),          # an empty sequence; a KV head per query head
        ([77, 400], 5, 1, 128, 24),          # a group of 5; blocks that end inside a tile
        ([90, 3], 16, 1, 128, 32),           # two column tiles
        ([129], 28, 2, 64, 48),              # a group of 14
        ([200, 31], 9, 1, 256, 7),           # two head tiles at head_dim 256, odd blocks
        ([64, 640], 40, 2, 128, 1),          # a group of 20: two head tiles of up to 16
        ([50] * 70, 4, 1, 64, 64),
        ([2000, 1, 700], 8, 1, 256, 128),
        ([1] * 300, 2, 2, 64, 16),           # more sequences than CTA threads
        ([1500] + [3] * 40, 16, 8, 64, 1024),
    ],
)
def test_attention_matches_its_definition(lengths, query_heads, kv_heads, dim, size, dtype, kind):
    import radeon_kernels as rk

    p = Problem(lengths, query_heads, kv_heads, dim, size, dtype, kind, "int32" if len(lengths) % 2 else "int64",
                seed=sum(lengths))
    out = p.run()
    assert rk.get_last_dispatch()["selected"] == "native/paged_attention_decode_8bit"
    p.check(out)
    assert device_status() == _native.RK_OK
    import torch

    assert torch.equal(out.view(torch.int16), p.run().view(torch.int16))  # the same bits every time


@pytest.mark.parametrize(
    "lengths,query_heads,kv_heads,dim,size",
    [([20000], 4, 1, 128, 16), ([12000], 8, 1, 256, 64), ([9000, 3, 14000], 6, 2, 64, 24), ([40000, 40000], 1, 1, 64, 128),
     ([30001], 17, 1, 64, 32), ([6000, 6000, 6000], 16, 1, 128, 8)])
def test_sequences_that_fill_the_gpu(lengths, query_heads, kv_heads, dim, size):
    """A head of a sequence is spread over all SMs; whichever comes last, the result is the same."""
    import torch

    p = Problem(lengths, query_heads, kv_heads, dim, size, "bf16", "int8", seed=sum(lengths))
    out = p.run()
    p.check(out)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        captured = [p.run() for _ in range(3)]
    for _ in range(5):
        for c in captured:
            c.zero_()
        graph.replay()
        assert all(torch.equal(c, out) for c in captured)


@pytest.mark.parametrize("scale", [1e-4, 0.5, 3])
def test_attention_scale(scale):
    p = Problem([100, 700], 8, 2, 128, 16, seed=3)
    p.check(p.run(scale), scale)


@pytest.mark.parametrize("size", [8, 16, 24, 64])
def test_only_live_positions_count(size):
    """What lies behind a sequence -- NaN rows, scales that are none, tables out of range -- is not read."""
    import torch

    lengths = [1, 37, 100, 0]
    p = Problem(lengths, 8, 2, 128, size, "fp16", "e4m3", seed=size)
    nan = torch.tensor(0x7F, dtype=torch.uint8, device="cuda")
    for b, n in enumerate(lengths):
        used = -(-n // size)
        if n % size:
            block = int(p.tables[b, used - 1])
            for cache in p.caches:
                cache.view(torch.uint8)[block, n % size :] = nan
        p.tables[b, used:] = 2**30  # never looked up
    unused = set(range(p.caches[0].shape[0])) - set(int(x) for b, n in enumerate(lengths) for x in p.tables[b, : -(-n // size)])
    for block in unused:
        p.caches[0].view(torch.uint8)[block] = nan
        p.scales[0][block] = p.scales[1][block] = float("nan")
    out = p.run()
    for cache in p.caches:  # the reference sees zeros there
        raw = cache.view(torch.uint8)
        raw[raw == nan] = 0
    p.check(out)
    assert device_status() == _native.RK_OK


def test_bad_pages_are_skipped_and_reported():
    for bad in (-1, -(2**31), 10**6, 2**31 - 1):
        p = Problem([100, 40, 16], 8, 2, 128, 16, seed=9)
        p.tables[0, 2] = bad
        p.tables[2, 0] = bad  # all of a sequence
        p.check(p.run())
        assert device_status() == _native.RK_ERR_INVALID_ARGUMENT
    p = Problem([100, 40], 8, 2, 128, 16, index="int64", seed=9)
    p.tables[1, 1] = 2**40
    p.check(p.run())
    assert device_status() == _native.RK_ERR_INVALID_ARGUMENT


def test_lengths_beyond_the_table_and_negative():
    p = Problem([64, 64, 64], 4, 2, 64, 16, extra=0, seed=4)
    p.lengths[1], p.lengths[2] = 10**6, -5
    p.check(p.run())
    assert device_status() == _native.RK_OK


@pytest.mark.parametrize("kind", ["e4m3", "int8"])
def test_scales_far_apart(kind):
    """Blocks whose scales differ by 2^30, the largest masked out by their scores or not; zero scales."""
    for case in range(4):
        p = Problem([200, 130], 8, 2, 128, 16, "fp16", kind, seed=20 + case)
        with np.errstate(all="ignore"):
            for b in range(2):
                for j in range(8):
                    block = int(p.tables[b, j])
                    if case == 0:
                        p.scales[1][block] = 2.0 ** (-5 * j) / 64
                    elif case == 1:
                        p.scales[1][block] = 2.0 ** (-5 * (7 - j)) / 64
                    elif case == 2:
                        p.scales[j % 2][block] = 0.0
                    else:
                        p.scales[0][block] *= 2.0 ** (j - 4)
        p.check(p.run())


@pytest.mark.parametrize("batch, kv_heads, dim", [(33, 3, 256), (1000, 2, 64), (5000, 1, 128)])
def test_thousands_of_short_sequences(batch, kv_heads, dim):
    p = Problem([(7 * b) % 4 if b % 11 else 40 for b in range(batch)], 2 * kv_heads, kv_heads, dim, 8, "fp16", "int8", seed=batch)
    p.check(p.run())


@pytest.mark.parametrize("tokens", [255, 256, 257, 512, 513])
def test_append_at_the_edges_of_its_forms(tokens):
    rng = np.random.default_rng(tokens)
    for lengths in ([tokens], [1] * tokens, [tokens - 200, 90, 110]):
        blocks = sum(-(-n // 16) + 1 for n in lengths) + 1
        slots = _prefill_slots(rng, blocks, 16, lengths)
        _append(rng, _rows(rng, tokens, 1, 64, "fp16"), slots, "e4m3", blocks, 16)


@pytest.mark.parametrize("exponent", [-126, -120, 120, 127])
def test_value_scales_at_the_ends_of_fp32(exponent):
    p = Problem([1, 45, 300], 8, 2, 128, 16, "bf16", "int8", seed=31)
    p.caches[1].clamp_(-1, 1)  # the output stays finite
    p.scales[1].fill_(2.0**exponent)
    p.check(p.run())


def test_all_value_scales_zero():
    import torch

    p = Problem([70], 4, 1, 64, 16, seed=2)
    p.scales[1].zero_()
    out = p.run()
    assert torch.equal(out, torch.zeros_like(out))


@pytest.mark.parametrize("dtype", ["bf16", "fp16"])
def test_queries_of_any_magnitude(dtype):
    for query_scale in (1e-30, 1e-3, 30.0, 1e4) if dtype == "bf16" else (1e-6, 30.0, 1e3):
        p = Problem([90, 300], 8, 2, 128, 16, dtype, seed=5, query_scale=query_scale)
        if query_scale > 1e3:
            for s in p.scales[:1]:
                s *= 1e-4
        p.query[0, 1] = 0  # equal weights
        p.query[0, 2, 7] *= 300  # one component far above the others
        p.check(p.run())


def test_non_finite_queries_and_rows():
    import torch

    p = Problem([50, 50], 4, 2, 64, 16, seed=6)
    p.query[0, 1, 3] = float("nan")
    out = p.run()
    assert torch.isnan(out[0, 1]).all() and torch.isfinite(out[0, 0]).all() and torch.isfinite(out[1]).all()
    # A NaN key reaches every head that reads it, a NaN value only its dimension.
    p = Problem([50, 50], 4, 2, 64, 16, seed=6)
    p.caches[0].view(torch.uint8)[int(p.tables[0, 1]), 3, 0, 5] = 0x7F
    p.caches[1].view(torch.uint8)[int(p.tables[1, 0]), 2, 1, 9] = 0x7F
    out = p.run()
    assert torch.isnan(out[0, :2]).all() and torch.isfinite(out[0, 2:]).all()
    assert torch.isnan(out[1, 2:, 9]).all()
    assert torch.isfinite(out[1, :2]).all() and torch.isfinite(out[1, 2:, :9]).all() and torch.isfinite(out[1, 2:, 10:]).all()


def test_a_peaked_softmax():
    """Scores far apart: one position takes all the weight, wherever it lies."""
    for at in (0, 63, 64, 1023, 1999):
        p = Problem([2000], 8, 1, 128, 16, "fp16", "int8", seed=at)
        block, row = int(p.tables[0, at // 16]), at % 16
        import torch

        p.caches[0][block, row, 0] = torch.sign(p.query[0, 0].float()).to(torch.int8) * 127
        p.check(p.run(2.0), 2.0)


@pytest.mark.parametrize("kind", ["e4m3", "int8"])
def test_offsets_past_32_bits(kind):
    """A cache of more than 2^31 elements, read at its end."""
    import torch

    import radeon_kernels as rk

    blocks, size, heads, dim = 17000, 128, 8, 128  # 2.2e9 elements each
    caches = [torch.zeros((blocks, size, heads, dim), dtype=_torch_dtype(kind), device="cuda") for _ in range(2)]
    scales = [torch.ones((blocks, heads), device="cuda") / 16 for _ in range(2)]
    tokens = 150
    rng = np.random.default_rng(1)
    rows = _rows(rng, tokens, heads, dim, "bf16", spread=0.0)
    ids = [blocks - 1, blocks - 3]
    slots = torch.tensor([ids[i // size] * size + i % size for i in range(tokens)], device="cuda")
    rk.paged_cache_append_8bit(*rows, *caches, *scales, slots)
    table = torch.tensor([ids], device="cuda")
    query = torch.from_numpy(rng.normal(size=(1, 16, dim))).bfloat16().cuda()
    out = rk.paged_attention_decode_8bit(query, *caches, *scales, table, torch.tensor([tokens], device="cuda"))
    few = torch.tensor([1, 0], device="cuda")  # the same blocks, as a small cache
    raw = [c.view(torch.uint8)[ids].view(c.dtype) for c in caches]
    want, bound = ref.attention(query.double().cpu().numpy(), *[_values(c) for c in raw],
                                *[s[ids].double().cpu().numpy() for s in scales], np.array([[0, 1]]), np.array([tokens]),
                                ref.default_scale(dim), "bf16")
    del few
    assert (np.abs(out.double().cpu().numpy() - want) <= bound).all()
    stored = _values(raw[0]) * scales[0][ids].double().cpu().numpy()[:, None, :, None]
    x = rows[0].double().cpu().numpy()
    # Half a step: 2^-4 of the value in e4m3, half a scale in int8 (and e4m3's smallest steps).
    top = scales[0][ids].double().cpu().numpy()[:, None, :, None] * np.ones_like(stored)
    half = (top / 2 if kind == "int8" else np.maximum(np.abs(stored) * 2.0**-4 * 1.07, top * 2.0**-10)).reshape(-1, heads, dim)
    assert (np.abs(stored.reshape(-1, heads, dim)[:tokens] - x) <= half[:tokens]).all()


def test_misaligned_query_and_refused_caches():
    import torch

    import radeon_kernels as rk

    p = Problem([70], 8, 2, 128, 16, seed=1)
    flat = torch.empty(p.query.numel() + 1, dtype=p.query.dtype, device="cuda")
    query = flat[1:].view(p.query.shape)
    query.copy_(p.query)
    aligned = p.run()
    p.query = query
    assert torch.equal(aligned, p.run())
    shape = p.caches[0].shape
    raw = torch.zeros(p.caches[0].numel() + 1, dtype=torch.int8, device="cuda")[1:].view(shape)
    with pytest.raises(RuntimeError, match="16-byte boundary"):
        rk.paged_attention_decode_8bit(p.query, raw, raw, *p.scales, p.tables, p.lengths)


def test_attention_on_two_streams_and_in_two_graphs():
    """Calls that overlap have workspaces of their own."""
    import torch

    a, b = Problem([3000, 70], 16, 2, 128, 16, seed=1), Problem([900] * 9, 8, 8, 64, 32, "fp16", "int8", seed=2)
    want = [a.run(), b.run()]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in range(2)]
    outs = [[], []]
    for _ in range(10):
        for i, p in enumerate((a, b)):
            with torch.cuda.stream(streams[i]):
                outs[i].append(p.run())
    torch.cuda.synchronize()
    for i in range(2):
        assert all(torch.equal(o, want[i]) for o in outs[i])
    graphs, results = [], []
    for p in (a, b):
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            results.append(p.run())
        graphs.append(graph)
    for _ in range(5):
        for i in range(2):
            with torch.cuda.stream(streams[i]):
                graphs[i].replay()
    torch.cuda.synchronize()
    assert torch.equal(results[0], want[0]) and torch.equal(results[1], want[1])
    # A replay follows its inputs, lengths among them.
    a.lengths.copy_(torch.tensor([17, 70]))
    a.query.neg_()
    graphs[0].replay()
    a.check(results[0])


# ------------------------------------------------------------------- a run of all four
@pytest.mark.parametrize("graph", [False, True], ids=["eager", "graph"])
@pytest.mark.parametrize("kind", ["e4m3", "int8"])
def test_a_prefill_and_decode_loop(kind, graph):
    """Prompts are placed, rotated, stored and read back over ten decode steps; everything is
    followed by the definitions from the same inputs, the attention within its bounds."""
    import torch

    import radeon_kernels as rk

    batch, hq, hk, dim, size, width = 5, 8, 2, 64, 8, 12
    pool = batch * width + 5
    gen = torch.Generator(device="cuda").manual_seed(3)
    rng = np.random.default_rng(3)
    free = torch.randperm(pool, generator=gen, device="cuda").to(torch.int32)
    tables = torch.full((batch, width), -1, dtype=torch.int32, device="cuda")
    lengths = torch.zeros(batch, dtype=torch.int32, device="cuda")
    caches = [_random_cache(rng, (pool, size, hk, dim), kind) for _ in range(2)]
    scales = [torch.full((pool, hk), 7.0, device="cuda") for _ in range(2)]
    frequencies = rk.rotary_frequencies(dim, scaling="yarn", factor=4.0, original_length=64)
    new = torch.tensor([13, 0, 1, 40, 8], dtype=torch.int32, device="cuda")
    ones = torch.ones(batch, dtype=torch.int32, device="cuda")

    def step(joint, tables, lengths, new, free, tokens):
        slots, positions, lengths, used = rk.paged_slots(tables, lengths, new, free, num_tokens=tokens, block_size=size)
        query, key = rk.rotary_embedding(joint[:, :hq], joint[:, hq : hq + hk], positions, frequencies, amplitude=1.1)
        rk.paged_cache_append_8bit(key, joint[:, hq + hk :], *caches, *scales, slots)
        return slots, positions, lengths, used, query, key

    def follow(joint, before, new, free, tokens, got):
        tables0, lengths0, caches0, scales0 = before
        slots, positions, lengths, used, query, key = got
        want = ref.slots(tables0, lengths0, new.cpu().numpy(), free.tolist(), tokens, size)
        np.testing.assert_array_equal(slots.cpu().numpy(), want[0])
        np.testing.assert_array_equal(tables.cpu().numpy(), want[4])
        np.testing.assert_array_equal(lengths.cpu().numpy(), want[2])
        turned, slack = ref.rotary(joint[:, :hq].double().cpu().numpy(), want[1], frequencies.cpu().numpy(), False, 1.1)
        assert (np.abs(query.double().cpu().numpy() - turned) <= slack * 1.01 + ref.rounding(turned, "bf16")).all()
        for i, rows in enumerate((key, joint[:, hq + hk :])):
            stored, now, _ = ref.append(rows.double().cpu().numpy(), caches0[i], scales0[i], want[0], kind)
            np.testing.assert_array_equal(_values(caches[i]), stored)
            np.testing.assert_array_equal(scales[i].double().cpu().numpy(), now)

    def snapshot():
        return (tables.cpu().numpy(), lengths.cpu().numpy(), [_values(c) for c in caches],
                [s.double().cpu().numpy() for s in scales])

    tokens = 64  # two tokens of padding
    joint = torch.randn((tokens, hq + 2 * hk, dim), generator=gen, device="cuda").bfloat16()
    before = snapshot()
    got = step(joint, tables, lengths, new, free, tokens)
    follow(joint, before, new, free, tokens, got)
    lengths, free = got[2], free[int(got[3]) :].clone()

    def decode(joint):
        out = step(joint, tables, lengths, ones, free, batch)
        return (*out, rk.paged_attention_decode_8bit(out[4], *caches, *scales, tables, out[2]))

    joint = torch.randn((batch, hq + 2 * hk, dim), generator=gen, device="cuda").bfloat16()
    replay = None
    if graph:
        keep = [t.clone() for t in (tables, *caches, *scales)]
        replay = torch.cuda.CUDAGraph()
        with torch.cuda.graph(replay):
            captured = decode(joint)
        for t, k in zip((tables, *caches, *scales), keep):
            t.copy_(k)
    for _ in range(10):
        joint.copy_(torch.randn(joint.shape, generator=gen, device="cuda"))
        before = snapshot()
        if replay is None:
            got = decode(joint)
        else:
            replay.replay()
            got = tuple(t.clone() for t in captured)
        follow(joint, before, ones, free, batch, got[:6])
        want, bound = ref.attention(got[4].double().cpu().numpy(), *[_values(c) for c in caches],
                                    *[s.double().cpu().numpy() for s in scales], tables.cpu().numpy(),
                                    got[2].cpu().numpy(), ref.default_scale(dim), "bf16")
        assert (np.abs(got[6].double().cpu().numpy() - want) <= bound).all()
        used = int(got[3])
        lengths.copy_(got[2])
        free.copy_(torch.roll(free, -used))
    assert device_status() == _native.RK_OK


# --------------------------------------------------------------------- many divisions of work
def _plain64(p):
    """The definition in float64 on the GPU, sequence by sequence, and the bound of ref.attention."""
    import torch

    dim, heads = p.query.shape[2], p.caches[0].shape[2]
    outs, bounds = [], []
    for b, n in enumerate(p.lengths.tolist()):
        blocks = p.tables[b, : -(-n // p.size)].long()
        k, v = [(c.view(torch.uint8)[blocks].view(c.dtype).double() * s[blocks].double()[:, None, :, None])
                .reshape(-1, heads, dim)[:n] for c, s in zip(p.caches, p.scales)]
        q = p.query[b].double().view(heads, -1, dim)
        s = torch.einsum("hgd,thd->hgt", q, k) * dim**-0.5
        w = torch.softmax(s, -1)
        outs.append(torch.einsum("hgt,thd->hgd", w, v).reshape(-1, dim))
        a = torch.einsum("hgt,thd->hgd", w, v.abs())
        near = (torch.einsum("hgd,thd->hgt", q.abs(), k.abs()) * dim**-0.5).amax(-1, keepdim=True)
        down = (k.abs().sum(-1).amax(0) * dim**-0.5 * 2.0**-25)[:, None, None] * q.abs().amax(-1, keepdim=True)
        bound = a * (2.0**-10 + 2 * (near * (dim + 16) * 2.0**-24 + 2.0**-18 + down))
        bound = bound + n * 2.0**-25 * w.amax(-1, keepdim=True) * v.abs().amax()
        bounds.append(bound.reshape(-1, dim))
    out, bound = torch.stack(outs), torch.stack(bounds)
    return out, bound + out.abs() * ref.HALF_STEP[p.dtype] * (1 + 2.0**-10) + ref.TINY[p.dtype]


@pytest.mark.parametrize("seed", range(24))
def test_attention_of_many_lengths(seed):
    """Random batches: every way in which the warps' shares can cut the sequences and heads.  Three
    calls back to back, the middle one of another batch: workspaces are handed on uncleared."""
    import torch

    rng = np.random.default_rng(100 + seed)
    dim = int(rng.choice([64, 128, 256]))
    kv_heads, group = int(rng.choice([1, 2, 3, 8])), int(rng.choice([1, 4, 5, 8, 12]))
    batch = int(rng.choice([1, 2, 5, 17, 70, 150]))
    longest = int(rng.choice([40, 500, 3000, 9000]) if batch < 50 else rng.choice([40, 900]))
    lengths = np.maximum(1, (longest * rng.random(batch) ** 3)).astype(int).tolist()
    make = lambda n, s: Problem(n, kv_heads * group, kv_heads, dim, int(rng.choice([8, 16, 32, 20])),  # noqa: E731
                                str(rng.choice(["bf16", "fp16"])), str(rng.choice(["e4m3", "int8"])),
                                str(rng.choice(["int32", "int64"])), seed=s)
    p, other = make(lengths, seed), make(lengths[::-1][: max(1, batch // 2)], seed + 1000)
    outs = [p.run(), other.run(), p.run(), p.run()]
    want, bound = _plain64(p)
    for out in (outs[0], outs[2], outs[3]):
        assert ((out.double() - want).abs() <= bound).all()
        assert torch.equal(out, outs[0])
    want, bound = _plain64(other)
    assert ((outs[1].double() - want).abs() <= bound).all()


def test_refusals_after_calls_of_the_same_kind():
    """A call that differs from a served one only in what the front-end checks is refused as ever."""
    import torch

    import radeon_kernels as rk

    p = Problem([70, 3], 8, 2, 128, 16, seed=1)
    p.run()
    p.run()
    args = [p.query, *p.caches, *p.scales, p.tables, p.lengths]
    for at, bad, error in (
        (0, p.query[:1], ValueError), (0, p.query.cpu(), ValueError), (0, p.query[None], ValueError),
        (2, p.caches[1].view(torch.uint8), TypeError), (3, p.scales[0].double(), TypeError), (4, p.scales[1][:-1], ValueError),
        (5, p.tables.long(), TypeError), (5, p.tables.t().contiguous().t(), ValueError), (6, [3, 4], TypeError),
        (0, p.query.clone().requires_grad_(True), ValueError), (0, p.query.transpose(0, 1).contiguous().transpose(0, 1), ValueError),
    ):
        with pytest.raises(error, match="paged_attention_decode_8bit"):
            rk.paged_attention_decode_8bit(*args[:at], bad, *args[at + 1 :])
    for scale, error in ((0.0, ValueError), (float("inf"), ValueError), (-1.0, ValueError), (True, TypeError), ("a", TypeError)):
        with pytest.raises(error, match="paged_attention_decode_8bit scale"):
            rk.paged_attention_decode_8bit(*args, scale)
    rows = torch.zeros((2, 2, 128), dtype=torch.bfloat16, device="cuda")
    slots = torch.tensor([-1, -1], device="cuda")
    rk.paged_cache_append_8bit(rows, rows, *p.caches, *p.scales, slots)
    for bad in ((rows, rows[:1]), (rows.half(), rows), (rows[..., :64], rows[..., :64])):
        with pytest.raises((ValueError, TypeError), match="paged_cache_append_8bit"):
            rk.paged_cache_append_8bit(*bad, *p.caches, *p.scales, slots)
    with pytest.raises(ValueError, match="one slot per token"):
        rk.paged_cache_append_8bit(rows, rows, *p.caches, *p.scales, slots[:1])
    lengths = torch.ones(2, dtype=torch.int32, device="cuda")
    tables = torch.zeros((2, 3), dtype=torch.int32, device="cuda")
    rk.paged_slots(tables, lengths, lengths, lengths, num_tokens=2, block_size=4)
    with pytest.raises(TypeError, match="same dtype"):
        rk.paged_slots(tables, lengths.long(), lengths, lengths, num_tokens=2, block_size=4)
    with pytest.raises(ValueError, match="num_tokens"):
        rk.paged_slots(tables, lengths, lengths, lengths, num_tokens=-1, block_size=4)
    with pytest.raises(TypeError, match="num_tokens"):
        rk.paged_slots(tables, lengths, lengths, lengths, num_tokens=True, block_size=4)
    frequencies, positions = rk.rotary_frequencies(128), torch.arange(2, device="cuda")
    rk.rotary_embedding(rows, rows, positions, frequencies)
    for changed, error in (
        ((rows, rows, positions[:1], frequencies), ValueError), ((rows, rows[:1], positions, frequencies), ValueError),
        ((rows, rows.half(), positions, frequencies), TypeError), ((rows, rows, positions.cpu(), frequencies), ValueError),
    ):
        with pytest.raises(error, match="rotary_embedding"):
            rk.rotary_embedding(*changed)
    with pytest.raises(TypeError, match="interleaved"):
        rk.rotary_embedding(rows, rows, positions, frequencies, interleaved=0)
    device_status()


# ------------------------------------------------------------- weights far below the largest
def _alike(codes, unit, heads, dim, kind, dtype, seed):
    """1184 sequences over the same blocks, one KV head: a range for every warp of the GPU, so that a warp
    holds all positions of a range.  Position t's score is codes[t] * unit exactly; value codes are
    whole numbers from 1 to 15.  Returns the problem of one sequence and a call for all of them."""
    import torch

    length = len(codes)
    p = Problem([length], heads, 1, dim, 32, dtype, kind, seed=seed)
    pool = p.caches[0].shape[0]
    order = p.tables[0, : -(-length // 32)].long().cpu()
    keys, values = torch.zeros((len(order) * 32, dim)), torch.zeros((len(order) * 32, dim))
    keys[:length, 0] = torch.tensor(codes).float()
    values[:length] = torch.from_numpy(p.rng.integers(1, 16, (length, dim))).float()

    def placed(x):
        out = torch.zeros((pool, 32, 1, dim))
        out[order] = x.view(-1, 32, 1, dim)
        stored = out.to(_torch_dtype(kind))
        assert torch.equal(stored.float(), out)  # the codes are values of the type
        return stored.cuda()

    p.caches = [placed(keys), placed(values)]
    p.scales = [torch.ones((pool, 1), device="cuda") for _ in range(2)]
    p.query.zero_()
    p.query[:, :, 0] = unit

    def run():
        import radeon_kernels as rk

        query, tables, lengths = (x.expand(1184, *x.shape[1:]).contiguous() for x in (p.query, p.tables, p.lengths))
        out = rk.paged_attention_decode_8bit(query, *p.caches, *p.scales, tables, lengths, 1.0)
        assert torch.equal(out.view(torch.int16), out[:1].expand_as(out).contiguous().view(torch.int16))
        return out[:1].double().cpu().numpy()

    return p, run


def _definition(p):
    return ref.attention(p.query.double().cpu().numpy(), *[_values(c) for c in p.caches],
                         *[s.double().cpu().numpy() for s in p.scales], p.tables.cpu().numpy(), p.lengths.cpu().numpy(),
                         1.0, p.dtype)


def _tight(codes, unit, p):
    """The attention's bound for `_alike`: the terms of ref.attention, but each weight of V is off by half
    a step of fp16 (2^-11 of itself) or by 2^-36 of the largest, whichever is more; a score is one
    product, off by 2^-24 of itself, and so is its distance to the maximum."""
    import torch

    n = len(codes)
    blocks = p.tables[0, : -(-n // 32)].long()
    v = p.caches[1].view(torch.uint8)[blocks].view(p.caches[1].dtype).float().reshape(-1, p.query.shape[2])[:n].double().cpu().numpy()
    s = np.array(codes) * unit
    w = np.exp(s - s.max())
    w /= w.sum()
    out = w @ v
    bound = out * (2.0**-11 * (1 + 2.0**-10) + 2 * (3 * np.abs(s).max() * 2.0**-24 + 2.0**-18))
    return out, bound + n * 2.0**-36 * w.max() * 15 + ref.rounding(out, p.dtype)


@pytest.mark.parametrize("kind", ["e4m3", "int8"])
@pytest.mark.parametrize("dtype", ["bf16", "fp16"])
@pytest.mark.parametrize("dim, heads", [(64, 4), (128, 8), (128, 16), (256, 3)])
@pytest.mark.parametrize("sink", [0, 5000, 8191])
def test_weights_far_below_one_whose_value_is_zero(dim, heads, sink, dtype, kind):
    """A position that takes nearly all the weight and has no value: the others, 2^-25 to 2^-29 of it
    each, are the output."""
    import torch

    codes = np.random.default_rng(sink).integers(0, 10, 8192)
    codes[sink] = 80
    p, run = _alike(codes, 0.25, heads, dim, kind, dtype, seed=sink)
    p.caches[1].view(torch.uint8)[int(p.tables[0, sink // 32]), sink % 32] = 0
    out, bound = _tight(codes, 0.25, p)
    np.testing.assert_allclose(out, _definition(p)[0][0, 0], rtol=1e-12)
    assert (bound < out * 2.0**-6).all()  # it says something
    got = run()
    assert (np.abs(got - out) <= bound).all(), np.max(np.abs(got - out) / bound)


@pytest.mark.parametrize("kind", ["e4m3", "int8"])
@pytest.mark.parametrize("dim, heads", [(64, 4), (128, 8), (128, 16), (256, 3)])
@pytest.mark.parametrize("rise", [0, 4, 28])
def test_value_scales_of_zero_before_larger_ones(dim, heads, rise, kind):
    """Blocks whose value scale is 0 hold the largest scores, the blocks behind them have large value
    scales: weights that vanish leave a 0, those that do not count as ever."""
    for low in (-60, -30, 0):
        codes = [60] * 64 + [60 + rise] * 64 + [low] * 128
        p, run = _alike(codes, 1.0, heads, dim, kind, "bf16", seed=-low)
        p.scales[1][p.tables[0, :4].long()] = 0.0
        for scale in (2.0**4, 2.0**60, 2.0**100):
            p.scales[1][p.tables[0, 4:8].long()] = scale
            got = run()
            want, bound = _definition(p)
            assert np.isfinite(got).all(), (low, scale)
            # Exponentials below 2^-126 of the largest are 0.
            assert (np.abs(got - want) <= bound + 256 * 2.0**-126 * scale * 15).all(), (low, scale)


@pytest.mark.parametrize("query_heads, dim", [(1, 64), (3, 128), (5, 256), (13, 128), (16, 64)])
def test_joins_in_two_steps_of_every_number_of_heads(query_heads, dim):
    """One sequence over all SMs, whose parts are joined a group of CTAs at a time into the first one's:
    odd numbers of heads leave half of a warp idle; the same bits every time."""
    import torch

    p = Problem([40000 if dim < 256 else 20000], query_heads, 1, dim, 64, "fp16", "e4m3", seed=query_heads)
    out = p.run()
    want, bound = _plain64(p)
    assert ((out.double() - want).abs() <= bound).all()
    for _ in range(50):
        assert torch.equal(p.run(), out)
