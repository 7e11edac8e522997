"""How the 8-bit decode attention deals its work out to warps, by the kernel's own header on the CPU:
every unit goes to one warp, and no warp looks anything up for a sequence past the last."""

from __future__ import annotations

import ctypes
import subprocess

import numpy as np
import pytest

from conftest import PKG_ROOT, REPO

SMS, CTAS_PER_SM = 148, 2


@pytest.fixture(scope="module")
def shares(tmp_path_factory):
    library = tmp_path_factory.mktemp("shares") / "shares.so"
    subprocess.run(["g++", "-O2", "-std=c++17", "-Wall", "-Werror", "-shared", "-fPIC", f"-I{PKG_ROOT / 'csrc'}",
                    str(REPO / "tests" / "paged8_shares.cpp"), "-o", str(library)], check=True)
    lib = ctypes.CDLL(str(library))
    lib.shares_ctas.argtypes, lib.shares_ctas.restype = [ctypes.c_int64] * 3, ctypes.c_int64
    lib.shares_walks.argtypes = [ctypes.c_void_p] + [ctypes.c_int] * 4 + [ctypes.c_int64] + [ctypes.c_void_p] * 2 + [ctypes.c_int64]
    lib.shares_walks.restype = ctypes.c_int64
    return lib


def _walks(lib, lengths, kv_heads, head_groups, head_dim, room):
    """(first [warps, 2], visits [units, 5], units of each sequence) for tables that hold `room` positions."""
    unit = lib.shares_unit(head_dim)
    units = [max(1, -(-n // unit)) for n in lengths]
    ctas = lib.shares_ctas(len(lengths) * kv_heads * head_groups, -(-room // unit), SMS * CTAS_PER_SM)
    assert 1 <= ctas <= SMS * CTAS_PER_SM
    first = np.zeros((ctas * lib.shares_warps(), 2), np.int64)
    most = sum(units) * kv_heads * head_groups
    visits = np.zeros((most + 1, 5), np.int32)
    held = np.array(lengths, np.int32)
    n = lib.shares_walks(held.ctypes.data, len(lengths), kv_heads, head_groups, head_dim, ctas, first.ctypes.data,
                         visits.ctypes.data, most + 1)
    return first, visits[:n], units


# (lengths, KV heads, head groups, head_dim, positions of a table row)
SMALL = [
    ([1003], 8, 1, 128, 1008),            # 272 places: a place for every warp, some of them behind the last range
    ([1], 1, 1, 128, 32),                 # fewer places than warps
    ([1] * 512, 1, 1, 128, 16384),        # 1536 places: one or two to a warp
    ([1] * 500, 1, 1, 128, 16384),
    ([70, 0, 5], 4, 1, 64, 4096),
    ([3] * 97, 2, 2, 256, 512),
    ([40] * 70, 3, 1, 256, 2048),
    ([2000, 1, 700], 1, 1, 256, 4096),
    ([1500] + [3] * 40, 8, 1, 128, 2048),
    ([131072], 8, 1, 128, 131072),
]


@pytest.mark.parametrize("case", SMALL + [
    ([int(x) for x in np.random.default_rng(s).integers(0, 10 ** (1 + s % 4), 1 + 37 * (s % 9))], 1 + s % 8, 1 + s % 3,
     (64, 128, 256)[s % 3], 10 ** (1 + s % 4) + 16) for s in range(60)])
def test_every_unit_once_and_nothing_past_the_batch(shares, case):
    lengths, kv_heads, head_groups, head_dim, room = case
    first, visits, units = _walks(shares, *case)
    # What a warp looks up when it begins -- rows of the block tables, queries -- is the batch's.
    assert (first[first[:, 1] == 1, 0] < len(lengths)).all()
    seen = visits[:, 1:]
    assert (seen[:, 0] < len(lengths)).all()
    want = [(b, h, g, c) for b, n in enumerate(units) for h in range(kv_heads) for g in range(head_groups) for c in range(n)]
    assert len(seen) == len(want)
    assert (seen == np.array(want, np.int32)).all()  # warp by warp, in order


def test_shares_that_begin_behind_the_last_range(shares):
    """The calls above include warps that stand past the last sequence; those look nothing up."""
    for at in (0, 2):
        first, _, _ = _walks(shares, *SMALL[at])
        past = first[:, 0] >= len(SMALL[at][0])
        assert past.any() and not first[past, 1].any()
