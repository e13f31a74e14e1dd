"""Which blocks the products of ``chunk_attention`` read (``csrc/chunk_plan.h``, built for the host): those that hold a
visible token of the sequence and no others, though a row tile visits whole token tiles.  The block-table entries of blocks
in front of a sliding window may hold anything, so following one would read anywhere."""
import ctypes
import pathlib
import random
import subprocess

import numpy as np
import pytest

HERE = pathlib.Path(__file__).resolve().parent
FORMS = [(256, 64), (64, 64), (32, 128)]


@pytest.fixture(scope="module")
def lib(tmp_path_factory):
    so = tmp_path_factory.mktemp("reads") / "chunk_reads_host.so"
    subprocess.run(["g++", "-O1", "-std=c++17", "-shared", "-fPIC", "-o", str(so), str(HERE / "chunk_reads_host.cpp")], check=True)
    return ctypes.CDLL(str(so))


def reads_of(lib, shape, n, length):
    pointer = lambda x: x.ctypes.data_as(ctypes.c_void_p)  # noqa: E731
    s, room = np.array(shape, np.int32), 1 << 16
    got = np.zeros((room, 4), np.int32)
    count = lib.host_reads(pointer(s), n, length, pointer(got), room)
    assert count <= room
    return got[:count]


def seen_by(shape, n, length, r=None):
    """Tokens that a row of row tile r (of any, if None) sees."""
    rows, _, group, _, causal, window, first = shape
    seen = np.zeros(length, bool)
    tokens = range(n) if r is None else range(r * rows // group, min(((r + 1) * rows - 1) // group, n - 1) + 1)
    for i in tokens:
        end = max(0, length - n + i + 1) if causal else length
        seen[max(0, end - window) if window else 0:end] = True
        if window:
            seen[:min(first, end)] = True
    return seen


def check(lib, shape, n, length):
    got = reads_of(lib, shape, n, length)
    assert ((got[:, 2] >= 0) & (got[:, 2] < max(length, 1))).all()
    anyone = seen_by(shape, n, length)
    for block in (16, 32, 128):
        visible = np.unique(np.flatnonzero(anyone) // block)
        assert np.isin(got[:, 2] // block, visible).all(), (shape, n, length, block)
    for r in np.unique(got[:, 0]):
        own = seen_by(shape, n, length, r)
        for _, t, at, hidden in got[got[:, 0] == r]:
            some = own[t:t + 16].any()
            assert not (some and hidden) and (at // 16 == t // 16 or not some), (shape, n, length, r, t)
            if hidden:  # (its values count as nothing)
                assert t + 16 <= length


@pytest.mark.parametrize("rows,tile", FORMS)
def test_windows(lib, rows, tile):
    """Windows and first tokens that begin and end inside a token tile."""
    for n, length, window, first, group in ((3, 1000, 100, 1, 4), (300, 5000, 1000, 4, 4), (1, 500, 1, 0, 1), (20, 777, 63, 1, 4),
                                            (200, 900, 64, 64, 4), (1, 4000, 16, 130, 8), (4, 64, 1, 300, 2), (9, 4, 3, 2, 3)):
        check(lib, (rows, tile, group, 2, 1, window, first), n, length)


@pytest.mark.parametrize("rows,tile", FORMS)
def test_drawn(lib, rows, tile):
    r = random.Random(rows)
    for _ in range(150):
        n, causal = r.choice([1, 2, 5, 40, 300]), r.random() < 0.9
        length = max(0, n + r.choice([0, 1, r.randint(0, 3000), -r.randint(0, 5)]))
        window = r.choice([0, 1, 15, 16, 17, 30, 64, 100, 129, 1000]) if causal else 0
        check(lib, (rows, tile, r.choice([1, 2, 3, 4, 6, 8, 16]), 1, int(causal), window, r.choice([0, 1, 5, 16, 64, 70, 200])), n, length)
