"""The order in which the waves of the shared-prefix kernel hand each other tiles (``csrc/prefix_tiles.h``),
run on the host with every wave's LDS accesses recorded.

Between two barriers nothing orders the waves, so a buffer that one wave reads there must not be written by
another, and what it reads must have been written, by every wave that decodes a share of it, before
the last barrier.  All waves have to pass the same number of barriers."""
import ctypes
import pathlib
import subprocess
import tempfile

import numpy as np
import pytest

HERE = pathlib.Path(__file__).resolve().parent
NAMES = ("keys", "factors", "values")
_lib = None


def lib():
    global _lib
    if _lib is None:
        with tempfile.TemporaryDirectory() as d:
            so = pathlib.Path(d) / "prefix_tiles_host.so"
            subprocess.run(["g++", "-O1", "-std=c++17", "-shared", "-fPIC", "-o", str(so), str(HERE / "prefix_tiles_host.cpp")],
                           check=True)
            _lib = ctypes.CDLL(str(so))
        _lib.host_accesses.argtypes = [ctypes.c_int] * 5 + [ctypes.c_void_p, ctypes.c_int, ctypes.c_void_p]
    return _lib


# waves (late, decodes K, decodes V) of the two forms: eight waves in two halves, two waves that do both
FORMS = {2: [(w >= 4, w < 4, w >= 4) for w in range(8)], 1: [(False, True, True)] * 2}


def accesses(wt, n):
    """Rows (wave, barriers passed, place, buffer, tile, write), and the barriers of each wave."""
    rows, barriers = [], []
    for wave, (late, k, v) in enumerate(FORMS[wt]):
        room, passed = 16 * (n + 2), ctypes.c_int()
        out = np.zeros((room, 5), np.int32)
        count = lib().host_accesses(wt, n, int(late), int(k), int(v), out.ctypes.data, room, ctypes.byref(passed))
        assert count > 0
        rows += [(wave, *map(int, r)) for r in out[:count]]
        barriers.append(passed.value)
    return rows, barriers


@pytest.mark.parametrize("wt", sorted(FORMS))
@pytest.mark.parametrize("n", [1, 2, 3, 4, 5, 8, 33])
def test_no_wave_writes_what_another_reads(wt, n):
    rows, barriers = accesses(wt, n)
    assert len(set(barriers)) == 1
    writes = [r for r in rows if r[5]]
    writers = {place: {w for w, _, p, _, _, _ in writes if p == place} for place in range(3)}
    read = {place: set() for place in range(3)}
    for wave, at, place, buffer, tile, write in rows:
        if write:
            continue
        read[place].add((wave, tile))
        what = f"wave {wave} reads the {NAMES[place]} of tile {tile} after barrier {at}"
        beside = [(w, t) for w, a, p, b, t, _ in writes if (a, p, b) == (at, place, buffer) and w != wave]
        assert not beside, f"{what} while (wave, tile) {beside} write there"
        for w in writers[place]:
            before = [(a, t) for v, a, p, b, t, _ in writes if (v, p, b) == (w, place, buffer) and a < at]
            assert before and max(before)[1] == tile, f"{what}: wave {w} left tile {max(before)[1] if before else None} there"
    for place in range(3):  # every wave works through all tiles
        assert read[place] == {(w, t) for w in range(len(FORMS[wt])) for t in range(n)}
