"""How a ``chunk_attention`` call is cut into workgroups (``csrc/chunk_plan.h``), built for the host.  For any batch the cuts
do not decrease, every visited token tile of every row tile falls to exactly one workgroup, and a row tile visits every
token tile that one of its rows sees."""
import ctypes
import pathlib
import random
import subprocess

import numpy as np
import pytest

HERE = pathlib.Path(__file__).resolve().parent


@pytest.fixture(scope="module")
def lib(tmp_path_factory):
    so = tmp_path_factory.mktemp("plan") / "chunk_plan_host.so"
    subprocess.run(["g++", "-O1", "-std=c++17", "-shared", "-fPIC", "-o", str(so), str(HERE / "chunk_plan_host.cpp")], check=True)
    lib = ctypes.CDLL(str(so))
    lib.host_work.restype = ctypes.c_double
    return lib


def ints(x):
    x = np.ascontiguousarray(x, np.int32)
    return x, x.ctypes.data_as(ctypes.c_void_p)


class Plan:
    def __init__(self, lib, shape, starts, lens, tokens, longest, groups):
        self.shape, batch = shape, len(lens)
        (_, s), (keep, st), (keep2, ln) = ints(shape), ints(starts), ints(lens)
        cuts = np.zeros((groups + 1, 4), np.int32)
        lib.host_cuts(s, st, ln, batch, tokens, longest, groups, ints(cuts)[1])
        self.cuts = [tuple(int(v) for v in c) for c in cuts]
        self.seqs, self.visits = [], []
        for b in range(batch):
            seq, room = np.zeros(3, np.int32), 1 + tokens * shape[2] // shape[0] + 1
            v = np.zeros((room, 3), np.int32)
            n = lib.host_visits(s, st, ln, b, tokens, longest, ints(seq)[1], ints(v)[1], room)
            assert n <= room
            self.seqs.append(tuple(int(x) for x in seq))
            self.visits.append([tuple(int(x) for x in row) for row in v[:n]])

    def check(self):
        """Walks the list as a workgroup does, from each cut to the next."""
        batch, heads = len(self.seqs), self.shape[3]
        cuts = self.cuts
        assert cuts[-1] == (batch, 0, 0, 0) and all(a <= b for a, b in zip(cuts, cuts[1:]))
        got = {}
        for at, end in zip(cuts, cuts[1:]):
            if at == end:
                continue
            b, h, r, i = at
            while b < batch:
                count = self.visits[b][r][2]
                last = (b, h, r) == end[:3]
                stop = end[3] if last else count
                assert 0 <= i <= stop <= count, (at, end)
                if i < stop or (count == 0 and not last):
                    got.setdefault((b, h, r), []).append((i, stop))
                if last:
                    break
                i, r = 0, r + 1
                if r == len(self.visits[b]):
                    r, h = 0, h + 1
                    if h == heads:
                        h, b = 0, b + 1
                        while b < batch and not self.visits[b]:
                            b += 1
                assert (b, h, r, 0) <= end
        for b, tiles in enumerate(self.visits):
            for h in range(heads):
                for r, (_, _, count) in enumerate(tiles):
                    runs = got.pop((b, h, r))
                    assert runs[0][0] == 0 and runs[-1][1] == count
                    assert all(x[1] == y[0] for x, y in zip(runs, runs[1:]))
        assert not got

    def check_visits(self):
        rows, tile, group, _, causal, window, first = self.shape
        for (row0, n, length), tiles in zip(self.seqs, self.visits):
            assert len(tiles) == -(-n * group // rows)
            for r, (head, skip, count) in enumerate(tiles):
                places = [i if i < head else i + skip for i in range(count)]
                assert len(set(places)) == count
                if count:
                    assert max(places) * tile < length
                needed = set()
                for t in range(r * rows // group, min(((r + 1) * rows - 1) // group, n - 1) + 1):
                    end = max(0, length - n + t + 1) if causal else length
                    begin = max(0, end - window) if window else 0
                    needed |= set(range(begin // tile, -(-end // tile)))
                    if window:
                        needed |= set(range(0, -(-min(first, end) // tile)))
                assert needed <= set(places)


def draw(r):
    group, heads = r.choice([1, 2, 3, 4, 6, 8, 16]), r.choice([1, 2, 3, 8])
    rows, tile = r.choice([(256, 64), (64, 64), (32, 128)])
    causal = r.random() < 0.8
    window = r.choice([0, 0, 1, 30, 64, 500]) if causal else 0
    return (rows, tile, group, heads, int(causal), window, r.choice([0, 0, 5, 64, 200]))


@pytest.mark.parametrize("seed", range(6))
def test_every_tile_has_one_workgroup(lib, seed):
    r = random.Random(seed)
    for _ in range(60):
        batch = r.choice([1, 1, 2, 3, 8, 40, 200])
        most = r.choice([1, 4, 40, 400])
        counts = [r.choice([0, 1, r.randint(0, most), most]) for _ in range(batch)]
        lens = [max(0, n + r.choice([0, 0, 1, r.randint(0, 3000), -r.randint(0, 5)])) for n in counts]
        starts = np.concatenate([[0], np.cumsum(counts)]) + r.choice([0, 3])
        p = Plan(lib, draw(r), starts, lens, int(starts[-1]) + r.choice([0, 2]) + 1, 1 << 20, r.choice([1, 2, 7, 256, 512]))
        assert [q[1:] for q in p.seqs] == list(zip(counts, lens))
        p.check()
        p.check_visits()


def test_ends_of_the_range(lib):
    r = random.Random(9)
    for counts, lens in (([0] * 5, [7] * 5), ([1], [0]), ([1], [1]), ([3, 0, 0], [2, 0, 5]), ([0, 0, 1], [9, 9, 1]),
                         ([1 << 15], [1 << 15]), ([1, 9000], [1 << 20, 1 << 20]), ([0, 1] * 1000, [5, 1] * 1000)):
        starts = np.concatenate([[0], np.cumsum(counts)])
        for _ in range(4):
            p = Plan(lib, draw(r), starts, lens, max(1, int(starts[-1])), 1 << 20, 512)
            p.check()


def test_values_past_the_tensors(lib):
    """Whatever starts and lengths hold, tokens stay inside the query and lengths inside the table."""
    r = random.Random(10)
    wild = [-2 ** 31, -7, 0, 3, 11, 20, 21, 1000, 2 ** 31 - 1]
    for _ in range(200):
        batch = r.choice([1, 3, 9])
        p = Plan(lib, draw(r), [r.choice(wild) for _ in range(batch + 1)], [r.choice(wild) for _ in range(batch)], 20, 640, 64)
        for row0, n, length in p.seqs:
            assert 0 <= row0 and n >= 0 and row0 + n <= 20 and 0 <= length <= 640
        p.check()


def test_shares_are_even(lib):
    """A workgroup's stretch is no longer than its share and what a cut may move (2 tiles at either end), and one."""
    for shape, counts, lens in (((256, 64, 4, 8, 1, 0, 0), [8192], [8192]), ((32, 128, 8, 8, 1, 0, 0), [4] * 64, [4096] * 64),
                                ((256, 64, 8, 4, 1, 1024, 64), [2048] * 3, [9000] * 3)):
        starts, groups = np.concatenate([[0], np.cumsum(counts)]), 256
        p = Plan(lib, shape, starts, lens, int(starts[-1]), 1 << 20, groups)
        p.check()
        spans = np.zeros(groups)
        list_of = [(b, h, r) for b in range(len(counts)) for h in range(shape[3]) for r in range(len(p.visits[b]))]
        place, at = {}, 0.0
        for key in list_of:
            place[key] = at
            at += 3 + p.visits[key[0]][key[2]][2]
        where = lambda c: at if c[0] == len(counts) else place[c[:3]] + (c[3] and 3 + c[3])  # noqa: E731
        spans = np.diff([where(c) for c in p.cuts])
        assert spans.max() <= at / groups * 1.1 + 2 * 2 + 1 + 3, (spans.max(), at / groups)
