"""How the sequences' own tokens behind a shared prefix are planned (``csrc/step_plan.h``): a sequence shorter than
the prefix has up to prefix_len - 1 of them, and no workgroup may be left alone with those."""
import ctypes
import pathlib
import subprocess
import tempfile

import pytest

import step_cut_host as host

HERE = pathlib.Path(__file__).resolve().parent


@pytest.fixture(scope="module")
def own_blocks():
    with tempfile.TemporaryDirectory() as d:
        so = pathlib.Path(d) / "own_blocks_host.so"
        subprocess.run(["g++", "-O1", "-std=c++17", "-shared", "-fPIC", "-o", str(so), str(HERE / "own_blocks_host.cpp")], check=True)
        return ctypes.CDLL(str(so)).host_own_blocks


@pytest.mark.parametrize("batch,prefix,tail,short", [(64, 32768, 100, [29000]), (64, 8192, 100, [8000] * 4), (24, 16384, 300, [15000]),
                                                     (8, 65536, 40, [60000]), (64, 8192, 1100, [8191])])
def test_sequences_shorter_than_the_prefix_are_cut(own_blocks, batch, prefix, tail, short):
    blocks = own_blocks((prefix + tail + 15) // 16, prefix // 16)
    p = host.plan(batch, 8, blocks, 32)
    lens = short + [tail] * (batch - len(short))  # tokens of their own
    tiles = [sum(end - first for _, first, end, _, _ in host.segments(lens, 32, p, x)) for x in range(p.nx)]
    total = sum(-(-n // 16) for n in lens)
    assert sum(tiles) == total
    # a 16th of the longest, or twice the even share
    assert max(tiles) <= max(-(-max(short) // 16 // 16), 2 * -(-total // p.nx)), (max(tiles), total, p)


def test_blocks(own_blocks):
    assert own_blocks(100, 0) == 100
    assert own_blocks(100, 20) == 80
    assert own_blocks(100, 90) == 90
    assert own_blocks(100, 100) == 100
