"""The workgroups that the plan of ``chunk_attention`` counts on (``chunk_attention.hip``): one of eight waves per CU for
row tiles of 256 rows, two of four waves for smaller ones.  The built library's own code objects say what every instance
needs: 256 registers a wave at most (two waves per SIMD) and a share of the CU's 160 KB LDS."""
import pathlib
import re

import pytest

from test_prefix_places import READELF, kernels
from tq4_decode import build


@pytest.mark.skipif(not pathlib.Path(READELF).exists(), reason="needs llvm-readelf")
def test_every_instance_fits_its_places(tmp_path):
    if not build.LIB.exists():
        build.build()
    many, some, few = set(), set(), set()
    for name, (registers, lds) in kernels(tmp_path).items():
        tiles = re.search(r"chunk_kernelILi(\d)ELb(\d)ELb(\d)ELb(\d)ELi(\d)ELi(\d)ELi64ELi(\d)ELb(\d)E", name)
        flat = re.search(r"chunk_few_kernelILi(\d)ELb(\d)ELb(\d)ELb(\d)ELb(\d)E", name)
        if not (tiles or flat):
            continue
        assert registers <= 256, (name, registers)
        if tiles and tiles.group(5) == "8":
            many.add(tiles.groups())
            assert lds <= 160 * 1024, (name, lds)
        else:
            (some if tiles else few).add((tiles or flat).groups())
            assert lds <= 80 * 1024, (name, lds)
    # two layouts, four presets, two precisions
    assert len(many) == len(some) == len(few) == 16
