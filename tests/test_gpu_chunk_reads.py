"""``ops.chunk_attention`` with a window over block tables whose entries in front of it are anybody's: here they name a page
of NaNs, and the results are those of the whole table, bit for bit (``tests/test_chunk_reads.py`` has which blocks are
read at all)."""
import numpy as np
import pytest
import torch

from chunk_plain import Batch, visible
from test_gpu_chunk import call, check

pytestmark = pytest.mark.gpu


# row tiles of 32 rows; of 64 (more than 16 pairs of sequence and kv-head); of 256; of 256 and 32
@pytest.mark.parametrize("pairs", [[(2, 500), (3, 1000)], [(12, 600), (9, 330)] * 5, [(300, 1900), (150, 420)],
                                   [(1, 300), (600, 1500), (2, 900)] * 4], ids=str)
@pytest.mark.parametrize("preset,layout,bs", [("4bit", "soa", 16), ("4bit", "aos", 32), ("k8v4", "aos_heads", 16), ("3bit", "soa", 16)])
@pytest.mark.parametrize("window,first", [(1, 0), (100, 1), (200, 37)])
def test_entries_in_front_of_the_window(dev, pairs, preset, layout, bs, window, first):
    b = Batch(80, pairs, 2, 4, bs=bs, preset=preset, layout=layout)
    whole, hidden = b.table.copy(), 0
    for i, (n, length) in enumerate(pairs):
        seen = np.resize(visible(n, length, True, window, first).any(0), -(-length // bs) * bs)
        seen[length:] = False
        blocks = np.flatnonzero(~seen.reshape(-1, bs).any(1))
        b.table[i, blocks] = 0
        hidden += len(blocks)
    assert hidden > 0 and not np.array_equal(whole, b.table)
    for lse in (False, True):
        got = call(b, dev, window=window, first=first, lse=lse)
        check(b, got, "others' entries", window=window, first=first, lse=lse)
        cut, b.table = b.table, whole
        want = call(b, dev, window=window, first=first, lse=lse)
        b.table = cut
        for x, y in zip(got if lse else [got], want if lse else [want]):
            assert torch.equal(x, y)
