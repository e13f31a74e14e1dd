"""Several new tokens per sequence over the cache (``ops.chunk_attention``) against plain masked attention in float64.

Sizes sit where the products can go wrong: chunks of one token, of one and several row tiles (32, 64 and 256 rows) and
past their ends, lengths around the 64-token tile and the pages, row tiles cut between workgroups, windows that
begin inside a tile, first tokens that end inside one, rows that see nothing.  Bar: half a step of the output type, 1e-4,
and eight standard deviations of what rounding the products' operands to f16 does (``chunk_plain.attend``: a score's
error is the sum over its dims of each rounded factor's, a weighted value has one or two rounded factors)."""
import numpy as np
import pytest
import torch

import span_plain as plain
from chunk_plain import D, HALF_STEP, Batch
from tq4_decode import codebook, ops

pytestmark = pytest.mark.gpu


def call(b, dev, causal=True, window=0, first=0, sinks=False, lse=False, workspace=None, query=None, out_dtype=None, **more):
    kb, vb = plain.PRESETS[b.preset]
    to = lambda x: torch.from_numpy(np.ascontiguousarray(x)).to(dev)  # noqa: E731
    cents = None if kb == 8 else to(codebook.centroids(D, kb).astype(np.float32))
    cache = b.cache.transpose(1, 2).contiguous().to(dev).transpose(1, 2) if b.layout == "aos_heads" else b.cache.to(dev)
    return ops.chunk_attention(
        b.query.to(dev) if query is None else query, None if kb == 8 else to(b.rot), cache, to(b.table), to(b.lens),
        to(b.starts), cents, causal=causal, window=window, first_tokens=first, key_bits=kb, value_bits=vb,
        layout="soa" if b.layout == "soa" else "aos", return_lse=lse, workspace=workspace, out_dtype=out_dtype,
        sinks=to(b.sinks) if sinks else None, **more)


def check(b, got, what, lse=False, **how):
    out, sums, dev_out, dev_lse = b.want(lse=lse, **how)
    have = (got[0] if lse else got).double().cpu().numpy()
    r = np.concatenate([np.arange(s, s + n) for s, (n, _) in zip(b.starts, b.pairs)]).astype(int)
    step = HALF_STEP[b.dtype]
    assert np.array_equal(np.isnan(have[r]), np.isnan(out[r])), what
    fine = np.isfinite(out[r])
    over = np.abs(have[r] - out[r]) - step * np.abs(out[r]) - 8 * dev_out[r] * (1 + step)
    assert not fine.any() or over[fine].max() <= 1e-4, f"{what}: {over[fine].max():.2e} over"
    if lse:
        have = got[1].double().cpu().numpy()[r]
        fine = np.isfinite(sums[r])
        assert np.array_equal(have[~fine], sums[r][~fine]), what
        assert not fine.any() or (np.abs(have - sums[r]) - 8 * dev_lse[r])[fine].max() <= 1e-4, what


LENGTHS = [
    [(1, 1)], [(1, 333)], [(4, 337)], [(2, 2), (1, 64), (3, 65), (4, 63)], [(0, 10), (5, 17), (0, 0), (1, 4096)],
    [(8, 8), (7, 128), (1, 1000), (3, 129)], [(16, 700)], [(40, 40), (13, 500)], [(64, 64)], [(65, 190), (1, 30), (129, 129)],
    [(300, 300)], [(257, 1000), (90, 91)], [(700, 2000), (1, 5), (0, 7), (333, 333)],
    # (more than 16 pairs of sequence and kv-head: row tiles of 64 and of 32 rows)
    [(40, 200), (9, 64), (12, 12), (11, 333), (0, 5)] * 4, [(25, 130), (1, 900), (100, 101), (20, 64)] * 5,
]


@pytest.mark.parametrize("pairs", LENGTHS, ids=str)
@pytest.mark.parametrize("hk,group", [(1, 1), (2, 4), (1, 6), (2, 16)])
def test_lengths(dev, pairs, hk, group):
    b = Batch(len(pairs) + hk, pairs, hk, group)
    check(b, call(b, dev), "causal")
    check(b, call(b, dev, lse=True), "with sums", lse=True)


@pytest.mark.parametrize("preset", list(plain.PRESETS))
@pytest.mark.parametrize("layout", ["soa", "aos", "aos_heads"])
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16], ids=["bf16", "fp16"])
@pytest.mark.parametrize("pairs", [[(3, 130), (1, 77)], [(150, 333), (9, 200)], [(10, 100), (20, 20)],
                                   [(10, 100), (20, 20), (11, 65)] * 4], ids=str)
def test_presets(dev, preset, layout, dtype, pairs):
    b = Batch(7, pairs, 2, 4, bs=32, preset=preset, layout=layout, dtype=dtype)
    check(b, call(b, dev), "causal")
    check(b, call(b, dev, sinks=True), "sinks", sinks=True)
    check(b, call(b, dev, causal=False, lse=True), "context", causal=False, lse=True)


@pytest.mark.parametrize("window,first", [(1, 0), (16, 0), (63, 1), (64, 64), (100, 5), (65, 130), (4096, 3), (1, 300)])
@pytest.mark.parametrize("pairs", [[(1, 500), (3, 300)], [(20, 777)], [(200, 900), (130, 130)], [(20, 777), (9, 300)] * 5], ids=str)
def test_windows(dev, window, first, pairs):
    b = Batch(11, pairs, 2, 4)
    check(b, call(b, dev, window=window, first=first), "window", window=window, first=first)
    check(b, call(b, dev, window=window, first=first, sinks=True, lse=True), "window", window=window, first=first, sinks=True,
          lse=True)


def test_rows_that_see_nothing(dev):
    # more new tokens than the cache holds: the first ones lie before it; and no tokens at all
    for pairs in ([(9, 4), (5, 0), (2, 2)], [(300, 100), (70, 0)]):
        b = Batch(3, pairs, 2, 4)
        for sinks in (False, True):
            check(b, call(b, dev, lse=True, sinks=sinks), "nothing", lse=True, sinks=sinks)
            check(b, call(b, dev, sinks=sinks), "nothing", sinks=sinks)
