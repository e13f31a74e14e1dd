"""What ``ops.chunk_attention`` may meet besides its sizes: values past f16's range, NaNs in tokens that some rows do not
see, rows of no sequence, strided queries, wide tables, large blocks and batches, lengths that change between a
captured graph's replays, two calls at once, and blocks past 4 GiB.

Bars as in ``test_gpu_chunk``, against masked attention in float64."""
import numpy as np
import pytest
import torch

import span_plain as plain
from chunk_plain import D, HALF_STEP, RHO, Batch, visible
from test_gpu_chunk import call, check
from test_gpu_prefix_bits import scalars_of
from tq4_decode import codebook, ops

pytestmark = pytest.mark.gpu
# row tiles of 32 rows, one and several a sequence; of 64 (more than 16 pairs of sequence and kv-head); of 256
SIZES = pytest.mark.parametrize("pairs", [[(2, 333), (7, 90)], [(12, 300), (9, 130)], [(12, 300), (9, 130)] * 5,
                                          [(150, 420), (40, 77)]], ids=str)


def log_uniform(low, high):
    return lambda rng, shape: np.exp(rng.uniform(np.log(low), np.log(high), shape))


def scalars(seed, *how):
    """A hook of `Batch`: other scales, zeros (and norms)."""
    def put(batch, cache, table, k, v):
        _, k[...], v[...] = scalars_of(*how)(np.random.default_rng(seed), cache, batch.preset, batch.layout)
    return put


@SIZES
@pytest.mark.parametrize("preset,layout", [("4bit", "soa"), ("3bit", "aos"), ("k8v4", "soa"), ("k3v4", "aos")])
@pytest.mark.parametrize("lse", [False, True])
def test_values_past_f16(dev, pairs, preset, layout, lse):
    """Scales up to f16's largest beside small ones, and scores that pass the running maximum by much.

    Bar: every token's weight is off by at most 2^-11 (its rounding) and the scores' share (eight deviations of
    rounding both factors and the rotation; none with a log-sum-exp), and so is the sum of all, which counts twice; its value by 2^-11 (twice, for one
    that is stored a 32nd as large) and by 2^-10 of the middle codes' distance where its scale is part of the weight:
    8 codes of 15, so at most 16/15 of the largest |v| of the token."""
    b = Batch(21, pairs, 2, 4, preset=preset, layout=layout, query_scale=4.0, spoil=False,
              change=scalars(5, log_uniform(0.01, 65000.0), lambda rng, shape: rng.uniform(-65000.0, 65000.0, shape)))
    got = call(b, dev, lse=lse)
    have = (got[0] if lse else got).double().cpu().numpy()
    assert np.isfinite(have).all()
    q = b.query.double().numpy()
    q = q if preset == "k8v4" else q @ b.rot.astype(np.float64)
    for i, (n, length) in enumerate(pairs):
        t = np.arange(length)
        at = b.table[i, t // b.bs], t % b.bs
        seen = np.repeat(visible(n, length, True, 0, 0), b.group, axis=0)
        for h in range(b.hk):
            k, v = b.k[at][:, h], b.v[at][:, h]
            qq = q[b.starts[i]:b.starts[i] + n, h * b.group:(h + 1) * b.group].reshape(-1, D)
            s = np.where(seen, qq @ k.T * D ** -0.5, -np.inf)
            p = np.exp(s - s.max(-1, keepdims=True))
            p /= p.sum(-1, keepdims=True)
            dev_s = 0 if lse or preset == "k8v4" else RHO * D ** -0.5 * np.sqrt(
                (2 * (qq ** 2) @ (k ** 2).T + 1.5 / D * (qq ** 2).sum(-1)[:, None] * (k ** 2).sum(-1)).max(-1))
            size = p @ np.abs(v).max(-1)
            bar = (2.0 ** -8 * 1.01) * np.abs(p @ v) + ((2.0 ** -9 + 2 * 8 * dev_s + 2.0 ** -11) * size)[..., None] + 1e-4
            part = have[b.starts[i]:b.starts[i] + n, h * b.group:(h + 1) * b.group].reshape(-1, D)
            assert (np.abs(part - p @ v) <= bar).all(), (i, h, (np.abs(part - p @ v) / bar).max())


@SIZES
@pytest.mark.parametrize("lse", [False, True])
def test_small_queries_of_large_keys(dev, pairs, lse):
    """Queries near f16's denormals, keys near its top: scores of ordinary size."""
    b = Batch(22, pairs, 2, 4, query_scale=2.0 ** -12, spoil=False,
              change=scalars(6, log_uniform(0.05, 0.4), lambda rng, s: rng.uniform(-3, 0.2, s), log_uniform(8000.0, 60000.0)))
    check(b, call(b, dev, lse=lse), "small queries", lse=lse)
    b = Batch(23, pairs, 2, 4, query_scale=2.0 ** 17, spoil=False,
              change=scalars(7, log_uniform(0.05, 0.4), lambda rng, s: rng.uniform(-3, 0.2, s), log_uniform(1e-4, 1e-3)))
    check(b, call(b, dev, lse=lse), "large queries", lse=lse)


@pytest.mark.parametrize("pairs", [[(4, 333), (7, 90)], [(12, 300), (9, 130)], [(12, 300), (9, 130)] * 5,
                                   [(150, 420), (40, 77)]], ids=str)
@pytest.mark.parametrize("preset,layout", [("4bit", "soa"), ("4bit", "aos"), ("k8v4", "aos"), ("3bit", "soa")])
@pytest.mark.parametrize("lse,window", [(False, 0), (True, 0), (False, 24), (True, 24)])
def test_nans_that_a_row_does_not_see(dev, pairs, preset, layout, lse, window):
    """The last new token's key and value are NaN, and where there is a window those of the token that only the first row
    still sees: every row that sees neither is as if they were not there."""
    b = Batch(24, pairs, 2, 4, preset=preset, layout=layout)
    bad = []
    for i, (n, length) in enumerate(pairs):
        bad += [(i, length - 1)] + ([(i, length - n + 1 - window)] if window else [])
    plain.spoil(b.cache, [(int(b.table[i, t // b.bs]), t % b.bs) for i, t in bad], preset, layout)
    want = b.want(window=window, lse=lse)
    got = call(b, dev, lse=lse, window=window)
    have = (got[0] if lse else got).double().cpu().numpy()
    for i, (n, length) in enumerate(pairs):
        seen = visible(n, length, True, window, 0)
        blind = ~seen[:, [t for j, t in bad if j == i]].any(1)
        rows = b.starts[i] + np.flatnonzero(blind)
        assert len(rows)
        over = np.abs(have[rows] - want[0][rows]) - HALF_STEP[b.dtype] * np.abs(want[0][rows]) - 8.1 * want[2][rows]
        assert over.max() <= 1e-4, (i, over.max())
        assert np.isnan(have[b.starts[i] + np.flatnonzero(~blind)]).all()


@SIZES
def test_rows_of_no_sequence_stay(dev, pairs):
    b = Batch(25, pairs, 2, 4, pad=(3, 5))
    ws = ops.ChunkWorkspace(b.tokens, len(pairs), 8, 2, dev)
    ws.out.fill_(7.0)
    ws.lse.fill_(9.0)
    got = call(b, dev, lse=True, workspace=ws)
    assert got[0].data_ptr() == ws.out.data_ptr()
    check(b, got, "padded", lse=True)
    for r in (slice(0, 3), slice(b.tokens - 5, b.tokens)):
        assert (ws.out[r] == 7.0).all() and (ws.lse[r] == 9.0).all()
    # nothing to do at all
    empty = Batch(26, [(0, 20), (0, 0)], 2, 4, pad=(1, 1))
    ws = ops.ChunkWorkspace(2, 2, 8, 2, dev)
    ws.out.fill_(7.0)
    assert (call(empty, dev, workspace=ws) == 7.0).all()


@SIZES
@pytest.mark.parametrize("out_dtype", [torch.bfloat16, torch.float16], ids=["to_bf16", "to_fp16"])
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16], ids=["bf16", "fp16"])
def test_strided_queries_and_other_outputs(dev, pairs, dtype, out_dtype):
    b = Batch(27, pairs, 2, 4, dtype=dtype)
    qkv = torch.randn(b.tokens, 8 + 2 * 2, D).to(dtype).to(dev)  # a projection's output
    qkv[:, :8] = b.query.to(dev)
    got = call(b, dev, query=qkv[:, :8], out_dtype=out_dtype)
    assert got.dtype == out_dtype and got.is_contiguous()
    b.dtype = out_dtype  # (the results' precision follows the outputs)
    check(b, got, "strided")


def test_one_strided_token(dev):
    b = Batch(28, [(1, 100)], 1, 1)
    wide = torch.zeros(1, 1, D + 5).to(dev).to(torch.bfloat16)
    wide[:, :, :D] = b.query.to(dev)
    check(b, call(b, dev, query=wide[:, :, :D]), "one token")


@pytest.mark.parametrize("bs", [64, 128, 256])
@pytest.mark.parametrize("hk,group", [(1, 3), (3, 5), (1, 12), (2, 32)])
def test_blocks_and_groups(dev, bs, hk, group):
    for pairs in ([(3, 500), (1, 64)], [(70, 300), (33, 33)]):
        b = Batch(29, pairs, hk, group, bs=bs, wide=20)
        check(b, call(b, dev), "blocks")
        check(b, call(b, dev, window=50, first=10, lse=True), "blocks, window", window=50, first=10, lse=True)


@SIZES
def test_sinks(dev, pairs):
    b = Batch(30, pairs, 2, 4)
    b.sinks[:] = [-np.inf, 0.0, 40.0, -40.0, 3.0, -np.inf, 88.0, -88.0]
    check(b, call(b, dev, sinks=True, lse=True), "sinks", sinks=True, lse=True)
    check(b, call(b, dev, sinks=True), "sinks", sinks=True)


def test_large_batches(dev):
    """More sequences than the plan holds in LDS; most without new tokens, or with one."""
    rng = np.random.default_rng(31)
    pairs = [(int(rng.choice([0, 1, 1, 2])), int(rng.integers(0, 70))) for _ in range(1500)]
    pairs = [(min(n, length), length) for n, length in pairs]
    b = Batch(31, pairs, 1, 2)
    check(b, call(b, dev, lse=True), "1500 sequences", lse=True)
    pairs = [(0, 5)] * 1100 + [(300, 300)] + [(0, 0)] * 100 + [(200, 1000)]
    b = Batch(32, pairs, 1, 2)
    check(b, call(b, dev), "two of 1302")


def test_starts_and_lengths_past_the_tensors(dev):
    """They end where the query's tokens and the table's blocks do."""
    b = Batch(33, [(4, 64), (6, 48)], 2, 4)
    want = call(b, dev)
    lens, starts = b.lens.copy(), b.starts.copy()
    b.lens[0], b.starts[2], b.starts[0] = 10 ** 9, 2 ** 31 - 1, -5
    got = call(b, dev)
    assert torch.equal(got, want)
    b.lens, b.starts = lens, starts


@pytest.mark.parametrize("lse", [False, True])
@pytest.mark.parametrize("tokens,kinds", [
    (48, [[(5, 200), (3, 64), (0, 9), (40, 400)], [(48, 48), (0, 0), (0, 0), (0, 0)], [(1, 1), (1, 300), (2, 2), (44, 333)],
          [(12, 700), (12, 12), (12, 90), (12, 13)]]),
    # (sequences of up to 24 tokens have a product of their own: some, none, all, all but one)
    (400, [[(24, 200), (3, 64), (0, 9), (373, 400)], [(100, 100), (100, 300), (25, 30), (175, 700)], [(24, 24), (1, 2), (20, 600), (5, 5)],
           [(1, 700), (1, 1), (1, 333), (397, 397)]]),
])
def test_replays_follow_lengths_and_starts(dev, lse, tokens, kinds):
    batches = [Batch(40 + i, p, 2, 4, wide=44, pad=(0, tokens - sum(n for n, _ in p))) for i, p in enumerate(kinds)]
    pool = max(b.cache.shape[0] for b in batches)
    first = batches[0]
    put = lambda x: torch.from_numpy(np.ascontiguousarray(x)).to(dev)  # noqa: E731
    cache = torch.zeros((pool,) + tuple(first.cache.shape[1:]), dtype=torch.uint8, device=dev)
    query, table = torch.zeros(tokens, 8, D, dtype=torch.bfloat16, device=dev), put(first.table)
    lens, starts, rot = put(first.lens), put(first.starts), put(first.rot)
    ws = ops.ChunkWorkspace(tokens, 4, 8, 2, dev)
    args = (query, rot, cache, table, lens, starts, put(codebook.centroids(D, 4).astype(np.float32)))

    def fill(b):
        cache[:b.cache.shape[0]] = b.cache.to(dev)
        query.copy_(b.query)
        for x, y in ((table, b.table), (lens, b.lens), (starts, b.starts), (rot, b.rot)):
            x.copy_(put(y))

    fill(first)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        ops.chunk_attention(*args, return_lse=lse, workspace=ws)
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        ops.chunk_attention(*args, return_lse=lse, workspace=ws)
    for b in batches + batches[::-1]:
        fill(b)
        ws.scratch.fill_(float("nan"))
        ws.out.zero_()
        ws.lse.zero_()
        graph.replay()
        torch.cuda.synchronize()
        got = (ws.out.clone(), ws.lse.clone()) if lse else ws.out.clone()
        check(b, got, "replayed", lse=lse)
        eager = call(b, dev, lse=lse)  # (the same plan, the same sums)
        rows = slice(int(b.starts[0]), int(b.starts[-1]))
        for x, y in zip(got if lse else [got], eager if lse else [eager]):
            assert torch.equal(x[rows], y[rows])


def test_two_calls_at_once(dev):
    one, two = Batch(50, [(300, 900), (5, 40)], 2, 4), Batch(51, [(4, 2000)] * 8, 2, 4)
    want = [call(b, dev).clone() for b in (one, two)]
    streams = [torch.cuda.Stream(), torch.cuda.Stream()]
    torch.cuda.synchronize()
    for _ in range(5):
        got = []
        for b, st in zip((one, two), streams):
            with torch.cuda.stream(st):
                got.append(call(b, dev))
        torch.cuda.synchronize()
        assert all(torch.equal(x, y) for x, y in zip(got, want))


@pytest.mark.parametrize("layout", ["soa", "aos"])
@pytest.mark.parametrize("pairs", [[(3, 300), (2, 45)], [(200, 400)]], ids=str)
def test_blocks_past_4_gib(dev, layout, pairs):
    b = Batch(60, pairs, 8, 4, layout=layout)
    n, shape = b.cache.shape[0], tuple(b.cache.shape[1:])
    per = int(np.prod(shape))
    pool = (1 << 32) // per + 2000
    at = torch.arange(n) * 2 + pool - 2 * n
    big = torch.zeros((pool,) + shape, dtype=torch.uint8, device=dev)
    big[at.to(dev)] = b.cache.to(dev)
    table = torch.from_numpy(b.table).long()
    put = lambda x: torch.from_numpy(np.ascontiguousarray(x)).to(dev)  # noqa: E731
    print(f"blocks {int(at.min())} .. {int(at.max())} of {pool}", flush=True)
    got = ops.chunk_attention(b.query.to(dev), put(b.rot), big, at[table].int().to(dev), put(b.lens), put(b.starts),
                              put(codebook.centroids(D, 4).astype(np.float32)), layout="soa" if layout == "soa" else "aos")
    check(b, got, "past 4 GiB")
    # and the reader, from the same blocks
    slots = torch.arange(n * 16)
    small = ops.cache_load(b.cache.to(dev), slots.int().to(dev), put(b.rot), put(codebook.centroids(D, 4).astype(np.float32)),
                           layout="soa" if layout == "soa" else "aos")
    far = ops.cache_load(big, (at[slots // 16] * 16 + slots % 16).int().to(dev), put(b.rot),
                         put(codebook.centroids(D, 4).astype(np.float32)), layout="soa" if layout == "soa" else "aos")
    assert all(torch.equal(x.view(torch.int16), y.view(torch.int16)) for x, y in zip(small, far))


@pytest.mark.parametrize("preset,layout", [("4bit", "soa"), ("3bit", "aos"), ("k8v4", "aos_heads")])
@pytest.mark.parametrize("pairs", [
    [(1, 300), (1, 77), (600, 900), (1, 1), (0, 20), (2, 500)] * 2,  # tiles of 256 rows and of 32
    [(1, 300), (30, 90), (8, 8), (9, 200), (25, 25)] * 4,            # of 64 and of 32
], ids=str)
def test_single_tokens_beside_chunks(dev, preset, layout, pairs):
    b = Batch(70, pairs, 4, 4, preset=preset, layout=layout)
    for how in (dict(), dict(lse=True), dict(window=60, first=7), dict(sinks=True), dict(causal=False, lse=True)):
        check(b, call(b, dev, **how), str(how), **how)
