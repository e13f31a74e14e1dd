"""``ops.chunk_attention`` on two streams whose kernels run at the same time, each call with a workspace of its own."""
import numpy as np
import pytest
import torch

import span_plain as plain
from chunk_plain import D, Batch
from tq4_decode import codebook, ops

pytestmark = pytest.mark.gpu


def ready(b, dev):
    """A call whose inputs and workspace are on the device: nothing but its kernels is left to run."""
    kb, vb = plain.PRESETS[b.preset]
    put = lambda x: torch.from_numpy(np.ascontiguousarray(x)).to(dev)  # noqa: E731
    args = (b.query.to(dev), put(b.rot), b.cache.to(dev), put(b.table), put(b.lens), put(b.starts),
            put(codebook.centroids(D, kb).astype(np.float32)))
    ws = ops.ChunkWorkspace(b.tokens, len(b.pairs), b.hk * b.group, b.hk, dev)

    def call():
        return ops.chunk_attention(*args, return_lse=True, workspace=ws, key_bits=kb, value_bits=vb, layout=b.layout)
    return call, ws


@pytest.mark.parametrize("one,two", [([(1500, 4000), (5, 40)], [(4, 6000)] * 24), ([(64, 3000)] * 12, [(1, 900), (700, 2500)] * 3)],
                         ids=["tiles_of_256_and_32", "tiles_of_64_and_256"])
def test_streams_at_the_same_time(dev, one, two):
    """Calls of 100 us and more each, put on two streams in turn without a wait between them."""
    calls = [ready(Batch(90 + i, pairs, 2, 4, layout=layout), dev) for i, (pairs, layout) in enumerate(((one, "soa"), (two, "aos")))]
    want = [[x.clone() for x in call()] for call, _ in calls]
    streams = [torch.cuda.Stream(), torch.cuda.Stream()]
    for _ in range(3):
        for _, ws in calls:
            ws.out.zero_()
            ws.lse.zero_()
            ws.scratch.fill_(float("nan"))
        torch.cuda.synchronize()
        for _ in range(8):
            for (call, _), st in zip(calls, streams):
                with torch.cuda.stream(st):
                    call()
        torch.cuda.synchronize()
        for (_, ws), (out, lse) in zip(calls, want):
            assert torch.equal(ws.out, out) and torch.equal(ws.lse, lse)
