"""Calls of ``ops.rope_store`` at the edges of what it takes: sections that deal the frequencies evenly round the axes,
and queries turned in place."""
import pytest
import torch

from test_gpu_rope_store import build, check
from tq4_decode import ops

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("rot,sections", [(64, (11, 11, 10)), (16, (3, 3, 2)), (128, (22, 21, 21)), (96, (12, 12, 12, 12))])
@pytest.mark.parametrize("neox", [True, False])
def test_evenly_dealt_axes(dev, rot, sections, neox):
    for preset in ("4bit", "k8v4"):
        check(dev, build(21, 90, 4, 2, preset, rot=rot, neox=neox, sections=sections, in_turn=True))


@pytest.mark.parametrize("which", ["key", "value", "tail"])
def test_queries_in_place_among_keys_or_values(dev, which):
    """query_out is query: refused where keys or values lie in the same memory, also in part."""
    c = build(22, 24, 2, 2, fused=False)
    put = lambda x: torch.from_numpy(x).to(dev)  # noqa: E731
    mem = torch.cat([c["q"], c["k"]]).to(dev)
    q, k, v = mem[:24], c["k"].to(dev), c["v"].to(dev)
    if which == "key":
        k = q
    elif which == "value":
        v = q
    else:
        k = mem[12:36]
    args = (c["positions"].to(dev), c["table"].to(dev), c["cache"].to(dev), put(c["slots"]), put(c["rot_t"]), put(c["mids"]),
            put(c["cents"]))
    with pytest.raises(RuntimeError, match="query_out"):
        ops.rope_store(q, k, v, *args, query_out=q)
    # apart from them they may be the same rows
    out = ops.rope_store(q, k, v, *args)
    assert torch.equal(mem[:24].cpu(), c["q"]) and out.data_ptr() != q.data_ptr()
