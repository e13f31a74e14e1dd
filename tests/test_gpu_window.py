"""Sliding-window decode with first tokens that stay visible (``ops.window_decode``) against plain
attention over the visible tokens in float64.

Lengths and windows sit where the list of visible tiles can go wrong: a window that starts inside the
first tokens' tile, at a tile's edge, in the tile behind; windows of one token and longer than the
sequence; no first tokens, and more than the sequence has; blocks of several tiles; sequences in one
workgroup, in parts, and past the block-table entries a wave keeps.  Hidden pages' table entries point
at a page of NaNs.  Bar: 1e-4 plus half a step of the output type (the attention entries' bar)."""
import numpy as np
import pytest
import torch

import span_plain as plain
from tq4_decode import _lib, codebook, ops

pytestmark = pytest.mark.gpu
D = 128
HALF_STEP = {torch.float32: 0.0, torch.bfloat16: 2.0 ** -8, torch.float16: 2.0 ** -11}
EDGES = [1, 2, 15, 16, 17, 31, 32, 33, 47, 48, 49, 63, 64, 65, 100, 0, 777]


def visible(n, window, first):
    return [t for t in range(max(n, 0)) if t < first or t >= n - window]


def build(seed, lens, window, first, hk, group, bs=16, preset="4bit", layout="soa", wide=0, dtype=torch.float32):
    """Inputs on the CPU and the float64 result; page 0 is never a visible one and holds NaNs."""
    rng = np.random.default_rng(seed)
    width = max(wide, -(-max(max(lens), 1) // bs))
    seen = [sorted({t // bs for t in visible(n, window, first)}) for n in lens]
    pool = 1 + sum(map(len, seen))
    cache, k, v = plain.make_cache(rng, pool, bs, hk, preset, layout)
    cache.select(0, 0).fill_(0xFF)  # (fp16 scalars of all ones: NaN)
    table = np.zeros((len(lens), width), np.int32)
    ids = iter(1 + rng.permutation(pool - 1))
    for b, entries in enumerate(seen):
        for e in entries:
            table[b, e] = next(ids)
    hq = hk * group
    query = torch.from_numpy(rng.standard_normal((len(lens), hq, D)).astype(np.float32)).to(dtype)
    rot = plain.rotation(rng)
    sinks = rng.normal(0, 2, hq).astype(np.float32)
    q = query.double().numpy()
    if preset != "k8v4":
        q = q @ rot.astype(np.float64)

    def want(with_sinks, scale=D ** -0.5):
        rows = []
        for b, n in enumerate(lens):
            t = np.array(visible(n, window, first), int)
            kk, vv = k[table[b, t // bs], t % bs], v[table[b, t // bs], t % bs]
            rows.append(plain.attend(q[b], kk.reshape(len(t), hk, D), vv.reshape(len(t), hk, D),
                                     sinks if with_sinks else None, scale))
        return np.stack([r[0] for r in rows]), np.stack([r[1] for r in rows])

    return dict(query=query, rot=torch.from_numpy(rot), cache=cache, table=torch.from_numpy(table),
                lens=torch.tensor(lens, dtype=torch.int32), sinks=torch.from_numpy(sinks), want=want, preset=preset,
                layout=layout)


def to_device(c, dev):
    """The cache keeps its view: a head-major one is moved as it lies in memory."""
    c = dict(c)
    for n in ("query", "rot", "table", "lens", "sinks"):
        c[n] = c[n].to(dev)
    heads = c["layout"] == "aos_heads"
    c["cache"] = c["cache"].transpose(1, 2).to(dev).transpose(1, 2) if heads else c["cache"].to(dev)
    kb = plain.PRESETS[c["preset"]][0]
    c["cents"] = None if kb == 8 else torch.from_numpy(codebook.centroids(D, kb)).to(dev)
    return c


def call(c, dev, window, first, splits, sinks=False, **kw):
    kb, vb = plain.PRESETS[c["preset"]]
    return ops.window_decode(c["query"], None if kb == 8 else c["rot"], c["cache"], c["table"], c["lens"], c["cents"],
                             splits, window, first_tokens=first, key_bits=kb, value_bits=vb,
                             layout="soa" if c["layout"] == "soa" else "aos", sinks=c["sinks"] if sinks else None, **kw)


def check(dev, c, window, first, splits, sinks=False, **kw):
    d = to_device(c, dev)
    out, lse = call(d, dev, window, first, splits, sinks, **kw)
    torch.cuda.synchronize()
    want, want_lse = c["want"](sinks)
    plain.close(out.float().cpu().numpy(), want, HALF_STEP[out.dtype], "out")
    plain.close(lse.cpu().numpy(), want_lse, 0.0, "lse")


@pytest.mark.parametrize("window", [1, 15, 16, 17, 31, 33, 64, 5000])
@pytest.mark.parametrize("first", [0, 1, 16, 18])
def test_edges(dev, window, first):
    check(dev, build(1, EDGES, window, first, 2, 4), window, first, 8)


@pytest.mark.parametrize("preset", list(plain.PRESETS))
@pytest.mark.parametrize("layout", ["soa", "aos", "aos_heads"])
def test_presets_and_layouts(dev, preset, layout):
    for group in (4, 8):
        check(dev, build(2, EDGES + [1500], 200, 5, 2, group, preset=preset, layout=layout), 200, 5, 8, sinks=group == 8)


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16, torch.float16])
@pytest.mark.parametrize("preset", ["4bit", "k8v4"])
def test_query_types_and_output_types(dev, dtype, preset):
    c = build(3, [300, 0, 40, 1000], 250, 4, 8, 4, preset=preset, dtype=dtype)
    check(dev, c, 250, 4, 32)
    check(dev, c, 250, 4, 32, out_dtype=torch.float32)


@pytest.mark.parametrize("bs", [16, 32, 64, 128])
@pytest.mark.parametrize("wide", [0, 700])
def test_blocks_and_table_widths(dev, bs, wide):
    lens = [2000, 1999, 1, 130, 64, 0, 900]
    check(dev, build(4, lens, 333, 70, 8, 4, bs=bs, wide=wide), 333, 70, 16, sinks=True)


# one workgroup per sequence, parts, stretches over several sequences, long runs of a wave, few rows
FORMS = {
    "parts": ([9000, 8000, 40], 4096, 100, 8, 4, 32),
    "stretches": ([int(x) for x in np.linspace(30, 3000, 70)], 900, 4, 8, 4, 32),
    "one row": ([3001], 2500, 0, 8, 4, 1),
    "past the block-table entries": ([140000, 100], 70000, 33, 1, 4, 2),
    "batch past the device": ([100] * 300, 50, 3, 8, 4, 4),
    "three kv-heads, group of 6": ([1500, 700, 1, 0, 90, 333], 300, 20, 3, 6, 32),
    "one kv-head, group of 16": ([2500, 80], 2000, 17, 1, 16, 32),
    "group of 1": ([500, 20, 333], 100, 2, 4, 1, 8),
}


@pytest.mark.parametrize("name", FORMS)
def test_forms(dev, name):
    lens, window, first, hk, group, splits = FORMS[name]
    check(dev, build(5, lens, window, first, hk, group), window, first, splits, sinks="parts" in name)


def test_a_window_past_every_length_is_the_full_step(dev):
    c = to_device(build(6, [700, 1, 33, 0], 1 << 30, 0, 8, 4), dev)
    cents = c["cents"]
    for window, first in ((1 << 30, 0), (0x7FFFFFFF, 0x7FFFFFFF), (1, 0x7FFFFFFF), (700, 0)):
        out, lse = call(c, dev, window, first, 8)
        full, full_lse = ops.full_decode(c["query"], c["rot"], c["cache"], c["table"], c["lens"], cents, 8)
        plain.close(out.cpu().numpy(), full.cpu().numpy(), 0.0, "out", atol=1e-5)
        plain.close(lse.cpu().numpy(), full_lse.cpu().numpy(), 0.0, "lse", atol=1e-5)


def test_masked_tokens_of_a_visible_page_do_not_count(dev):
    """Hidden tokens that share a tile with visible ones hold NaN scalars."""
    c = build(7, [70], 20, 3, 1, 4)
    flat = c["cache"].view(c["cache"].size(0), -1)
    meta = flat[:, 16 * 128:].view(torch.float16).view(-1, 1, 3, 16)
    pages = c["table"][0].long()
    for t in list(range(3, 16)) + [48, 49]:
        meta[pages[t // 16], 0, :, t % 16] = float("nan")
    for t in (70 - 64 + i for i in range(10)):  # and behind the last token
        meta[pages[4], 0, :, t] = float("inf")
    check(dev, c, 20, 3, 4)


def test_workspaces_streams_and_graph(dev):
    c = to_device(build(8, [900, 1999, 2000, 640], 1 << 30, 0, 8, 4, dtype=torch.bfloat16), dev)  # (every page there)
    ws = ops.DecodeWorkspace(4, 32, 16, dev, torch.bfloat16)
    want, want_lse = call(c, dev, 500, 4, 16)
    side = torch.cuda.Stream()
    with torch.cuda.stream(side):
        side.wait_stream(torch.cuda.default_stream())
        out, lse = call(c, dev, 500, 4, 16, workspace=ws)
    side.synchronize()
    assert out is ws.out and torch.equal(out.isnan(), want.isnan()) and torch.equal(lse, want_lse)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        call(c, dev, 500, 4, 16, workspace=ws)
    for lens in ([900, 17, 2000, 0], [30, 1999, 1, 640], [4, 505, 1024, 1]):
        c["lens"].copy_(torch.tensor(lens, dtype=torch.int32))
        ws.out.zero_()
        graph.replay()
        torch.cuda.synchronize()
        got = ws.out.clone()
        eager, _ = call(c, dev, 500, 4, 16)
        assert torch.equal(got.isnan(), eager.isnan())
        assert torch.equal(got[~got.isnan()], eager[~eager.isnan()])


REFUSED = [
    (dict(window=0), "window"), (dict(window=2.0), "window"), (dict(first_tokens=-1), "first_tokens"),
    (dict(key_bits=5), "key/value bits"), (dict(bs=8), "power-of-two"), (dict(bs=48), "power-of-two"),
    (dict(attn_scale=0.0), "attn_scale"), (dict(layout="xyz"), "layout"),
]


@pytest.mark.parametrize("over,text", REFUSED)
def test_refusals(dev, over, text):
    over = dict(over)
    c = to_device(build(9, [60, 20], 10, 0, 2, 4, bs=over.pop("bs", 16)), dev)
    kw = dict(window=10, first_tokens=0, layout="soa", key_bits=4)
    kw.update(over)
    cents = torch.from_numpy(codebook.centroids(D, 4)).to(dev)
    with pytest.raises(RuntimeError, match=text):
        ops.window_decode(c["query"], c["rot"], c["cache"], c["table"], c["lens"], cents, 4, kw.pop("window"), **kw)
    bad = ops.DecodeWorkspace(2, 8, 5, dev, torch.float32)
    with pytest.raises(RuntimeError, match="workspace"):
        ops.window_decode(c["query"], c["rot"], c["cache"], c["table"], c["lens"], cents, 4, 10, workspace=bad)


def test_c_entry_refuses(dev):
    lib, p = _lib.load(), 1 << 12
    args = lambda **o: [o.get("query", p), 1, p, p, p, p, p, p, p, p, 1, p, 2, 8, 2, o.get("D", 128), 16, 4, 16 * 2 * 134,  # noqa: E731
                        4, 0, 0.1, None, o.get("kb", 4), 4, o.get("window", 5), o.get("first", 0), None]
    for o, code in ((dict(query=None), 1), (dict(query=p + 8), 1), (dict(D=64), 2), (dict(kb=8, window=0), 1),
                    (dict(kb=2), 2), (dict(window=0), 1), (dict(first=-1), 1)):
        assert lib.tq4_window_decode(*args(**o)) == code, o
