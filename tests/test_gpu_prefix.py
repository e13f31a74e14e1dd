"""Decode of a batch that shares its first pages (``ops.prefix_decode``) against plain attention over every
sequence's tokens in float64.

Sizes sit where the shared product can go wrong: prefixes that end inside its 64-token tile, one tile and
many, one split and several, row counts below and above its 32, 64 and 128 rows, tails of none and one
token, sequences shorter than the prefix (on other pages) and empty ones, tails in one workgroup and in
parts.  Bar: half a step of the output type, the attention entries' 1e-4, and eight standard deviations
of what rounding q, c, c n, n, p and v to f16 does to a row: each factor's relative error spread over
half a step (2^-11) has a deviation rho = 2^-11 / sqrt 3 at most, so a token's score is off by
2 rho sqrt(sum_d (q_d k_d scale)^2) = d_t, the output by sqrt(sum_t p_t^2 (d_t^2 (v_t - o)^2 + 2 rho^2 v_t^2)) and
the log-sum-exp by sqrt(sum_t p_t^2 d_t^2)."""
import numpy as np
import pytest
import torch

import span_plain as plain
from tq4_decode import _lib, codebook, ops

pytestmark = pytest.mark.gpu
D = 128
HALF_STEP = {torch.bfloat16: 2.0 ** -8, torch.float16: 2.0 ** -11}
RHO = 2.0 ** -11 / 3 ** 0.5


def build(seed, lens, prefix, hk, group, bs=16, preset="4bit", layout="soa", dtype=torch.float16, wide=0,
          query_scale=None):
    """Sequences as long as `prefix` share its pages; the others have pages of their own.  Page 0 is nobody's
    and holds NaNs."""
    rng = np.random.default_rng(seed)
    width = max(wide, prefix // bs, -(-max(lens) // bs))
    shared = prefix // bs
    own = [-(-n // bs) - (shared if n >= prefix else 0) for n in lens]
    pool = 1 + shared + sum(own)
    cache, k, v = plain.make_cache(rng, pool, bs, hk, preset, layout)
    cache.select(0, 0).fill_(0xFF)
    ids = 1 + rng.permutation(pool - 1)
    table, at = np.zeros((len(lens), width), np.int32), shared
    for b, n in enumerate(lens):
        start = 0
        if n >= prefix:
            table[b, :shared] = ids[:shared]
            start = shared
        table[b, start:start + own[b]] = ids[at:at + own[b]]
        at += own[b]
    hq = hk * group
    query = rng.standard_normal((len(lens), hq, D)).astype(np.float32)
    if query_scale is not None:
        query *= np.asarray(query_scale, np.float32).reshape(len(lens), -1, 1)
    query = torch.from_numpy(query).to(dtype)
    rot = plain.rotation(rng)
    sinks = rng.normal(0, 2, hq).astype(np.float32)
    q = query.double().numpy()
    if preset != "k8v4":
        q = q @ rot.astype(np.float64)

    def want(with_sinks):
        outs, lses, so, sl = [], [], [], []
        for b, n in enumerate(lens):
            t = np.arange(n)
            kk, vv = k[table[b, t // bs], t % bs], v[table[b, t // bs], t % bs]
            o, lse = plain.attend(q[b], kk, vv, sinks if with_sinks else None)
            outs.append(o)
            lses.append(lse)
            qg, og, lg = q[b].reshape(hk, group, D), o.reshape(hk, group, D), lse.reshape(hk, group, 1)
            p = np.exp(np.einsum("hgd,thd->hgt", qg, kk) * D ** -0.5 - lg) if n else np.zeros((hk, group, 0))
            d2 = 4 * RHO ** 2 * np.einsum("hgd,thd->hgt", qg ** 2, kk ** 2) / D
            vt = vv.transpose(1, 0, 2)[:, None]
            var = (p[..., None] ** 2 * (d2[..., None] * (vt - og[:, :, None]) ** 2 + 2 * RHO ** 2 * vt ** 2)).sum(2)
            so.append(np.sqrt(var).reshape(hq, D))
            sl.append(np.sqrt((p ** 2 * d2).sum(-1)).reshape(hq))
        return np.stack(outs), np.stack(lses), np.stack(so), np.stack(sl)

    return dict(query=query, rot=torch.from_numpy(rot), cache=cache, table=torch.from_numpy(table),
                lens=torch.tensor(lens, dtype=torch.int32), sinks=torch.from_numpy(sinks), want=want, preset=preset,
                layout=layout, prefix=prefix)


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


def call(c, splits, sinks=False, prefix=None, **kw):
    kb, vb = plain.PRESETS[c["preset"]]
    kw.setdefault("kernel", "shared")
    return ops.prefix_decode(c["query"], None if kb == 8 else c["rot"], c["cache"], c["table"], c["lens"], c["cents"],
                             splits, c["prefix"] if prefix is None else prefix, key_bits=kb, value_bits=vb,
                             layout="soa" if c["layout"] == "soa" else "aos", sinks=c["sinks"] if sinks else None, **kw)


def within(got, want, step, sigma, what):
    got = got.double().cpu().numpy()
    assert np.array_equal(np.isnan(got), np.isnan(want)), f"{what}: NaNs differ"
    fine = np.isfinite(want)
    assert np.array_equal(got[~fine & ~np.isnan(want)], want[~fine & ~np.isnan(want)]), f"{what}: infinities differ"
    over = np.abs(got[fine] - want[fine]) / (1e-4 + step * np.abs(want[fine]) + 8 * sigma[fine])
    assert over.size == 0 or over.max() <= 1.0, f"{what}: {over.max():.2f} times the bar"


def check(dev, c, splits, sinks=False, **kw):
    d = to_device(c, dev)
    out, lse = call(d, splits, sinks, **kw)
    torch.cuda.synchronize()
    o, l, so, sl = c["want"](sinks)
    within(out, o, HALF_STEP[out.dtype], so, "out")
    within(lse, l, 0.0, sl, "lse")


@pytest.mark.parametrize("prefix", [16, 32, 48, 64, 80, 128, 144, 656])
@pytest.mark.parametrize("hk,group", [(2, 4), (1, 8)])
def test_prefix_ends(dev, prefix, hk, group):
    lens = [prefix + t for t in (1, 0, 15, 16, 17, 33, 64, 100)] + [0, 3, prefix - 1]
    check(dev, build(1, lens, prefix, hk, group), 8, sinks=group == 8)


@pytest.mark.parametrize("batch,hk,group", [(1, 2, 1), (1, 1, 4), (7, 2, 4), (8, 2, 4), (9, 1, 4), (16, 1, 4), (17, 1, 4),
                                            (33, 1, 4), (65, 2, 2), (11, 1, 12), (130, 1, 8)])
def test_row_counts(dev, batch, hk, group):
    lens = [208 + (37 * i) % 90 for i in range(batch)]
    check(dev, build(2, lens, 208, hk, group, dtype=torch.bfloat16), 16)


@pytest.mark.parametrize("preset", list(plain.PRESETS))
@pytest.mark.parametrize("layout", ["soa", "aos", "aos_heads"])
def test_presets_and_layouts(dev, preset, layout):
    for batch, group, bs in ((5, 4, 16), (20, 8, 64)):
        lens = [320 + (61 * i) % 200 for i in range(batch - 2)] + [0, 40]
        check(dev, build(3, lens, 320, 2, group, bs=bs, preset=preset, layout=layout), 8, sinks=batch == 5)


@pytest.mark.parametrize("bs", [16, 32, 64, 128])
@pytest.mark.parametrize("wide", [0, 300])
def test_blocks_and_table_widths(dev, bs, wide):
    check(dev, build(4, [1024, 1025, 1500, 2000, 0, 1023, 128], 1024, 4, 4, bs=bs, wide=wide), 16)


FORMS = {
    "a long prefix, many splits": ([12000] * 4 + [12001, 12040], 11984, 2, 4, 32),
    "long tails in parts": ([9000, 3000, 140, 128], 128, 4, 4, 32),
    "stretches over tails": ([128 + 29 * i for i in range(70)], 128, 2, 4, 32),
    "one row": ([3001, 2500], 1600, 2, 4, 1),
    "nobody has the prefix": ([0, 10, 100, 4], 128, 2, 4, 8),
    "the first to have it is the second": ([100, 128, 300, 0], 128, 2, 4, 8),
    "the first to have it is the last": ([i % 128 for i in range(69)] + [1000], 128, 2, 4, 8),
    "the first to have it opens the second 64": ([0] * 64 + [500, 128, 20], 128, 1, 2, 8),
    "batch past the device": ([64 + i % 9 for i in range(300)], 64, 2, 2, 4),
    "group of 16, three kv-heads": ([500, 333, 999], 320, 3, 16, 8),
}


@pytest.mark.parametrize("name", FORMS)
def test_forms(dev, name):
    lens, prefix, hk, group, splits = FORMS[name]
    check(dev, build(5, lens, prefix, hk, group), splits, sinks="parts" in name or "nobody" in name)


def test_every_prefix_length_gives_the_full_step(dev):
    """One table, several counts of shared blocks, 0 among them: the same rows up to f16 roundings."""
    c = build(6, [400, 401, 470, 399 + 64], 384, 4, 4, dtype=torch.bfloat16)
    for prefix in (0, 16, 64, 208, 384):
        c["prefix"] = prefix
        check(dev, c, 8)
    d = to_device(c, dev)
    out, lse = call(d, 8, prefix=0)
    full, full_lse = ops.full_decode(d["query"], d["rot"], d["cache"], d["table"], d["lens"], d["cents"], 8)
    assert torch.equal(out, full) and torch.equal(lse, full_lse)


@pytest.mark.parametrize("batch,prefix,hk,group,shares", [(8, 512, 2, 4, False), (2, 4096, 4, 4, False), (64, 4096, 8, 4, True),
                                                          (24, 12288, 8, 8, True)])
def test_auto_takes_one_of_the_two(dev, batch, prefix, hk, group, shares):
    """The rows of the sharing kernels where those pay, the full step's where they do not, bit for bit."""
    c = build(11, [prefix + 1 + (i * 13) % 60 for i in range(batch)], prefix, hk, group, dtype=torch.bfloat16)
    d = to_device(c, dev)
    out, lse = call(d, 16, kernel="auto")
    want, want_lse = call(d, 16, prefix=None if shares else 0)
    assert torch.equal(out, want) and torch.equal(lse, want_lse)


def test_large_small_and_zero_queries(dev):
    """Scores that span a hundred, nearly equal and equal ones, heads of every size in one batch."""
    scale = np.ones((3, 8))
    scale[0] = 10.0
    scale[1] = 0.0
    scale[2] = [1e-6, 1e-3, 0.1, 1, 3, 8, 1e-4, 0]
    check(dev, build(7, [500, 300, 700], 288, 2, 4, query_scale=scale), 8)
    check(dev, build(7, [500, 300, 700], 288, 2, 4, query_scale=scale, dtype=torch.bfloat16, preset="k8v4"), 8)


def test_a_row_of_nans_stays_a_row(dev):
    c = to_device(build(8, [200, 300, 210], 192, 2, 4), dev)
    clean, clean_lse = call(c, 8)
    c["query"][1, 2] = float("nan")
    out, lse = call(c, 8)
    keep = torch.ones(3, 8, dtype=torch.bool, device=dev)
    keep[1, 2] = False
    assert torch.equal(out[keep], clean[keep]) and torch.equal(lse[keep], clean_lse[keep])
    assert out[1, 2].isnan().all() and lse[1, 2].isnan()


def test_workspace_stream_and_graph(dev):
    c = to_device(build(9, [900, 513, 700, 512 + 300], 512, 4, 4, dtype=torch.bfloat16), dev)
    ws = ops.PrefixWorkspace(4, 16, 4, 16, dev, torch.bfloat16)
    want, want_lse = call(c, 16)
    side = torch.cuda.Stream()
    with torch.cuda.stream(side):
        side.wait_stream(torch.cuda.default_stream())
        out, lse = call(c, 16, workspace=ws)
    side.synchronize()
    assert out is ws.out and torch.equal(out, want) and torch.equal(lse, want_lse)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        call(c, 16, workspace=ws)
    for lens in ([900, 513, 700, 0], [513, 500, 520, 812], [512, 512, 2, 0], [899, 512, 0, 0]):
        c["lens"].copy_(torch.tensor(lens, dtype=torch.int32))
        ws.scratch.fill_(float("nan"))
        ws.out.zero_()
        graph.replay()
        torch.cuda.synchronize()
        got, got_lse = ws.out.clone(), ws.lse.clone()
        eager, eager_lse = call(c, 16)
        assert torch.equal(got.isnan(), eager.isnan()) and torch.equal(got[~got.isnan()], eager[~eager.isnan()])
        assert torch.equal(got_lse, eager_lse)
        assert [bool(r) for r in got.isnan().all(-1).all(-1)] == [n == 0 for n in lens]


@pytest.mark.parametrize("over,text", [
    (dict(prefix=8), "whole blocks"), (dict(prefix=1024), "whole blocks"), (dict(prefix=-16), "prefix_len"),
    (dict(prefix=True), "prefix_len"), (dict(kernel="simple"), "kernel"), (dict(out_dtype=torch.float32), "16-bit"), (dict(splits=5), "workspace"),
])
def test_refusals(dev, over, text):
    c = to_device(build(10, [60, 70], 32, 2, 4), dev)
    over = dict(over)
    ws = ops.PrefixWorkspace(2, 8, 2, 4, dev, torch.float16) if "splits" in over else None
    with pytest.raises(RuntimeError, match=text):
        call(c, over.pop("splits", 4), prefix=over.pop("prefix", 32), workspace=ws, **over)
    c["query"] = c["query"].float()
    with pytest.raises(RuntimeError, match="16-bit"):
        call(c, 4)


def test_c_entry_refuses(dev):
    lib, p = _lib.load(), 1 << 12
    need = lib.tq4_prefix_workspace_floats(2, 8, 2, 4)
    assert need > 0 and lib.tq4_prefix_workspace_floats(2, 7, 2, 4) == -1
    args = lambda **o: [o.get("query", p), 1, p, p, p, p, p, o.get("ws", p), o.get("floats", need), p, 1, p, 2, 8, 2, 128,  # noqa: E731
                        16, 4, 16 * 2 * 134, 4, 0, 0.1, None, o.get("kb", 4), 4, o.get("prefix", 32), 4, None]
    for o, code in ((dict(query=None), 1), (dict(ws=None), 1), (dict(floats=need - 1), 1), (dict(prefix=80), 1),
                    (dict(prefix=-1), 1), (dict(prefix=33), 1), (dict(kb=5), 2)):
        assert lib.tq4_prefix_decode(*args(**o)) == code, o
