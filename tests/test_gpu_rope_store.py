"""Rotary positions and the cache writer in one call (``ops.rope_store``) against the definition in float64.

Bar: the cache's bytes are those of the definition (codes, E4M3 bytes and fp16 scalars; V's in the writer's own
fp32 operations), and every other byte stays; rotated queries half a step of their type and 2^-22 of the
plane's size off (fp32: two roundings of products, one of the sum).  Below a type's normal range its
step no longer shrinks with the value: fp16 values under 2^-14 are 2^-24 apart, so half a step is 2^-25
there whatever the value (bf16 and fp32: 2^-134 and 2^-150)."""
import ctypes

import numpy as np
import pytest
import torch

import span_plain as plain
from tq4_decode import _lib, codebook, ops

pytestmark = pytest.mark.gpu
D = 128
TYPES = {"bf16": torch.bfloat16, "fp16": torch.float16, "fp32": torch.float32}
HALF_STEP = {"bf16": 2.0 ** -8, "fp16": 2.0 ** -11, "fp32": 2.0 ** -24}
LEAST = {"bf16": 2.0 ** -134, "fp16": 2.0 ** -25, "fp32": 2.0 ** -150}


def angles(rows, rot, dtype=torch.float32, base=1e4):
    a = np.arange(rows)[:, None] * base ** (-np.arange(rot // 2) * 2.0 / rot)
    return torch.from_numpy(np.concatenate([np.cos(a), np.sin(a)], 1)).to(dtype)


def axis_of(half, sections, in_turn):
    if sections is None:
        return np.zeros(half, int)
    if not in_turn:
        return np.repeat(np.arange(len(sections)), sections)
    n = len(sections)
    return np.array([j % n if j % n and j < n * sections[j % n] else 0 for j in range(half)])


def turn(x, positions, table, neox, axes):
    """x [N, H, 128] float64 rotated; the size of each element's plane."""
    rot, half = table.shape[1], table.shape[1] // 2
    pos = positions.reshape(-1, x.shape[0])[axes].T  # [N, half]
    f = np.arange(half)
    c, s = table[pos, f][:, None], table[pos, half + f][:, None]
    i0, i1 = (f, f + half) if neox else (2 * f, 2 * f + 1)
    out, size = x.copy(), np.abs(x)
    a, b = x[..., i0], x[..., i1]
    out[..., i0], out[..., i1] = a * c - b * s, b * c + a * s
    size[..., i0] = size[..., i1] = np.abs(a) + np.abs(b)
    return out, size


def expected(cache, key, value, slots, rot_t, mids, cents, kb, vb, layout, nc):
    """The cache's bytes [blocks, bs, hk, slot] (SoA: of the block's bytes) after the call; key already rotated."""
    cache = cache.copy()
    n_blocks, bs, hk, slot = cache.shape
    fields = []
    if kb == 8:
        k32 = torch.from_numpy(key).float().clamp(-448, 448)
        kc = k32.to(torch.float8_e4m3fn).view(torch.uint8).numpy()
    else:
        norm = np.sqrt((key ** 2).sum(-1))
        y = (key / (norm[..., None] + 1e-8)) @ rot_t.astype(np.float64)
        kc = np.searchsorted(mids.astype(np.float64), y, side="right")
        if nc:
            norm = norm / np.sqrt((cents.astype(np.float64)[kc] ** 2).sum(-1) + 1e-16)
        fields.append(norm.astype(np.float32).astype(np.float16))
    top = (1 << vb) - 1
    v = value.astype(np.float32)
    zero = v.min(-1)
    scale = np.maximum((v.max(-1) - zero) / np.float32(top), np.float32(1e-8))
    vc = np.clip(((v - zero[..., None]) / scale[..., None] + np.float32(0.5)).astype(np.int64), 0, top)
    fields += [scale.astype(np.float16), zero.astype(np.float16)]
    kby, vby = plain.pack(kc, kb), plain.pack(vc, vb)
    live = (slots >= 0) & (slots < n_blocks * bs)
    blk, off = slots[live] // bs, slots[live] % bs
    if layout == "soa":
        rec = kby.shape[-1] + vby.shape[-1]
        flat = cache.reshape(n_blocks, -1)
        data = flat[:, :bs * hk * rec].reshape(n_blocks, bs, hk, rec).copy()
        meta = flat[:, bs * hk * rec:].copy().view(np.float16).reshape(n_blocks, hk, len(fields), bs)
        data[blk, off] = np.concatenate([kby, vby], -1)[live]
        for i, f in enumerate(fields):
            meta[blk, :, i, off] = f[live]
        flat[:, :bs * hk * rec] = data.reshape(n_blocks, -1)
        flat[:, bs * hk * rec:] = meta.reshape(n_blocks, -1).view(np.uint8)
        return flat.reshape(cache.shape)
    cells = [np.ascontiguousarray(f[..., None]).view(np.uint8) for f in fields]
    cache[blk, off] = np.concatenate([kby] + cells[:-2] + [vby] + cells[-2:], -1)[live]
    return cache


def build(seed, n, hq, hk, preset="4bit", layout="soa", dtype="bf16", bs=16, rot=D, neox=True, sections=None,
          in_turn=False, table="fp32", fused=True, rows=600):
    rng = np.random.default_rng(seed)
    gen = torch.Generator().manual_seed(seed)
    kb, vb = plain.PRESETS[preset]
    t = TYPES[dtype]
    qkv = torch.randn(n, (hq + 2 * hk) * D, generator=gen)
    qkv[:, hq * D:(hq + hk) * D] *= torch.rand(n, 1, generator=gen) * 3
    qkv = qkv.to(t)
    q, k, v = (x.view(n, -1, D) for x in qkv.split([hq * D, hk * D, hk * D], 1))
    if not fused:
        q, k, v = q.contiguous(), k.contiguous(), v.contiguous()
    blocks = n // bs + 3
    slots = rng.permutation(blocks * bs)[:n].astype(np.int32)
    slots[rng.random(n) < 0.1] = -1
    axes = 1 if sections is None else len(sections)
    positions = torch.from_numpy(rng.integers(0, rows, (axes, n)))
    shape = (blocks, hk, bs) if layout == "aos_heads" else (blocks, bs, hk)
    cache = torch.full(shape + (plain.slot_bytes(kb, vb),), 0xA5, dtype=torch.uint8)
    cents = codebook.centroids(D, kb) if kb != 8 else None
    mids = codebook.midpoints(D, kb) if kb != 8 else None
    return dict(q=q, k=k, v=v, positions=positions if axes > 1 else positions[0], cache=cache, slots=slots,
                table=angles(rows, rot, torch.float32 if table == "fp32" else t), rot_t=plain.rotation(rng), cents=cents,
                mids=mids, kb=kb, vb=vb, layout=layout, neox=neox, sections=sections, in_turn=in_turn, dtype=dtype)


def call(c, dev, **over):
    """The call on `dev`; returns (queries, cache bytes [blocks, bs, hk, slot])."""
    put = lambda x: torch.from_numpy(x).to(dev) if x is not None else None  # noqa: E731
    qkv = [x if x is None else x.to(dev) if x.is_contiguous() else
           x._base.to(dev).as_strided(x.shape, x.stride(), x.storage_offset()) for x in (c["q"], c["k"], c["v"])]
    cache = c["cache"].to(dev)
    view = cache.transpose(1, 2) if c["layout"] == "aos_heads" else cache
    nc = c["layout"] == "soa" and c["kb"] != 8
    kw = dict(key_bits=c["kb"], value_bits=c["vb"], layout="soa" if c["layout"] == "soa" else "aos", norm_correction=nc,
              neox=c["neox"], sections=c["sections"], in_turn=c["in_turn"])
    kw.update(over)
    out = ops.rope_store(qkv[0], qkv[1], qkv[2], c["positions"].to(dev), c["table"].to(dev), view, put(c["slots"]),
                         put(c["rot_t"]) if c["kb"] != 8 else None, put(c["mids"]), put(c["cents"]) if nc else None, **kw)
    torch.cuda.synchronize()
    return out, view.cpu().numpy()


def check(dev, c, **over):
    out, got = call(c, dev, **over)
    axes = axis_of(c["table"].shape[1] // 2, c["sections"], c["in_turn"])
    pos, table = c["positions"].numpy(), c["table"].double().numpy()
    key, _ = turn(c["k"].double().numpy(), pos, table, c["neox"], axes)
    before = c["cache"].transpose(1, 2).numpy() if c["layout"] == "aos_heads" else c["cache"].numpy()
    want = expected(np.ascontiguousarray(before), key, c["v"].float().numpy(), c["slots"], c["rot_t"], c["mids"], c["cents"],
                    c["kb"], c["vb"], c["layout"], c["layout"] == "soa" and c["kb"] != 8)
    bad = np.argwhere(got != want)
    assert bad.size == 0, f"{len(bad)} of {want.size} bytes differ, first at {bad[0]}"
    if c["q"] is not None:
        q, size = turn(c["q"].double().numpy(), pos, table, c["neox"], axes)
        err = np.abs(out.double().cpu().numpy() - q) - HALF_STEP[c["dtype"]] * np.abs(q) - 2.0 ** -22 * size
        assert err.max() <= LEAST[c["dtype"]], f"queries off by {err.max():.2e}"


@pytest.mark.parametrize("preset", list(plain.PRESETS))
@pytest.mark.parametrize("layout", ["soa", "aos", "aos_heads"])
@pytest.mark.parametrize("dtype", ["bf16", "fp16", "fp32"])
def test_presets_layouts_types(dev, preset, layout, dtype):
    check(dev, build(1, 130, 8, 2, preset, layout, dtype, bs=32))


@pytest.mark.parametrize("rot", [16, 32, 64, 96, 128])
@pytest.mark.parametrize("neox", [True, False])
@pytest.mark.parametrize("preset", ["4bit", "k8v4"])
def test_rotated_dims(dev, rot, neox, preset):
    check(dev, build(2, 70, 4, 2, preset, rot=rot, neox=neox, table="same" if rot == 64 else "fp32"))


def test_one_axis_in_turn(dev):
    """Frequencies dealt round a single axis: the plain positions."""
    check(dev, build(3, 90, 4, 2, "4bit", in_turn=True))


@pytest.mark.parametrize("sections,in_turn", [((16, 24, 24), False), ((24, 20, 20), True), ((64, 0, 0), False), ((0, 33, 31), False),
                                              ((50, 14), False), ((10, 20, 30, 4), False), ((61, 1, 2), True), ((32, 32), True),
                                              ((22, 10, 16, 16), True)])
@pytest.mark.parametrize("neox", [True, False])
def test_axes(dev, sections, in_turn, neox):
    for preset in ("4bit", "k8v4"):
        check(dev, build(3, 90, 4, 2, preset, neox=neox, sections=sections, in_turn=in_turn))


@pytest.mark.parametrize("n,hq,hk", [(1, 1, 1), (1, 32, 8), (2, 7, 1), (3, 5, 5), (16, 8, 8), (17, 6, 3), (65, 16, 1), (33, 48, 6)])
def test_shapes(dev, n, hq, hk):
    check(dev, build(4, n, hq, hk))
    check(dev, build(4, n, hq, hk, fused=False, dtype="fp16"))


@pytest.mark.parametrize("preset,dtype", [("4bit", "bf16"), ("3bit", "fp16"), ("k8v4", "bf16"), ("k3v4", "fp32")])
def test_many_tokens(dev, preset, dtype):
    """Past the small launches' 1024 tiles, several tiles per wave: 160 000 rows, a few hundred next to a border."""
    check(dev, build(5, 20011, 3, 8, preset, dtype=dtype))


@pytest.mark.parametrize("n,preset,dtype,layout", [(9001, "4bit", "bf16", "soa"), (9001, "3bit", "fp32", "aos"),
                                                   (5000, "4bit", "fp16", "aos_heads"), (5000, "k8v4", "bf16", "soa")])
def test_many_tokens_on_several_axes(dev, n, preset, dtype, layout):
    """Both sides of the size from which the queries have a launch of their own; and the writer alone."""
    c = build(15, n, 2, 8, preset, layout=layout, dtype=dtype, sections=(16, 24, 24), in_turn=False)
    check(dev, c)
    _, want = call(c, dev)
    c["q"] = None
    out, got = call(c, dev)
    assert out is None and np.array_equal(got, want)


def test_query_out_among_the_inputs(dev):
    c = build(16, 20, 4, 2)
    q, k, v = (c[n].to(dev) for n in "qkv")
    qkv = torch.cat([x.reshape(20, -1) for x in (q, k, v)], 1)
    parts = [x.view(20, -1, D) for x in qkv.split([4 * D, 2 * D, 2 * D], 1)]
    put = lambda x: torch.from_numpy(x).to(dev)  # noqa: E731
    rest = (c["positions"].to(dev), c["table"].to(dev), c["cache"].to(dev), put(c["slots"]), put(c["rot_t"]), put(c["mids"]),
            put(c["cents"]))
    before = qkv.clone()
    for out in (qkv.view(-1)[:20 * 4 * D].view(20, 4, D), qkv.view(-1)[64:64 + 20 * 4 * D].view(20, 4, D)):
        with pytest.raises(RuntimeError, match="query_out"):
            ops.rope_store(*parts, *rest, query_out=out)
    with pytest.raises(RuntimeError, match="query_out"):
        ops.rope_store(q, k, v, *rest, query_out=torch.cat([k, v], 1)[:, :, :].contiguous()[:19])
    assert torch.equal(qkv, before)
    beside = torch.empty(2, 20, 4, D, dtype=q.dtype, device=dev)
    beside[0].copy_(q)
    got = ops.rope_store(beside[0], k, v, *rest, query_out=beside[1])
    assert torch.equal(got, ops.rope_store(*parts, *rest)) and torch.equal(beside[0], q)


@pytest.mark.parametrize("preset", ["4bit", "k3v4"])
def test_elements_next_to_midpoints(dev, preset):
    """Keys whose rotated direction lies on midpoints up to the type's own rounding: every row has elements that
    the fp32-grade path alone would leave to chance."""
    c = build(6, 40, 2, 2, preset, dtype="fp32", rows=50)
    rng = np.random.default_rng(7)
    y = c["mids"].astype(np.float64)[rng.integers(0, len(c["mids"]), (40, 2, D))]
    y[..., 64:] = rng.normal(0, D ** -0.5, (40, 2, 64))
    y /= np.sqrt((y ** 2).sum(-1, keepdims=True))
    for _ in range(30):  # the first half on midpoints, the whole of norm 1
        near = c["mids"].astype(np.float64)[np.abs(y[..., :64, None] - c["mids"]).argmin(-1)]
        y[..., :64] = near
        rest = 1 - (near ** 2).sum(-1, keepdims=True)
        assert (rest > 0).all()
        y[..., 64:] *= np.sqrt(rest / (y[..., 64:] ** 2).sum(-1, keepdims=True))
    rotated = y @ np.linalg.inv(c["rot_t"].astype(np.float64))
    axes = axis_of(64, None, False)
    back = c["table"].double().numpy().copy()
    back[:, 64:] *= -1
    k, _ = turn(rotated * 9.0, c["positions"].numpy(), back, True, axes)
    c["k"] = torch.from_numpy(k.astype(np.float32))
    check(dev, c)


def test_zero_rows_and_constant_values(dev):
    c = build(8, 50, 2, 4, dtype="fp16", fused=False)
    c["k"][3] = 0
    c["k"][7, 1] = 0
    c["k"][9, 0, 5:] = 0
    c["v"][11] = 1.5
    c["v"][12] = 0
    check(dev, c)


def test_large_and_small_norms(dev):
    c = build(9, 60, 2, 2, dtype="fp32", fused=False)
    c["k"] *= torch.logspace(-6, 4, 60)[:, None, None]
    check(dev, c)


def test_tokens_without_a_place(dev):
    """Slots past the cache and negative ones, positions outside the table: nothing written, NaN queries for the last."""
    c = build(10, 40, 4, 2)
    c["slots"][:4] = [-5, c["cache"].size(0) * 16, 2 ** 31 - 1, -2 ** 31]
    bad = torch.tensor([600, -1, 2 ** 40, -2 ** 40])
    inside = c["positions"].clone()
    c["positions"][4:8] = bad
    out, got = call(c, dev)
    nan = out.isnan().all(-1).all(-1).cpu()
    assert nan[4:8].all() and not out[:4].isnan().any() and not out[8:].isnan().any()
    slots = c["slots"].copy()
    c["slots"][4:8] = -1
    c["positions"] = inside
    _, want = call(c, dev)
    assert np.array_equal(got, want)
    c["slots"] = slots
    # one bad axis of three is enough
    c = build(10, 40, 4, 2, sections=(16, 24, 24))
    c["positions"][2, 5] = 600
    out, _ = call(c, dev)
    assert out[5].isnan().all() and out.isnan().any(-1).any(-1).sum() == 1


def test_queries_in_place_and_no_queries(dev):
    c = build(11, 77, 6, 2, fused=False)
    want, cache = call(c, dev)
    q = c["q"].to(dev)
    keep = c["q"]
    c["q"] = q
    got, cache2 = call(c, dev, query_out=q)
    assert got is q and torch.equal(got, want) and np.array_equal(cache, cache2)
    c["q"] = None
    none, cache3 = call(c, dev)
    assert none is None and np.array_equal(cache, cache3)
    c["q"] = keep
    c0 = build(11, 77, 6, 2)
    for n in ("q", "k", "v"):
        c0[n] = c0[n][:0].contiguous()
    c0["slots"], c0["positions"] = c0["slots"][:0], c0["positions"][:0]
    out, untouched = call(c0, dev)
    assert out.shape == (0, 6, D) and (untouched == 0xA5).all()


def test_stream_and_graph(dev):
    c = build(12, 64, 8, 2, sections=(16, 24, 24))
    want, cache = call(c, dev)
    put = lambda x: torch.from_numpy(x).to(dev)  # noqa: E731
    q, k, v = (c[n].contiguous().to(dev) for n in "qkv")
    pos, table, slots = c["positions"].to(dev), c["table"].to(dev), put(c["slots"])
    rot, mids, cents = put(c["rot_t"]), put(c["mids"]), put(c["cents"])
    out, mem = torch.empty_like(q), c["cache"].to(dev)
    args = (q, k, v, pos, table, mem, slots, rot, mids, cents)
    kw = dict(sections=(16, 24, 24), query_out=out)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        ops.rope_store(*args, **kw)
    side.synchronize()
    assert torch.equal(out, want) and np.array_equal(mem.cpu().numpy(), cache)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        ops.rope_store(*args, **kw)
    for i in range(3):
        pos.copy_(torch.randint(0, 600, pos.shape))
        k.copy_(torch.randn(k.shape).to(k.dtype))
        mem.fill_(0x5A)
        graph.replay()
        torch.cuda.synchronize()
        eager = torch.full_like(mem, 0x5A)
        want = ops.rope_store(*args[:5], eager, *args[6:], sections=(16, 24, 24))
        assert torch.equal(mem, eager) and torch.equal(out, want)


def test_the_writers_bytes_without_rotation(dev):
    """Angle 0 everywhere: the writer's own call differs at most where the definition is next to a border."""
    c = build(13, 500, 1, 8, dtype="bf16", fused=False)
    c["table"][:, :64], c["table"][:, 64:] = 1.0, 0.0
    _, got = call(c, dev)
    cache = c["cache"].to(dev)
    put = lambda x: torch.from_numpy(x).to(dev)  # noqa: E731
    ops.store(c["k"].to(dev), c["v"].to(dev), cache, put(c["slots"]), put(c["rot_t"]), put(c["mids"]), put(c["cents"]))
    same = (cache.cpu().numpy() == got).mean()
    assert same > 0.999


REFUSED = [
    (dict(key_bits=5), "key/value bits"), (dict(sections=(10, 20)), "sections"), (dict(sections=(64,)), "sections"),
    (dict(sections=(0, 40, 24), in_turn=True), "sections in turn"), (dict(layout="x"), "layout"),
    (dict(query_out="short"), "query_out"), (dict(cents=False), "centroids"), (dict(table=72), "rot_dim"),
    (dict(table=144), "rot_dim"), (dict(stride=4), "16-byte"), (dict(positions=torch.int32), "int64"),
    (dict(heads=3), "heads"),
]


@pytest.mark.parametrize("over,text", REFUSED)
def test_refusals(dev, over, text):
    over = dict(over)
    c = build(14, 8, 2, 2, fused=False)
    q, k, v = (c[n].to(dev) for n in "qkv")
    put = lambda x: torch.from_numpy(x).to(dev)  # noqa: E731
    table, pos, cents = c["table"].to(dev), c["positions"].to(dev), put(c["cents"])
    if "query_out" in over:
        over["query_out"] = q[:4]
    if over.pop("cents", None) is False:
        cents = None
    if "table" in over:
        table = torch.zeros(10, over.pop("table"), device=dev)
    if "positions" in over:
        pos = pos.to(over.pop("positions"))
    if "stride" in over:
        n = over.pop("stride")
        k = torch.zeros(8, 2 * D + n, dtype=k.dtype, device=dev)[:, :2 * D].view(8, 2, D)
    if "heads" in over:
        v = torch.zeros(8, over.pop("heads"), D, dtype=v.dtype, device=dev)
    if "sections" in over and over["sections"] != (10, 20) and len(over["sections"]) == 3:
        pos = pos.expand(3, 8)
    with pytest.raises(RuntimeError, match=text):
        ops.rope_store(q, k, v, pos, table, c["cache"].to(dev), put(c["slots"]), put(c["rot_t"]), put(c["mids"]), cents, **over)


def test_c_entry_refuses(dev):
    lib, p = _lib.load(), 1 << 12
    ax = (ctypes.c_int32 * 64)(*([0] * 63 + [3]))

    def args(**o):
        d = dict(q=p, qo=p, k=p, v=p, dt=1, qs=256, ks=256, vs=256, pos=p, ast=0, axes=1, ax=None, cs=p, cdt=0, rows=10, rot=128, neox=1,
                 sl=p, rt=p, mid=p, cen=p, cache=p, nb=4, N=4, Hq=2, Hk=2, D=128, bs=16, stride=16 * 2 * 134, lay=0, nc=1, kb=4,
                 vb=4, st=None)
        d.update(o)
        return list(d.values())

    for o, code in ((dict(k=None), 1), (dict(qo=None), 1), (dict(q=None), 1), (dict(dt=3), 1), (dict(cdt=2), 1), (dict(rot=24), 2),
                    (dict(rot=0), 2), (dict(D=64), 2), (dict(axes=5), 1), (dict(axes=2), 1), (dict(axes=3, ax=ax), 1),
                    (dict(ks=255), 1), (dict(ks=-256), 1), (dict(stride=100), 1), (dict(lay=4), 1), (dict(cen=None), 1), (dict(kb=6), 2),
                    (dict(N=-1), 1), (dict(rows=0), 1), (dict(cache=p + 4), 1), (dict(N=2 ** 30, Hk=4, stride=16 * 4 * 134), 1),
                    (dict(N=0), 0)):
        assert lib.tq4_rope_store(*args(**o)) == code, o
