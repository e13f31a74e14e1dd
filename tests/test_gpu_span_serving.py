"""The position-rotating writer and the windowed and shared-prefix steps as a server uses them together:
a prefix written once, ragged prompts behind it, then decode steps replayed from one captured graph (the
new token's queries and keys rotated, its key and value appended, one layer's step over all tokens and
one's over a window), with a padding sequence.  Then what any of them may meet in a cache: NaNs in every
token that is not visible, and block addresses past 4 GiB.

The reference is plain float64 attention over the values that the cache's bytes stand for, with the
queries that the writer returned.  Bars: the window's step 1e-4 plus half a step of the output type; the
shared prefix besides a rounding of each weight to f16 (2^-11 of sum p |v| at most); queries half a step
plus eight fp32 roundings of the rotation; stored values half a level and two f16 roundings of
scale and offset (2^-11 of 15 levels and of the offset each, counted twice)."""
import numpy as np
import pytest
import torch

import span_plain as plain
from test_gpu_rope_store import angles, axis_of, turn
from tq4_decode import codebook, ops

pytestmark = pytest.mark.gpu
D, BS = 128, 16
HALF_STEP = {torch.bfloat16: 2.0 ** -8, torch.float16: 2.0 ** -11}


def codes(kb, dev):
    if kb == 8:
        return None, None
    return (torch.from_numpy(codebook.centroids(D, kb)).to(dev), torch.from_numpy(codebook.midpoints(D, kb)).to(dev))


@pytest.mark.parametrize("preset,layout,dtype", [("4bit", "soa", torch.bfloat16), ("4bit", "aos", torch.float16),
                                                 ("k8v4", "aos_heads", torch.bfloat16), ("3bit", "soa", torch.float16)])
@pytest.mark.parametrize("kernel", ["auto", "shared"])
def test_prefill_then_replayed_decode_steps(dev, preset, layout, dtype, kernel):
    kb, vb = plain.PRESETS[preset]
    rng, gen = np.random.default_rng(1), torch.Generator().manual_seed(1)
    hk, group, prefix, window, first, splits = 2, 4, 64, 24, 3, 4
    hq = hk * group
    own = [0, 1, 15, 40, 70]  # and a padding sequence in the middle
    batch, width, steps, pad = 6, 12, 3, 2
    slot = plain.slot_bytes(kb, vb)
    pool = 1 + prefix // BS + (batch - 1) * 8
    if layout == "aos_heads":
        cache = torch.full((pool, hk, BS, slot), 0xFF, dtype=torch.uint8, device=dev).transpose(1, 2)
    else:
        cache = torch.full((pool, BS, hk, slot), 0xFF, dtype=torch.uint8, device=dev)
    ids = 1 + rng.permutation(pool - 1)
    seqs = [b for b in range(batch) if b != pad]
    table = np.zeros((batch, width), np.int32)
    for i, b in enumerate(seqs):
        table[b, :4] = ids[:4]
        table[b, 4:12] = ids[4 + 8 * i:12 + 8 * i]
    lens = np.zeros(batch, np.int64)
    lens[seqs] = [prefix + n for n in own]
    rot_t = plain.rotation(rng)
    put = lambda x: torch.from_numpy(np.ascontiguousarray(x)).to(dev)  # noqa: E731
    cents, mids = codes(kb, dev)
    cos_sin = angles(200, D).to(dev)
    rot = put(rot_t)
    rot_arg, nc = None if kb == 8 else rot, layout == "soa" and kb != 8
    kw = dict(key_bits=kb, value_bits=vb, layout="soa" if layout == "soa" else "aos")
    store_kw = dict(kw, norm_correction=nc)
    aux = (rot_arg, mids, cents if nc else None)
    tokens = {}  # (block, offset) -> (value rows, position)

    def write(qkv, positions, places, query=False, out=None, pos=None, slots=None):
        n = qkv.shape[0]
        q, k, v = (x.view(n, -1, D) for x in qkv.split([hq * D, hk * D, hk * D], 1))
        pos = put(np.asarray(positions, np.int64)) if pos is None else pos
        slots = put(np.array([b * BS + o if b >= 0 else -1 for b, o in places], np.int32)) if slots is None else slots
        return ops.rope_store(q if query else None, k, v, pos, cos_sin, cache, slots, *aux, query_out=out, **store_kw)

    def remember(qkv, places):
        for i, at in enumerate(places):
            if at[0] >= 0:
                tokens[at] = qkv[i, (hq + hk) * D:].double().cpu().numpy().reshape(hk, D)

    fresh = lambda n: torch.randn(n, (hq + 2 * hk) * D, generator=gen).to(dtype)  # noqa: E731
    place = lambda b, t: (int(table[b, t // BS]), int(t % BS))  # noqa: E731
    qkv, places = fresh(prefix).to(dev), [place(seqs[0], t) for t in range(prefix)]
    assert write(qkv, range(prefix), places) is None
    remember(qkv, places)
    at = [(b, prefix + t) for b, n in zip(seqs, own) for t in range(n)]
    qkv, places = fresh(len(at)).to(dev), [place(b, t) for b, t in at]
    write(qkv, [t for _, t in at], places)
    remember(qkv, places)

    static = dict(qkv=torch.zeros(batch, (hq + 2 * hk) * D, dtype=dtype, device=dev),
                  pos=torch.zeros(batch, dtype=torch.int64, device=dev),
                  slots=torch.full((batch,), -1, dtype=torch.int32, device=dev),
                  lens=torch.zeros(batch, dtype=torch.int32, device=dev))
    dev_table, q_out = put(table), torch.empty(batch, hq, D, dtype=dtype, device=dev)
    whole = ops.PrefixWorkspace(batch, hq, hk, splits, dev, dtype)
    local = ops.DecodeWorkspace(batch, hq, splits, dev, dtype)

    def step():
        write(static["qkv"], None, None, True, q_out, static["pos"], static["slots"])
        ops.prefix_decode(q_out, rot_arg, cache, dev_table, static["lens"], cents, splits, prefix, workspace=whole,
                          kernel=kernel, **kw)
        ops.window_decode(q_out, rot_arg, cache, dev_table, static["lens"], cents, splits, window, first_tokens=first,
                          workspace=local, **kw)

    step()  # (padding alone: nothing written)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        step()
    for _ in range(steps):
        lens[seqs] += 1
        qkv = fresh(batch)
        places = [place(b, lens[b] - 1) if lens[b] else (-1, 0) for b in range(batch)]
        static["qkv"].copy_(qkv)
        static["pos"].copy_(torch.from_numpy(np.maximum(lens - 1, 0)))
        static["slots"].copy_(torch.tensor([b * BS + o if b >= 0 else -1 for b, o in places], dtype=torch.int32))
        static["lens"].copy_(torch.from_numpy(lens.astype(np.int32)))
        graph.replay()
        torch.cuda.synchronize()
        remember(qkv, places)

        q_in = qkv[:, :hq * D].double().numpy().reshape(batch, hq, D)
        want_q, size = turn(q_in, np.maximum(lens - 1, 0), cos_sin.double().cpu().numpy(), True, axis_of(64, None, False))
        got_q = q_out.double().cpu().numpy()
        assert (np.abs(got_q - want_q) <= HALF_STEP[dtype] * np.abs(want_q) + 8 * 2.0 ** -24 * size + 2.0 ** -25).all()

        kc, vc, fields = plain.split_cache(cache.cpu().numpy(), kb, vb, layout)
        with np.errstate(invalid="ignore"):
            k, v = plain.values_of(kc, vc, fields, kb, layout)
        for (block, off), value in tokens.items():
            level, low = (x[block, off].astype(np.float64)[:, None] for x in fields[-2:])
            assert (np.abs(v[block, off] - value) <= level * (0.5 + 30 * 2.0 ** -11) + 2 * 2.0 ** -11 * np.abs(low) + 1e-6).all()
        q = got_q if kb == 8 else got_q @ rot_t.astype(np.float64)
        for b in range(batch):
            t = np.arange(lens[b])
            kk, vv = k[table[b, t // BS], t % BS], v[table[b, t // BS], t % BS]
            o, lse = plain.attend(q[b], kk, vv)
            spread = plain.attend(q[b], kk, np.abs(vv))[0]
            seen = (t < first) | (t >= lens[b] - window)
            o_w, lse_w = plain.attend(q[b], kk[seen], vv[seen])
            step16 = HALF_STEP[dtype]
            plain.close(local.out[b].double().cpu().numpy(), o_w, step16, "window")
            plain.close(local.lse[b].cpu().numpy(), lse_w, 0.0, "window lse")
            got = whole.out[b].double().cpu().numpy()
            if lens[b] == 0:
                assert np.isnan(got).all() and np.isneginf(whole.lse[b].cpu().numpy()).all()
                continue
            assert (np.abs(got - o) <= 1e-4 + step16 * np.abs(o) + 2.0 ** -11 * spread).all()
            plain.close(whole.lse[b].cpu().numpy(), lse, 0.0, "lse")
    unused = [p for p in range(pool) if all((p, o) not in tokens for o in range(BS))]
    assert (cache[unused] == 0xFF).all()


@pytest.mark.parametrize("preset", list(plain.PRESETS))
@pytest.mark.parametrize("layout", ["soa", "aos"])
def test_nans_in_tokens_that_are_not_visible(dev, preset, layout):
    kb, vb = plain.PRESETS[preset]
    rng = np.random.default_rng(2)
    hk, hq, prefix, window, first = 2, 8, 32, 21, 5
    lens = [33, 64, 70, 101, 32]
    shared, most = prefix // BS, 7
    cache, k, v = plain.make_cache(rng, 1 + shared + len(lens) * (most - shared), BS, hk, preset, layout)
    ids = 1 + rng.permutation(cache.size(0) - 1)
    table = np.zeros((len(lens), most), np.int32)
    for b in range(len(lens)):
        table[b] = np.concatenate([ids[:shared], ids[shared + b * (most - shared):][:most - shared]])
    rot_t = plain.rotation(rng)
    query = torch.from_numpy(rng.standard_normal((len(lens), hq, D)).astype(np.float32)).to(torch.float16)
    q = query.double().numpy() if kb == 8 else query.double().numpy() @ rot_t.astype(np.float64)
    put = lambda x: torch.from_numpy(np.ascontiguousarray(x)).to(dev)  # noqa: E731
    cents, _ = codes(kb, dev)
    args = lambda c: (query.to(dev), None if kb == 8 else put(rot_t), c.to(dev), put(table),  # noqa: E731
                      torch.tensor(lens, dtype=torch.int32, device=dev), cents, 4)
    kw = dict(key_bits=kb, value_bits=vb, layout=layout)
    at = lambda b, t: (int(table[b, t // BS]), int(t % BS))  # noqa: E731
    behind = {at(b, t) for b, n in enumerate(lens) for t in range(n, most * BS)}
    past = cache.clone()
    plain.spoil(past, behind, preset, layout)
    out, lse = ops.prefix_decode(*args(past), prefix, kernel="shared", **kw)
    for b, n in enumerate(lens):
        t = np.arange(n)
        kk, vv = k[table[b, t // BS], t % BS], v[table[b, t // BS], t % BS]
        o, l = plain.attend(q[b], kk, vv)
        spread = plain.attend(q[b], kk, np.abs(vv))[0]
        got = out[b].double().cpu().numpy()
        assert (np.abs(got - o) <= 1e-4 + 2.0 ** -11 * np.abs(o) + 2.0 ** -11 * spread).all()
        plain.close(lse[b].cpu().numpy(), l, 0.0, "lse")
    for b, n in enumerate(lens):  # each alone: the others see what it must not
        hidden = {at(b, t) for t in range(n) if first <= t < n - window}
        spoilt = cache.clone()
        plain.spoil(spoilt, behind | hidden, preset, layout)
        out, lse = ops.window_decode(*args(spoilt), window, first_tokens=first, **kw)
        t = np.array([t for t in range(n) if t < first or t >= n - window])
        o, l = plain.attend(q[b], k[table[b, t // BS], t % BS], v[table[b, t // BS], t % BS])
        plain.close(out[b].double().cpu().numpy(), o, 2.0 ** -11, "out")
        plain.close(lse[b].cpu().numpy(), l, 0.0, "lse")


@pytest.mark.parametrize("preset,layout", [("4bit", "soa"), ("4bit", "aos"), ("k8v4", "soa"), ("3bit", "soa")])
def test_blocks_past_4_gib(dev, preset, layout):
    """The same blocks in a small cache and at the end of one of more than 2^32 bytes: the same bytes written, the
    same rows read, nothing else touched."""
    kb, vb = plain.PRESETS[preset]
    rng = np.random.default_rng(3)
    hk, hq, n, prefix = 8, 32, 300, 64
    slot = plain.slot_bytes(kb, vb)
    few, blocks = 24, (1 << 32) // (BS * hk * slot) + 100
    qkv = torch.randn(n, (hq + 2 * hk) * D, generator=torch.Generator().manual_seed(3)).to(torch.bfloat16).to(dev)
    q, k, v = (x.view(n, -1, D) for x in qkv.split([hq * D, hk * D, hk * D], 1))
    put = lambda x: torch.from_numpy(np.ascontiguousarray(x)).to(dev)  # noqa: E731
    cents, mids = codes(kb, dev)
    rot = None if kb == 8 else put(plain.rotation(rng))
    order = np.arange(n)  # token t of the one sequence in block order[t // BS]
    table = rng.permutation(few)[:-(-n // BS)].astype(np.int32)
    kw = dict(key_bits=kb, value_bits=vb, layout=layout)
    nc = layout == "soa" and kb != 8
    cos_sin, pos = angles(n, D).to(dev), torch.arange(n, device=dev)
    seen = []
    for total, base in ((few, 0), (blocks, blocks - few)):
        cache = torch.zeros((total, BS, hk, slot), dtype=torch.uint8, device=dev)
        rows = (table.astype(np.int64) + base)
        slots = (rows[order // BS] * BS + order % BS).astype(np.int32)
        ops.rope_store(None, k, v, pos, cos_sin, cache, put(slots), rot, mids, cents if nc else None,
                       norm_correction=nc, **kw)
        args = (q[-2:].contiguous(), rot, cache, put(np.stack([rows, rows]).astype(np.int32)),
                torch.tensor([n, n - 70], dtype=torch.int32, device=dev), cents, 4)
        got = [cache[base:].clone(), *ops.window_decode(*args, 100, first_tokens=20, **kw),
               *ops.prefix_decode(*args, prefix, kernel="shared", **kw)]
        assert not cache[:base].any()
        assert all(not x.isnan().any() for x in got[1:])
        seen.append(got)
        del cache
    assert all(torch.equal(a, b) for a, b in zip(*seen))
