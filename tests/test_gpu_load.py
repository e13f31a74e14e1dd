"""Keys and values read back from the cache (``ops.cache_load``) against the codes' values in float64, and two
attention results joined (``ops.merge_states``).

Bars.  Values: one rounding (half a step of the type).  Keys as stored: the product with the norm, one fp32 rounding more,
and for AoS slots the norm's own division and root (four roundings).  Keys turned back, fp16 and fp32: factors
as f16 pairs, 2^-22 of each, and an fp32 sum of 384 products: 2^-21 + 384 2^-24 < 2^-15 of the sum of magnitudes; bf16:
eight standard deviations of rounding both factors to f16 (deviation 2^-11 / sqrt 3 of each) besides."""
import numpy as np
import pytest
import torch

import span_plain as plain
from tq4_decode import codebook, ops, workloads  # noqa: F401

pytestmark = pytest.mark.gpu
D = 128
HALF_STEP = {torch.float32: 2.0 ** -24, torch.bfloat16: 2.0 ** -8, torch.float16: 2.0 ** -11}
RHO = 2.0 ** -11 / 3 ** 0.5
TYPES = pytest.mark.parametrize("dtype", list(HALF_STEP), ids=["fp32", "bf16", "fp16"])


def expect(k, v, rot, kb, layout, dtype):
    """(key, its bar, value, its bar) of rows k, v in float64."""
    step = HALF_STEP[dtype]
    small = 2.0 ** -24 if dtype == torch.float16 else 2.0 ** -126
    if rot is None or kb == 8:
        bar = (step + (0 if kb == 8 else 2.0 ** -24) + (0 if layout == "soa" or kb == 8 else 2.0 ** -22)) * np.abs(k)
    else:
        r = rot.astype(np.float64)
        err = 2.0 ** -15 * (np.abs(k) @ np.abs(r.T))
        if dtype == torch.bfloat16:
            err = err + 8 * np.sqrt(2) * RHO * np.sqrt(k ** 2 @ (r.T) ** 2)
        k = k @ r.T
        bar = step * np.abs(k) + err
    # (for fp32 a value's fma is its only rounding; others round that once more)
    return k, bar + small, v, (step + (0 if dtype == torch.float32 else 2.0 ** -24)) * np.abs(v) + small


def device_cache(cache, layout, dev):
    return cache.transpose(1, 2).contiguous().to(dev).transpose(1, 2) if layout == "aos_heads" else cache.to(dev)


def load(cache, layout, slots, rot, kb, vb, dtype, dev, **more):
    to = lambda x: torch.from_numpy(np.ascontiguousarray(x)).to(dev)  # noqa: E731
    cents = None if kb == 8 else to(codebook.centroids(D, kb).astype(np.float32))
    return ops.cache_load(device_cache(cache, layout, dev), to(np.asarray(slots, np.int32)),
                          None if rot is None or kb == 8 else to(rot), cents, key_bits=kb, value_bits=vb,
                          layout="soa" if layout == "soa" else "aos", dtype=dtype, **more)


def compare(got, want, bar, what):
    over = np.abs(got.double().cpu().numpy() - want) - bar
    assert over.max() <= 0, f"{what}: {over.max():.2e} over"


@pytest.mark.parametrize("preset", list(plain.PRESETS))
@pytest.mark.parametrize("layout", ["soa", "aos", "aos_heads"])
@TYPES
@pytest.mark.parametrize("turned", [True, False], ids=["turned", "stored"])
def test_presets(dev, preset, layout, dtype, turned):
    rng = np.random.default_rng(5)
    kb, vb = plain.PRESETS[preset]
    for n, hk, bs in ((1, 1, 16), (37, 3, 16), (300, 8, 64)):
        blocks = -(-n // bs) + 2
        cache, k, v = plain.make_cache(rng, blocks, bs, hk, preset, layout)
        rot = plain.rotation(rng) if turned else None
        slots = rng.permutation(blocks * bs)[:n]
        key, value = load(cache, layout, slots, rot, kb, vb, dtype, dev)
        wk, bk, wv, bv = expect(k[slots // bs, slots % bs], v[slots // bs, slots % bs], rot, kb, layout, dtype)
        compare(key, wk, bk, f"key {n}")
        compare(value, wv, bv, f"value {n}")


@pytest.mark.parametrize("preset", ["4bit", "k8v4"])
@pytest.mark.parametrize("bs", [1, 3, 24])
def test_other_block_sizes(dev, preset, bs):
    rng = np.random.default_rng(bs)
    kb, vb = plain.PRESETS[preset]
    cache, k, v = plain.make_cache(rng, 50, bs, 4, preset, "aos")
    rot, slots = plain.rotation(rng), rng.integers(0, 50 * bs, 130)
    key, value = load(cache, "aos", slots, rot, kb, vb, torch.float16, dev)
    wk, bk, wv, bv = expect(k[slots // bs, slots % bs], v[slots // bs, slots % bs], rot, kb, "aos", torch.float16)
    compare(key, wk, bk, "key")
    compare(value, wv, bv, "value")


@pytest.mark.parametrize("layout", ["soa", "aos_heads"])
def test_slots_of_no_token_give_zeros(dev, layout):
    # their neighbours hold NaNs, and so does the place that a slot outside the cache is read from
    rng = np.random.default_rng(8)
    cache, k, v = plain.make_cache(rng, 3, 16, 2, "4bit", layout)
    plain.spoil(cache, [(0, 0), (0, 1), (2, 15)], "4bit", layout)
    slots = np.array([5, -1, 48, 47 - 16, 5, -2 ** 31, 2 ** 31 - 1, 20], np.int64)
    rot = plain.rotation(rng)
    for turn in (rot, None):
        key, value = load(cache, layout, slots, turn, 4, 4, torch.float32, dev)
        there = (slots >= 0) & (slots < 48)
        assert not key[torch.from_numpy(~there)].any() and not value[torch.from_numpy(~there)].any()
        s = slots[there]
        wk, bk, wv, bv = expect(k[s // 16, s % 16], v[s // 16, s % 16], turn, 4, layout, torch.float32)
        compare(key[torch.from_numpy(there)], wk, bk, "key")
        compare(value[torch.from_numpy(there)], wv, bv, "value")


def test_what_the_writer_left(dev):
    """Written by ``store``, read back: keys within the codebook's own error, values within half a code."""
    gen = torch.Generator(device="cuda").manual_seed(3)
    n, hk = 500, 4
    key = torch.randn(n, hk, D, generator=gen, device=dev)
    value = torch.randn(n, hk, D, generator=gen, device=dev)
    cents = torch.from_numpy(codebook.centroids(D, 4).astype(np.float32)).to(dev)
    mids = ((cents[1:] + cents[:-1]) / 2).contiguous()
    rot = torch.from_numpy(plain.rotation(np.random.default_rng(0))).to(dev)
    cache = torch.zeros(40, 16, hk, 134, dtype=torch.uint8, device=dev)
    slots = torch.randperm(640, generator=gen, device=dev)[:n].to(torch.int32)
    ops.store(key, value, cache, slots, rot, mids, cents, layout="soa", norm_correction=True)
    k, v = ops.cache_load(cache, slots, rot, cents, dtype=torch.float32)
    # a Gaussian's 16-level quantiser leaves 0.95 % of its power; a rotated row's dims are close to Gaussian
    assert (k - key).square().sum() < 0.011 * key.square().sum()
    step = (value.amax(-1) - value.amin(-1)) / 15
    assert ((v - value).abs() <= step[..., None] * 0.5 * 1.01 + value.abs().amax(-1, keepdim=True) * 2.0 ** -10 * 2).all()


@TYPES
def test_given_outputs_and_graph(dev, dtype):
    rng = np.random.default_rng(1)
    cache, k, v = plain.make_cache(rng, 20, 16, 8, "4bit", "soa")
    rot, slots = torch.from_numpy(plain.rotation(rng)).to(dev), torch.arange(100, dtype=torch.int32, device=dev)
    cents = torch.from_numpy(codebook.centroids(D, 4).astype(np.float32)).to(dev)
    cache = cache.to(dev)
    key, value = (torch.empty(100, 8, D, dtype=dtype, device=dev) for _ in range(2))
    run = lambda: ops.cache_load(cache, slots, rot, cents, dtype=dtype, key=key, value=value)  # noqa: E731
    got = run()
    assert got[0] is key and got[1] is value
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        run()
    for shift in (0, 7, 200):
        slots.copy_(torch.arange(shift, shift + 100, device=dev))
        key.zero_(), value.zero_()
        g.replay()
        torch.cuda.synchronize()
        s = np.arange(shift, shift + 100)
        wk, bk, wv, bv = expect(k[s // 16, s % 16], v[s // 16, s % 16], rot.cpu().numpy(), 4, "soa", dtype)
        compare(key, wk, bk, "key")
        compare(value, wv, bv, "value")


# ---- merge_states ----------------------------------------------------------------------------
# The weights' error: two exponentials and a quotient of them, 2^-20 in all; the sum of two products, rounded.

def joined(a, la, b, lb):
    with np.errstate(all="ignore"):
        top = np.maximum(la, lb)
        wa, wb = (np.where(x == -np.inf, 0, np.exp(x - top)) for x in (la, lb))
        total = wa + wb
        none = total == 0
        pa, pb = (np.where((w == 0)[..., None], 0, np.where(none, 0, w / total)[..., None] * x) for w, x in ((wa, a), (wb, b)))
        return pa + pb, np.where(none, -np.inf, top + np.log(total)), np.abs(pa) + np.abs(pb)


@TYPES
@pytest.mark.parametrize("shape", [(1,), (5, 3), (63, 1), (17, 32), (1000, 8)], ids=str)
def test_merge(dev, dtype, shape):
    rng = np.random.default_rng(len(shape))
    make = lambda: torch.from_numpy(rng.standard_normal(shape + (D,)).astype(np.float32)).to(dtype)  # noqa: E731
    a, b = make(), make()
    la, lb = (torch.from_numpy((8 * rng.standard_normal(shape)).astype(np.float32)) for _ in range(2))
    for l, x, p in ((la, a, 0.2), (lb, b, 0.2)):
        none = torch.from_numpy(rng.random(shape) < p)
        l[none] = -np.inf
        x[none] = float("nan")
    want, sums, size = joined(a.double().numpy(), la.double().numpy(), b.double().numpy(), lb.double().numpy())
    for place in ("new", "a", "b"):
        da, dla, db, dlb = (x.to(dev) for x in (a, la, b, lb))
        given = {"new": {}, "a": dict(out=da, lse=dla), "b": dict(out=db, lse=dlb)}[place]
        out, lse = ops.merge_states(da, dla, db, dlb, **given)
        assert not given or (out is given["out"] and lse is given["lse"])
        over = np.abs(out.double().cpu().numpy() - want) - HALF_STEP[dtype] * np.abs(want) - 2.0 ** -20 * size
        assert over.max() <= (2.0 ** -25 if dtype == torch.float16 else 0), over.max()
        got = lse.double().cpu().numpy()
        fine = np.isfinite(sums)
        assert np.array_equal(got[~fine], sums[~fine])
        assert not fine.any() or (np.abs(got - sums)[fine] <= 2.0 ** -22 + 2.0 ** -22 * np.abs(sums[fine])).all()


def test_merge_of_nothing(dev):
    out, lse = ops.merge_states(torch.empty(0, 4, D, device=dev), torch.empty(0, 4, device=dev),
                                torch.empty(0, 4, D, device=dev), torch.empty(0, 4, device=dev))
    assert out.shape == (0, 4, D) and lse.shape == (0, 4)
