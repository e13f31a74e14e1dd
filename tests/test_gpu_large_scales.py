"""V scales up to f16's largest number beside small ones in the matrix-core steps (``full_decode``, ``window_decode``, and
``prefix_decode`` where it takes the sequences' own steps): a weight, softmax weight times scale, is an f16 pair and must
stay in f16's range while the running maximum lags behind.

Against float64.  Bar: a token's score is off by less than 6e-6 (f16 pairs: 2^-21 of 128 products, eight deviations, and
fp32 roundings of its size), so the output by 2 * 6e-6 of sum p |v| at most, fp32 sums and weights of 2^-20 aside: 2^-16
of it in all; half a step of a 16-bit output besides."""
import numpy as np
import pytest
import torch

import span_plain as plain
from test_gpu_prefix_bits import scalars_of
from tq4_decode import codebook, ops

pytestmark = pytest.mark.gpu
D, BS = 128, 16


def case(seed, preset, layout, batch, most, hk, group, dev):
    rng = np.random.default_rng(seed)
    lens = np.array([1 + (most - 1) * (b + 1) // batch for b in range(batch)], np.int32)
    width = -(-most // BS)
    cache, _, _ = plain.make_cache(rng, batch * width, BS, hk, preset, layout)
    log = lambda rng, shape: np.exp(rng.uniform(np.log(0.01), np.log(65000.0), shape))  # noqa: E731
    zero = lambda rng, shape: rng.uniform(-65000.0, 65000.0, shape)  # noqa: E731
    cache, k, v = scalars_of(log, zero)(rng, cache, preset, layout)
    table = rng.permutation(batch * width).astype(np.int32).reshape(batch, width)
    query = torch.from_numpy(rng.standard_normal((batch, hk * group, D)).astype(np.float32)).to(torch.bfloat16)
    rot = plain.rotation(rng)
    put = lambda x: torch.from_numpy(np.ascontiguousarray(x)).to(dev)  # noqa: E731
    kb, vb = plain.PRESETS[preset]
    q = query.double().numpy() if kb == 8 else query.double().numpy() @ rot.astype(np.float64)
    args = (query.to(dev), None if kb == 8 else put(rot), cache.to(dev), put(table), put(lens),
            None if kb == 8 else put(codebook.centroids(D, kb)), 16)

    def check(out, lse, seen):
        out, lse = out.double().cpu().numpy(), lse.double().cpu().numpy()
        for b, n in enumerate(lens):
            t = np.array([t for t in range(n) if seen(t, n)])
            kk, vv = k[table[b, t // BS], t % BS], v[table[b, t // BS], t % BS]
            o, l = plain.attend(q[b], kk, vv)
            size = plain.attend(q[b], kk, np.abs(vv))[0]
            assert (np.abs(out[b] - o) <= 2.0 ** -16 * size + 2.0 ** -8 * np.abs(o)).all(), b
            assert np.abs(lse[b] - l).max() <= 2e-5, b

    return args, dict(key_bits=kb, value_bits=vb, layout=layout), check


@pytest.mark.parametrize("preset,layout", [("4bit", "soa"), ("4bit", "aos"), ("k3v4", "soa"), ("3bit", "aos"), ("k8v4", "soa")])
@pytest.mark.parametrize("batch,most,hk,group", [(3, 900, 2, 4), (40, 400, 8, 4), (5, 1300, 2, 8), (300, 160, 4, 2)])
def test_windows_and_own_steps(dev, preset, layout, batch, most, hk, group):
    args, kw, check = case(batch, preset, layout, batch, most, hk, group, dev)
    out, lse = ops.window_decode(*args, 300, first_tokens=5, **kw)
    check(out, lse, lambda t, n: t < 5 or t >= n - 300)
    out, lse = ops.prefix_decode(*args, 0, **kw)
    check(out, lse, lambda t, n: True)


@pytest.mark.parametrize("layout", ["soa", "aos"])
@pytest.mark.parametrize("batch,most,hk,group", [(3, 900, 2, 4), (64, 500, 8, 4), (5, 1300, 2, 8)])
def test_full_steps(dev, layout, batch, most, hk, group):
    args, _, check = case(7, "4bit", layout, batch, most, hk, group, dev)
    out, lse = ops.full_decode(*args, layout=layout, out_dtype=torch.float32)
    check(out, lse, lambda t, n: True)
