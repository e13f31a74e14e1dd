"""The shared prefix (``ops.prefix_decode``) where its parts can go wrong, against float64: sequences a little shorter
than a long prefix, whose own tokens are many parts, and runs of tokens that weigh nothing."""
import numpy as np
import pytest
import torch

import span_plain as plain
from test_gpu_prefix import build, check
from tq4_decode import codebook, ops

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("preset,layout,dtype", [("4bit", "soa", torch.bfloat16), ("3bit", "aos", torch.float16), ("k8v4", "soa", torch.float16)])
@pytest.mark.parametrize("short", [[4095], [0, 4080, 17, 3000, 4095], [4095] * 5])
def test_long_sequences_below_the_prefix(dev, preset, layout, dtype, short):
    lens = [4096, 4100, *short, 4196, 4097]
    check(dev, build(12, lens, 4096, 2, 4, preset=preset, layout=layout, dtype=dtype), 16, sinks=len(short) == 5)


@pytest.mark.parametrize("preset,layout", [("4bit", "soa"), ("4bit", "aos"), ("3bit", "soa")])
@pytest.mark.parametrize("batch,infinite", [(5, 512), (5, 96), (40, 512), (40, 128)])
def test_runs_of_minus_infinity(dev, preset, layout, batch, infinite):
    """Keys of infinite norm on the far side of every query, in the first tiles or the whole prefix: scores of -inf, which
    weigh nothing beside the finite ones (a sequence without any: NaN and -inf, as plain attention)."""
    prefix, hk, group, bs = 512, 2, 4, 16
    kb, vb = plain.PRESETS[preset]
    rng = np.random.default_rng(5)
    lens = [prefix + (0 if b == 0 else 3 * b) for b in range(batch)]
    width = -(-max(lens) // bs)
    own = width - prefix // bs
    cache, k, v = plain.make_cache(rng, prefix // bs + batch * own, bs, hk, preset, layout)
    ids = rng.permutation(cache.size(0)).astype(np.int32)
    table = np.concatenate([np.tile(ids[:prefix // bs], (batch, 1)), ids[prefix // bs:].reshape(batch, own)], 1)
    raw, kc = cache.numpy(), plain.split_cache(cache.numpy(), kb, vb, layout)[0]
    codes, far = 16 * kb, np.float16(np.inf).tobytes()
    for t in range(infinite):  # codes of the lowest centroid against a query of positive elements
        block, off = table[0, t // bs], t % bs
        kc[block, off] = 0
        k[block, off] = -np.inf
        for h in range(hk):
            if layout == "soa":
                flat, rec = raw[block].reshape(-1), 16 * (kb + vb)
                at, norm = (off * hk + h) * rec, bs * hk * rec + 2 * (h * 3 * bs + off)
            else:
                flat, at, norm = raw[block, off, h], 0, codes
            flat[at:at + codes] = 0
            flat[norm:norm + 2] = np.frombuffer(far, np.uint8)
    query = torch.from_numpy(np.abs(rng.standard_normal((batch, hk * group, 128))).astype(np.float32) + 0.1).to(torch.float16)
    put = lambda x: torch.from_numpy(np.ascontiguousarray(x)).to(dev)  # noqa: E731
    out, lse = ops.prefix_decode(query.to(dev), torch.eye(128, device=dev), cache.to(dev), put(table),
                                 torch.tensor(lens, dtype=torch.int32, device=dev), put(codebook.centroids(128, kb)), 8, prefix,
                                 key_bits=kb, value_bits=vb, layout=layout, kernel="shared")
    out, lse = out.double().cpu().numpy(), lse.double().cpu().numpy()
    for b, n in enumerate(lens):
        t = np.arange(infinite, n)
        if len(t) == 0:
            assert np.isnan(out[b]).all() and np.isneginf(lse[b]).all()
            continue
        kk, vv = k[table[b, t // bs], t % bs], v[table[b, t // bs], t % bs]
        o, l = plain.attend(query[b].double().numpy(), kk, vv)
        size = plain.attend(query[b].double().numpy(), kk, np.abs(vv))[0]
        # (scores off by less than 2e-5, which sum |q_d k_d| up to four times a Gaussian query's makes of 6e-6)
        assert (np.abs(out[b] - o) <= 2.0 ** -11 * np.abs(o) + 4e-5 * size).all(), b
        assert np.abs(lse[b] - l).max() <= 2e-5, b
