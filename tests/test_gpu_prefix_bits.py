"""How near the shared prefix comes to float64, at the size of the roundings that its kernel makes, and over
several tiles per workgroup.

Bars.  A score is a sum of 128 products q_d k_d: the rotated query, its f16 hi + lo parts, the centroid's and the
product of both lo parts that is left out are off by less than 2^-21 of an element together, spread over it
(deviation rho = 2^-21 / sqrt 3).  An element's error is the same for all tokens (the query's) or for all that
have its code (the centroid's), so it counts against the weighted mean of |k_d|: the log-sum-exp is off by
rho scale sqrt(sum_d (q_d sum_t p_t |k_td|)^2), eight deviations of which are allowed, and by fp32 roundings of its size and
of the scores' (2^-22).  A token's own score is off by d_t = rho scale sqrt(sum_d (q_d k_td)^2) + 2^-23 |s_t|, which moves the
output by p_t d_t |v_t - o|; a weight p_t times V's scale is rounded to f16 for bf16 outputs (2^-11 of the distance of v_t from
the middle code's value, spread over it), to f16 hi + lo for fp16 outputs (2^-22); both over all tokens as the square root of
the sum of their squares, eight deviations.  Then half a step of the output, and fp32 sums (2^-21 of sum p |v|).
For comparison, single f16 operands (2^-12 of every element) put the log-sum-exp off by 1e-4, 10 to 50 times the bar."""
import numpy as np
import pytest
import torch

import span_plain as plain
from tq4_decode import codebook, ops

pytestmark = pytest.mark.gpu
D = 128
HALF_STEP = {torch.bfloat16: 2.0 ** -8, torch.float16: 2.0 ** -11}
RHO = 2.0 ** -21 / 3 ** 0.5


def build(seed, batch, prefix, tail, hk, group, bs=16, preset="4bit", layout="soa", dtype=torch.float16, scalars=None):
    """`batch` sequences behind `prefix` shared tokens, with up to `tail` tokens of their own (the first: none)."""
    rng = np.random.default_rng(seed)
    own = -(-tail // bs)
    pool = prefix // bs + batch * own
    cache, k, v = plain.make_cache(rng, pool, bs, hk, preset, layout)
    if scalars is not None:
        cache, k, v = scalars(rng, cache, preset, layout)
    ids = rng.permutation(pool).astype(np.int32)
    table = np.zeros((batch, prefix // bs + own), np.int32)
    table[:, :prefix // bs] = ids[:prefix // bs]
    table[:, prefix // bs:] = ids[prefix // bs:].reshape(batch, own)
    lens = np.array([prefix + (0 if b == 0 else 1 + (tail - 1) * b // batch) for b in range(batch)], np.int32)
    query = torch.from_numpy(rng.standard_normal((batch, hk * group, D)).astype(np.float32)).to(dtype)
    return dict(cache=cache, k=k, v=v, table=table, lens=lens, query=query, rot=plain.rotation(rng), prefix=prefix, preset=preset,
                layout=layout, dtype=dtype, bs=bs, hk=hk)


def middle(c):
    """V at the middle code of every token of the cache."""
    kb, vb = plain.PRESETS[c["preset"]]
    heads = c["cache"].numpy()
    _, _, fields = plain.split_cache(heads, kb, vb, "soa" if c["layout"] == "soa" else "aos")
    f = [x.astype(np.float64)[..., None] for x in fields]
    return f[-2] * (1 << (vb - 1)) + f[-1]


def want(c, scale=D ** -0.5):
    """Outputs, log-sum-exps and their bars in float64."""
    kb = plain.PRESETS[c["preset"]][0]
    q = c["query"].double().numpy()
    if kb != 8:
        q = q @ c["rot"].astype(np.float64)
    batch, hq, hk, bs = *q.shape[:2], c["hk"], c["bs"]
    q = q.reshape(batch, hk, -1, D)
    mid = middle(c)
    parts = []  # (rows [hk, n, 128], K, V, middles [hk, tokens, .], sequences): the prefix, then every sequence's own

    def tokens(b, t):
        at = (c["table"][b, t // bs], t % bs)
        return [np.ascontiguousarray(x[at].transpose(1, 0, 2)) for x in (c["k"], c["v"], mid)]

    parts.append((q.transpose(1, 0, 2, 3).reshape(hk, -1, D), *tokens(0, np.arange(c["prefix"])), slice(None)))
    for b in range(batch):
        t = np.arange(c["prefix"], c["lens"][b])
        if len(t):
            parts.append((q[b], *tokens(b, t), slice(b, b + 1)))
    per_row = lambda x, n: x.reshape(hk, n, -1, x.shape[-1]).transpose(1, 0, 2, 3)  # noqa: E731  [sequences, hk, group, .]
    top = np.full((batch, hk, hq // hk, 1), -np.inf)
    for rows, k, _, _, seqs in parts:
        n = batch if seqs == slice(None) else 1
        s = np.matmul(rows, k.transpose(0, 2, 1)) * scale
        top[seqs] = np.maximum(top[seqs], per_row(s.max(-1, keepdims=True), n))
    shape = top.shape[:3]
    total, most = np.zeros(shape + (1,)), np.zeros(shape + (1,))
    out, size, mean_k = (np.zeros(shape + (D,)) for _ in range(3))
    kept = []
    for rows, k, v, m, seqs in parts:
        n = batch if seqs == slice(None) else 1
        s = np.matmul(rows, k.transpose(0, 2, 1)) * scale
        t = top[seqs].transpose(1, 0, 2, 3).reshape(hk, -1, 1)
        p = np.exp(s - t)
        total[seqs] += per_row(p.sum(-1, keepdims=True), n)
        most[seqs] = np.maximum(most[seqs], per_row(np.abs(s).max(-1, keepdims=True), n))
        out[seqs] += per_row(np.matmul(p, v), n)
        size[seqs] += per_row(np.matmul(p, np.abs(v)), n)
        mean_k[seqs] += per_row(np.matmul(p, np.abs(k)), n)
        kept.append((rows, k, v, m, seqs, n, s, p))
    out, size, mean_k, lse = out / total, size / total, mean_k / total, (top + np.log(total))[..., 0]
    weight = 2.0 ** -11 / 3 ** 0.5 if c["dtype"] == torch.bfloat16 else 2.0 ** -22
    var = np.zeros(shape + (D,))
    for rows, k, v, m, seqs, n, s, p in kept:
        w = (p / total[seqs].transpose(1, 0, 2, 3).reshape(hk, -1, 1)) ** 2
        d2 = (RHO * scale) ** 2 * np.matmul(rows ** 2, k.transpose(0, 2, 1) ** 2) + (2.0 ** -23 * s) ** 2
        wd = w * d2
        o = out[seqs].transpose(1, 0, 2, 3).reshape(hk, -1, D)
        x = np.matmul(wd, v * v) - 2 * o * np.matmul(wd, v) + o * o * wd.sum(-1, keepdims=True) + weight ** 2 * np.matmul(w, (v - m) ** 2)
        var[seqs] += per_row(np.maximum(x, 0), n)
    step = HALF_STEP[c["dtype"]]
    bar_out = step * np.abs(out) + 8 * np.sqrt(var) + 2.0 ** -21 * size + 1e-7
    bar_lse = 8 * RHO * scale * np.sqrt(((q * mean_k) ** 2).sum(-1)) + 2.0 ** -22 * (most[..., 0] + np.abs(lse) + 4)
    flat = lambda x: x.reshape((batch, hq) + x.shape[3:])  # noqa: E731
    return flat(out), flat(lse), flat(bar_out), flat(bar_lse)


def call(dev, c, splits, **kw):
    kb, vb = plain.PRESETS[c["preset"]]
    put = lambda x: torch.from_numpy(np.ascontiguousarray(x)).to(dev)  # noqa: E731
    heads = c["layout"] == "aos_heads"
    cache = c["cache"].transpose(1, 2).to(dev).transpose(1, 2) if heads else c["cache"].to(dev)
    cents = None if kb == 8 else put(codebook.centroids(D, kb))
    kw.setdefault("kernel", "shared")
    out, lse = ops.prefix_decode(c["query"].to(dev), None if kb == 8 else put(c["rot"]), cache, put(c["table"]), put(c["lens"]),
                                 cents, splits, c["prefix"], key_bits=kb, value_bits=vb,
                                 layout="soa" if c["layout"] == "soa" else "aos", **kw)
    torch.cuda.synchronize()
    return out.double().cpu().numpy(), lse.double().cpu().numpy()


def check_lse(dev, c, splits=8, scale=D ** -0.5):
    _, lse = call(dev, c, splits, attn_scale=scale)
    _, want_lse, _, bar = want(c, scale)
    assert (np.abs(lse - want_lse) / bar).max() <= 1.0, (np.abs(lse - want_lse) / bar).max()


@pytest.mark.parametrize("batch", [8, 20])
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
def test_query_elements_next_to_a_tie(dev, batch, dtype):
    """A query of elements whose product with the score scale is no tie of f16, but rounds to one in fp32: its hi
    part must be the one that its lo part was worked out from."""
    rng, log2e = np.random.default_rng(0), np.float32(1.4426950408889634)
    m = (1 + np.arange(128 if dtype == torch.bfloat16 else 1024) / (128.0 if dtype == torch.bfloat16 else 1024.0)).astype(np.float32)
    found = None
    while found is None:
        scale = np.float32(rng.uniform(0.06, 0.12))
        once, twice = (np.float64(m) * np.float64(scale * log2e)).astype(np.float16), (m * (scale * log2e)).astype(np.float16)
        if (once != twice).any():
            found = m[once != twice][0]
    c = build(1, batch, 96, 20, 2, 4, dtype=dtype)
    c["query"] = (torch.from_numpy(rng.choice([-1.0, 1.0], c["query"].shape).astype(np.float32)) * float(found)).to(dtype)
    c["rot"] = np.eye(D, dtype=np.float32)
    check_lse(dev, c, scale=float(scale))


@pytest.mark.parametrize("preset,layout", [("4bit", "soa"), ("4bit", "aos"), ("k3v4", "soa"), ("3bit", "aos_heads"), ("k8v4", "soa")])
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("batch,hk,group", [(150, 2, 8), (6, 2, 8)])
def test_log_sum_exps(dev, preset, layout, dtype, batch, hk, group):
    check_lse(dev, build(2, batch, 160, 30, hk, group, preset=preset, layout=layout, dtype=dtype))


FORMATS = [("4bit", "soa", torch.bfloat16), ("4bit", "aos", torch.float16), ("4bit", "soa", torch.float16), ("k3v4", "aos", torch.bfloat16),
           ("3bit", "aos_heads", torch.float16), ("k3v4", "soa", torch.float16), ("k8v4", "soa", torch.bfloat16), ("k8v4", "aos", torch.float16)]


def check(dev, c, splits, **kw):
    got = call(dev, c, splits, **kw)
    out, lse, bar_out, bar_lse = want(c)
    for what, x, y, bar in (("lse", got[1], lse, bar_lse), ("out", got[0], out, bar_out)):
        assert np.isfinite(x).all(), what
        assert (np.abs(x - y) / bar).max() <= 1.0, (what, (np.abs(x - y) / bar).max())


@pytest.mark.parametrize("preset,layout,dtype", FORMATS)
@pytest.mark.parametrize("batch,hk,group", [(40, 2, 8), (7, 2, 4)])
def test_outputs(dev, preset, layout, dtype, batch, hk, group):
    """V's codes are exact, its scales and middles fp32: fp16 outputs are as near as their own rounding."""
    check(dev, build(3, batch, 208, 40, hk, group, preset=preset, layout=layout, dtype=dtype), 8)


def scalars_of(scales, zeros, norms=None):
    """A hook of `build`: the cache with other scales and zeros of V (and norms)."""
    def put(rng, cache, preset, layout):
        kb, vb = plain.PRESETS[preset]
        n, bs, hk, slot = cache.shape
        assert layout != "aos_heads"
        raw = cache.numpy()
        kc, vc, fields = plain.split_cache(raw, kb, vb, layout)
        new = [f.copy() for f in fields]
        new[-2], new[-1] = scales(rng, (n, bs, hk)).astype(np.float16), zeros(rng, (n, bs, hk)).astype(np.float16)
        if norms is not None and kb != 8:
            new[0] = norms(rng, (n, bs, hk)).astype(np.float16)
        rec = 16 * (kb + vb)
        if layout == "soa":
            meta = np.stack([f.transpose(0, 2, 1) for f in new], 2)
            raw.reshape(n, -1)[:, bs * hk * rec:] = np.ascontiguousarray(meta).view(np.uint8).reshape(n, -1)
        else:
            at = 16 * kb + (0 if kb == 8 else 2) + 16 * vb
            for i, f in enumerate(new[-2:]):
                raw[..., at + 2 * i:at + 2 * i + 2] = np.ascontiguousarray(f[..., None]).view(np.uint8)
            if kb != 8:
                raw[..., 16 * kb:16 * kb + 2] = np.ascontiguousarray(new[0][..., None]).view(np.uint8)
        return (cache, *plain.values_of(kc, vc, new, kb, layout))
    return put


@pytest.mark.parametrize("preset,layout", [("4bit", "soa"), ("4bit", "aos"), ("3bit", "soa"), ("k8v4", "aos")])
@pytest.mark.parametrize("batch,prefix", [(40, 1040), (6, 528)])
def test_values_past_f16(dev, preset, layout, batch, prefix):
    """Scales up to f16's largest number beside small ones, values beyond it: finite, and as near as others."""
    log = lambda rng, shape: np.exp(rng.uniform(np.log(0.01), np.log(65000.0), shape))  # noqa: E731
    zero = lambda rng, shape: rng.uniform(-65000.0, 65000.0, shape)  # noqa: E731
    c = build(4, batch, prefix, 40, 8, 4, preset=preset, layout=layout, dtype=torch.bfloat16, scalars=scalars_of(log, zero))
    assert np.abs(c["v"]).max() > 3e5
    check(dev, c, 8)


@pytest.mark.parametrize("preset,layout,dtype", FORMATS)
@pytest.mark.parametrize("batch,hk,group,prefix", [(36, 8, 6, 3120), (12, 8, 5, 6192)])
def test_several_tiles_a_workgroup(dev, preset, layout, dtype, batch, hk, group, prefix):
    """Runs of three and four tiles on 256 CUs, the last tile ending early: 49 tiles of 64 tokens cut into 13 runs
    (216 rows, eight waves), 194 of 32 into 49 (60 rows, two waves)."""
    check(dev, build(5, batch, prefix, 24, hk, group, preset=preset, layout=layout, dtype=dtype), 8)


def test_sharing_by_rule_is_as_near(dev):
    """`kernel="auto"` where it shares: 64 x 4096, five tiles a workgroup."""
    c = build(6, 64, 4144, 30, 8, 4, dtype=torch.bfloat16)
    check(dev, c, 16, kernel="auto")
