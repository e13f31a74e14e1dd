"""Batches of sequences with several new tokens each, over caches of random codes, and plain masked attention over
them in float64: what the tests of ``ops.chunk_attention`` compare with."""
import numpy as np
import torch

import span_plain as plain

D = 128
HALF_STEP = {torch.bfloat16: 2.0 ** -8, torch.float16: 2.0 ** -11}
RHO = 2.0 ** -11 / 3 ** 0.5  # deviation of a relative error spread over half a step of f16


def visible(n, length, causal, window, first):
    """[n, length]: what each new token sees."""
    t, end = np.arange(length)[None], np.full((n, 1), length)
    if causal:
        end = length - n + 1 + np.arange(n)[:, None]
    seen = t < end
    if window:
        seen &= (t >= end - window) | (t < first)
    return seen


MOST_FROM_MIDDLE = 3.2  # |V - its value at the middle code|: 8 codes of the largest scale, 0.4


def attend(q, k, v, seen, sinks, scale, fine, rounded_keys):
    """q [n, Hq, 128], k / v [tokens, Hk, 128] -> out, lse, and the deviations that the roundings of the products' f16
    operands leave in them: of a score both factors (``fine``: f16 pairs, none; FP8 keys and their queries are exact),
    of a weighted value the weight and the value (``fine``: weight times scale)."""
    n, hq, _ = q.shape
    hk, tokens = k.shape[1], k.shape[0]
    g = hq // hk
    out, lse = np.zeros((n, hq, D)), np.full((n, hq), -np.inf)
    dev, dev_lse = np.zeros((n, hq, D)), np.zeros((n, hq))
    for h in range(hk):
        qq = q[:, h * g:(h + 1) * g].reshape(n * g, D)
        mask = np.repeat(seen, g, axis=0)
        with np.errstate(all="ignore"):
            s = np.where(mask, qq @ k[:, h].T * scale, -np.inf)
        sink = np.tile(sinks[h * g:(h + 1) * g], n)[:, None] if sinks is not None else np.full((n * g, 1), -np.inf)
        top = np.maximum(s.max(-1, initial=-np.inf)[:, None], sink)
        has = np.isfinite(top[:, 0]) | np.isnan(top[:, 0])
        base = np.where(np.isfinite(top), top, 0)
        p = np.where(mask, np.exp(s - base), 0)
        total = p.sum(-1, keepdims=True) + np.exp(sink - base)
        with np.errstate(all="ignore"):
            p = np.where(has[:, None], p / total, 0)
            seen_v = np.where(mask.any(0)[:, None], v[:, h], 0)  # (what nobody sees may be anything)
            o = p @ seen_v
            out[:, h * g:(h + 1) * g] = o.reshape(n, g, D)
            lse[:, h * g:(h + 1) * g] = np.where(has, (base + np.log(total))[:, 0], -np.inf).reshape(n, g)
            p2 = p * p
            # sum of w (v - o)^2
            spread = lambda w: w @ seen_v ** 2 - 2 * o * (w @ seen_v) + w.sum(-1, keepdims=True) * o ** 2  # noqa: E731
            if fine:  # V's scale times the weight, one rounding, times the code's distance from the middle one
                var = RHO ** 2 * (MOST_FROM_MIDDLE ** 2 * p2.sum(-1, keepdims=True))
            else:     # V; the weight, whose sum is that of the rounded ones: an error of one moves the result by v - o
                var = RHO ** 2 * (p2 @ seen_v ** 2 + spread(p2))
                # or, for few rows, as `fine`: a lone token of value 0 has an exact v and v - o = 0, but its weight e times
                # its scale s is rounded and meets the code's distance from the middle one, (v - middle) / s: off by
                # RHO e |v - middle|, while the middle value and the sum have e itself
                var = np.maximum(var, RHO ** 2 * MOST_FROM_MIDDLE ** 2 * p2.sum(-1, keepdims=True))
            if not fine and rounded_keys:
                # both factors, and the rotation's elements r[j][d], whose roundings move q[d] by RHO sqrt(sum_j q_j^2 r_jd^2): with
                # r^2 about 1 / 128 everywhere, |q|^2 |k|^2 / 128 (a half more for where it is not)
                k2 = k[:, h] ** 2
                d2 = RHO ** 2 * (2 * (qq ** 2) @ k2.T + 1.5 / D * (qq ** 2).sum(-1)[:, None] * k2.sum(-1)[None]) * scale ** 2
                w = p2 * np.where(mask, d2, 0)
                var = var + spread(w)
                dev_lse[:, h * g:(h + 1) * g] = np.sqrt(w.sum(-1)).reshape(n, g)
            dev[:, h * g:(h + 1) * g] = np.sqrt(np.maximum(np.broadcast_to(var, o.shape), 0)).reshape(n, g, D)
    return out, lse, dev, dev_lse


class Batch:
    """Sequences (new tokens, tokens in the cache); page 0 is nobody's and holds NaNs, as do the tokens behind each
    sequence's last one in its last page.  ``pad`` rows of no sequence in front of and behind the others."""

    def __init__(self, seed, pairs, hk, group, bs=16, preset="4bit", layout="soa", dtype=torch.bfloat16, pad=(0, 0),
                 wide=0, query_scale=1.0, spoil=True, change=None):
        rng = np.random.default_rng(seed)
        self.pairs, self.hk, self.group, self.preset, self.layout, self.dtype = pairs, hk, group, preset, layout, dtype
        blocks = [-(-n // bs) for _, n in pairs]
        pool = 1 + sum(blocks)
        cache, k, v = plain.make_cache(rng, pool, bs, hk, preset, layout)
        ids = 1 + rng.permutation(pool - 1)
        table = np.zeros((len(pairs), max([wide, 1] + blocks)), np.int32)
        at = 0
        for b, n in enumerate(blocks):
            table[b, :n] = ids[at:at + n]
            at += n
        if spoil:
            behind = [(0, t) for t in range(bs)]
            behind += [(int(table[b, n // bs]), t) for b, (_, n) in enumerate(pairs) if n % bs for t in range(n % bs, bs)]
            plain.spoil(cache, behind, preset, layout)
        if change is not None:
            change(self, cache, table, k, v)
        counts = [m for m, _ in pairs]
        self.starts = (pad[0] + np.concatenate([[0], np.cumsum(counts)])).astype(np.int32)
        self.tokens = int(self.starts[-1]) + pad[1]
        q = rng.standard_normal((self.tokens, hk * group, D)).astype(np.float32) * query_scale
        self.query = torch.from_numpy(q).to(dtype)
        self.rot = plain.rotation(rng)
        self.sinks = rng.normal(0, 2, hk * group).astype(np.float32)
        self.cache, self.table, self.k, self.v, self.bs = cache, table, k, v, bs
        self.lens = np.array([n for _, n in pairs], np.int32)

    def want(self, causal=True, window=0, first=0, sinks=False, lse=False, scale=D ** -0.5):
        q = self.query.double().numpy()
        if self.preset != "k8v4":
            q = q @ self.rot.astype(np.float64)
        fine = lse or self.dtype == torch.float16
        hq = self.hk * self.group
        parts = [np.zeros((self.tokens, hq, D)), np.zeros((self.tokens, hq)), np.zeros((self.tokens, hq, D)),
                 np.zeros((self.tokens, hq))]
        for b, (n, length) in enumerate(self.pairs):
            t = np.arange(length)
            at = self.table[b, t // self.bs], t % self.bs
            r = slice(self.starts[b], self.starts[b] + n)
            got = attend(q[r], self.k[at], self.v[at], visible(n, length, causal, window, first),
                         self.sinks.astype(np.float64) if sinks else None, scale, fine, self.preset != "k8v4")
            for whole, part in zip(parts, got):
                whole[r] = part
        return parts
