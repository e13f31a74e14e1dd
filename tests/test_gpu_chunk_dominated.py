"""``ops.chunk_attention`` on rows that one token dominates (an attention sink): a first token 9 to 17 nats above 4095
others, its value 0, so that the others' small weights are all that the result is made of.

Bar.  Half a step of the output; and of what the products' operands lose:

* a weight, rounded to f16 (2^-11 of it; below f16's normal range half a step of its denormals, 2^-25, where the row's
  largest weight is 2^8 or more: 2^-33 of that), moves the result by its share of v less the result;
* where V's scale is part of the weight (few rows, fp16 results, a log-sum-exp) that product is rounded: 2^-11 of it, or 2^-25
  where the largest weight times the power of two above the largest scale is 2^7 or more: 2^-32 of that; it meets
  the code's distance from the middle one;
* V in f16: 2^-11 of it;
* scores from single f16 (bf16 results, keys that are not FP8): eight deviations of rounding both factors and the rotation's
  elements (as in ``chunk_plain.attend``); from f16 pairs: 2^-22 of 25 in log2 units and of fp32 sums, 2^-15 altogether.

All sequences share one context, so that workgroups have whole row tiles: a cut one would have token 0 in one part only."""
import numpy as np
import pytest
import torch

import span_plain as plain
from chunk_plain import D, HALF_STEP, RHO
from test_gpu_chunk import call

pytestmark = pytest.mark.gpu
TOKENS, HK, GROUP = 4096, 8, 4


def make(rng, preset, layout, scale):
    """A cache whose V codes are of the upper half: values 8 to 15 times (3 bits: 4 to 7) their scale, but token 0's are 0."""
    kb, vb = plain.PRESETS[preset]
    cache, _, _ = plain.make_cache(rng, TOKENS // 16, 16, HK, preset, layout)
    kc, vc, fields = plain.split_cache(cache.numpy(), kb, vb, layout)
    vc = vc | (1 << (vb - 1))
    fields = [f.copy() for f in fields]
    fields[-2] = (scale * rng.uniform(0.5, 1.0, fields[-2].shape)).astype(np.float16)
    fields[-1] = np.zeros_like(fields[-1])
    fields[-2][0, 0] = 0
    k, v = plain.values_of(kc, vc, fields, kb, layout)
    if layout == "soa":
        rec = np.concatenate([plain.pack(kc, kb), plain.pack(vc, vb)], -1).reshape(len(vc), -1)
        meta = np.ascontiguousarray(np.stack([f.transpose(0, 2, 1) for f in fields], 2)).view(np.uint8).reshape(len(vc), -1)
        data = np.concatenate([rec, meta], 1).reshape(cache.shape)
    else:
        cells = [np.ascontiguousarray(f[..., None]).view(np.uint8) for f in fields]
        data = np.concatenate([plain.pack(kc, kb)] + cells[:-2] + [plain.pack(vc, vb)] + cells[-2:], -1)
    middle = ((1 << vb) - 1) / 2 * fields[-2].astype(np.float64)
    flat = lambda x: x.reshape((TOKENS,) + x.shape[2:])  # noqa: E731
    return torch.from_numpy(np.ascontiguousarray(data)), flat(k), flat(v), flat(middle)


class Shared:
    """What `test_gpu_chunk.call` takes: `batch` sequences of `n` new tokens each over the same blocks."""

    def __init__(self, seed, batch, n, preset, layout, dtype, scale):
        rng = np.random.default_rng(seed)
        self.preset, self.layout, self.dtype, self.n = preset, layout, dtype, n
        self.cache, self.k, self.v, self.middle = make(rng, preset, layout, scale)
        self.table = np.tile(np.arange(TOKENS // 16, dtype=np.int32), (batch, 1))
        self.lens = np.full(batch, TOKENS, np.int32)
        self.starts = (n * np.arange(batch + 1)).astype(np.int32)
        self.rot = plain.rotation(rng)
        self.top = rng.permutation(np.linspace(9, 17, batch * n * HK * GROUP)).reshape(batch * n, HK, GROUP, 1)
        first = self.k[0][None, :, None]
        q = self.top * D ** 0.5 * first / (first ** 2).sum(-1, keepdims=True) + 0.05 * rng.standard_normal((batch * n, HK, GROUP, D))
        q = q.reshape(batch * n, HK * GROUP, D)
        self.query = torch.from_numpy(q if preset == "k8v4" else q @ self.rot.astype(np.float64).T).to(dtype)
        self.sinks = None

    def want(self, b, h, fine, rounded):
        q = self.query[self.n * b:self.n * (b + 1), GROUP * h:GROUP * (h + 1)].double().numpy()
        q = (q if self.preset == "k8v4" else q @ self.rot.astype(np.float64)).reshape(-1, D)
        k, v, middle = self.k[:, h], self.v[:, h], self.middle[:, h]
        end = np.repeat(TOKENS - self.n + 1 + np.arange(self.n), GROUP)[:, None]
        s = np.where(np.arange(TOKENS)[None] < end, q @ k.T * D ** -0.5, -np.inf)
        p = np.exp(s - s.max(-1, keepdims=True))
        p /= p.sum(-1, keepdims=True)
        out = p @ v
        most, far = p.max(-1, keepdims=True), np.abs(v - middle[:, None])
        by_v = p @ v + out + 2.0 ** -22 * most * (v.sum(0) + TOKENS * out)  # (v and out are not negative)
        scale = 2.0 ** np.ceil(np.log2(self.middle.max() / 3.5))
        code = np.zeros_like(far)
        np.divide(far, middle[:, None] / 3.5, out=code, where=middle[:, None] > 0)
        by_code = p @ far + 2.0 ** -21 * most * scale * code.sum(0)
        bar = 2.0 ** -11 * (by_code if fine else np.maximum(by_v, by_code) + out)
        if rounded:
            d2 = RHO ** 2 * (2 * (q ** 2) @ (k ** 2).T + 1.5 / D * (q ** 2).sum(-1)[:, None] * (k ** 2).sum(-1)[None]) / D
            w = p * p * d2
            bar = bar + 8 * np.sqrt(np.maximum(w @ v ** 2 - 2 * out * (w @ v) + w.sum(-1, keepdims=True) * out ** 2, 0))
        return out, bar + 2.0 ** -15 * out


@pytest.mark.parametrize("batch,n", [(64, 2), (64, 16), (32, 64)], ids=["tiles_of_32", "of_64", "of_256"])
@pytest.mark.parametrize("preset,layout", [("4bit", "soa"), ("4bit", "aos"), ("3bit", "soa"), ("k8v4", "aos")])
@pytest.mark.parametrize("dtype,lse", [(torch.bfloat16, False), (torch.bfloat16, True), (torch.float16, False)],
                         ids=["bf16", "bf16_lse", "fp16"])
@pytest.mark.parametrize("scale", [2.0 ** -10, 0.25, 100.0])
def test_one_token_dominates(dev, batch, n, preset, layout, dtype, lse, scale):
    b = Shared(5, batch, n, preset, layout, dtype, scale)
    got = call(b, dev, lse=lse)
    have = (got[0] if lse else got).double().cpu().numpy()
    fine = lse or dtype == torch.float16
    for i, h in ((0, 0), (batch // 2, 3), (batch - 1, HK - 1)):
        out, bar = b.want(i, h, fine, not fine and preset != "k8v4")
        bar = bar + HALF_STEP[dtype] * (out + bar) + (2.0 ** -25 if dtype == torch.float16 else 0)
        err = np.abs(have[n * i:n * (i + 1), GROUP * h:GROUP * (h + 1)].reshape(-1, D) - out)
        worst = np.unravel_index((err / bar).argmax(), err.shape)
        assert (err <= bar).all(), (f"{(err / bar).max():.2f} of the bar: off by {err[worst] / out[worst]:.2%}, "
                                    f"{b.top[n * i:n * (i + 1), h].reshape(-1)[worst[0]]:.1f} nats")
