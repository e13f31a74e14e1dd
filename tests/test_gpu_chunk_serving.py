"""The operators on chunks of tokens as a server uses them together: prompts written and attended to chunk by chunk from one
captured graph (``rope_store``, then ``chunk_attention`` over the cache with and without a window), drafted tokens
behind them, and the same chunk from two parts: the tokens before it out of the cache, its own ones by other means from
``cache_load``'s rows, joined by ``merge_states``.

The reference is masked attention in float64 over the values that the cache's bytes stand for, with the queries that the
writer returned.  Bars as in ``test_gpu_chunk``."""
import numpy as np
import pytest
import torch

import span_plain as plain
from chunk_plain import D, HALF_STEP, attend, visible
from test_gpu_rope_store import angles
from test_gpu_span_serving import codes
from tq4_decode import ops

pytestmark = pytest.mark.gpu
BS, HK, GROUP = 16, 2, 4
HQ = HK * GROUP


class Server:
    """A cache, its table and the tokens of each sequence; `step` takes the new tokens of each."""

    def __init__(self, dev, preset, layout, dtype, seqs=3, width=24):
        self.dev, self.preset, self.layout, self.dtype = dev, preset, layout, dtype
        self.kb, self.vb = plain.PRESETS[preset]
        rng = np.random.default_rng(1)
        slot, pool = plain.slot_bytes(self.kb, self.vb), 1 + seqs * width
        shape = (pool, HK, BS, slot) if layout == "aos_heads" else (pool, BS, HK, slot)
        cache = torch.full(shape, 0xFF, dtype=torch.uint8, device=dev)
        self.cache = cache.transpose(1, 2) if layout == "aos_heads" else cache
        self.table = (1 + rng.permutation(pool - 1)).astype(np.int32).reshape(seqs, width)
        self.rot = plain.rotation(rng)
        self.cos_sin = angles(width * BS, D).to(dev)
        self.lens = np.zeros(seqs, int)
        self.kw = dict(key_bits=self.kb, value_bits=self.vb, layout="soa" if layout == "soa" else "aos")
        self.cents, self.mids = codes(self.kb, dev)
        self.rot_dev = None if self.kb == 8 else self.put(self.rot)

    def put(self, x):
        return torch.from_numpy(np.ascontiguousarray(x)).to(self.dev)

    def slot(self, b, t):
        return int(self.table[b, t // BS]) * BS + t % BS

    def buffers(self, tokens):
        self.tokens, seqs = tokens, len(self.lens)
        zeros = lambda *s, dtype=torch.int32: torch.zeros(*s, dtype=dtype, device=self.dev)  # noqa: E731
        self.qkv = zeros(tokens, (HQ + 2 * HK) * D, dtype=self.dtype)
        self.pos, self.slots = zeros(tokens, dtype=torch.int64), torch.full((tokens,), -1, dtype=torch.int32, device=self.dev)
        self.dev_lens, self.starts, self.dev_table = zeros(seqs), zeros(seqs + 1), self.put(self.table)
        self.q = zeros(tokens, HQ, D, dtype=self.dtype)
        self.whole, self.local = (ops.ChunkWorkspace(tokens, seqs, HQ, HK, self.dev, self.dtype) for _ in range(2))

    def run(self):
        q, k, v = (x.view(self.tokens, -1, D) for x in self.qkv.split([HQ * D, HK * D, HK * D], 1))
        soa = self.layout == "soa" and self.kb != 8
        ops.rope_store(q, k, v, self.pos, self.cos_sin, self.cache, self.slots, self.rot_dev, self.mids,
                       self.cents if soa else None, query_out=self.q, norm_correction=soa, **self.kw)
        args = (self.q, self.rot_dev, self.cache, self.dev_table, self.dev_lens, self.starts, self.cents)
        ops.chunk_attention(*args, workspace=self.whole, return_lse=True, **self.kw)
        ops.chunk_attention(*args, workspace=self.local, window=40, first_tokens=3, **self.kw)

    def fill(self, counts, gen):
        """New tokens for each sequence; the buffers' other rows belong to none and are not written."""
        starts = np.concatenate([[0], np.cumsum(counts)])
        qkv = torch.randn(self.tokens, self.qkv.size(1), generator=gen).to(self.dtype)
        pos, slots = np.zeros(self.tokens, np.int64), np.full(self.tokens, -1, np.int32)
        for b, n in enumerate(counts):
            for i in range(n):
                pos[starts[b] + i], slots[starts[b] + i] = self.lens[b] + i, self.slot(b, self.lens[b] + i)
        self.lens += counts
        for to, x in ((self.qkv, qkv), (self.pos, torch.from_numpy(pos)), (self.slots, torch.from_numpy(slots)),
                      (self.starts, torch.from_numpy(starts.astype(np.int32))),
                      (self.dev_lens, torch.from_numpy(self.lens.astype(np.int32)))):
            to.copy_(x)
        return starts

    def stored(self, b):
        kc, vc, fields = plain.split_cache(self.cache.cpu().numpy(), self.kb, self.vb, self.layout)
        with np.errstate(invalid="ignore"):
            k, v = plain.values_of(kc, vc, fields, self.kb, self.layout)
        t = np.arange(self.lens[b])
        return k[self.table[b, t // BS], t % BS], v[self.table[b, t // BS], t % BS]

    def queries(self, rows):
        q = self.q[rows].double().cpu().numpy()
        return q if self.kb == 8 else q @ self.rot.astype(np.float64)

    def compare(self, out, lse, rows, want, what, step=None):
        o, sums, dev_out, dev_lse = want
        step = HALF_STEP[self.dtype] if step is None else step
        over = np.abs(out[rows].double().cpu().numpy() - o) - step * np.abs(o) - 8 * dev_out * (1 + step)
        assert over.max() <= 1e-4, (what, over.max())
        if lse is not None:
            assert (np.abs(lse[rows].double().cpu().numpy() - sums) - 8 * dev_lse).max() <= 1e-4, what


CASES = pytest.mark.parametrize("preset,layout,dtype", [
    ("4bit", "soa", torch.bfloat16), ("4bit", "aos", torch.float16), ("k8v4", "aos_heads", torch.bfloat16),
    ("3bit", "soa", torch.float16), ("k3v4", "aos", torch.bfloat16)])


@CASES
@pytest.mark.parametrize("tokens,plan", [
    (96, [[64, 20, 12], [64, 0, 31], [0, 96, 0], [1, 1, 1], [5, 0, 4], [90, 3, 1]]),   # prompts in chunks
    (15, [[5, 5, 5], [15, 0, 0], [1, 2, 3], [0, 5, 4], [5, 1, 5]]),                    # drafts
])
def test_replayed_steps(dev, preset, layout, dtype, tokens, plan):
    s, gen = Server(dev, preset, layout, dtype), torch.Generator().manual_seed(3)
    s.buffers(tokens)
    s.run()  # (no sequence has tokens: nothing is written)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        s.run()
    for counts in plan:
        starts = s.fill(np.array(counts), gen)
        s.whole.out.fill_(7.0)
        graph.replay()
        torch.cuda.synchronize()
        assert (s.whole.out[starts[-1]:] == 7.0).all()
        for b, n in enumerate(counts):
            if n == 0:
                continue
            rows = slice(starts[b], starts[b] + n)
            k, v = s.stored(b)
            how = (None, D ** -0.5), (True, s.kb != 8)
            q = s.queries(rows)
            s.compare(s.whole.out, s.whole.lse, rows, attend(q, k, v, visible(n, s.lens[b], True, 0, 0), *how[0], *how[1]), "whole")
            s.compare(s.local.out, None, rows,
                      attend(q, k, v, visible(n, s.lens[b], True, 40, 3), *how[0], dtype == torch.float16, s.kb != 8), "window")
    used = {s.slot(b, t) for b in range(3) for t in range(s.lens[b])}
    data = s.cache.cpu()
    if s.layout != "soa":
        assert all((data[p, o] == 0xFF).all() for p in range(data.size(0)) for o in range(BS) if p * BS + o not in used)
    assert (data[0] == 0xFF).all()


@CASES
@pytest.mark.parametrize("counts", [[4, 1, 7], [60, 33, 0]], ids=str)
def test_a_chunk_from_two_parts(dev, preset, layout, dtype, counts):
    """The tokens before the chunk, each new token seeing all of them, and the chunk's own, causal: from the rows that
    ``cache_load`` returns, in the basis the queries are given in; joined, the result over all tokens.

    Bar: both parts and the joined row are rounded to the type (the parts weigh one together); what is loaded is
    within 2^-15 of the sum of magnitudes (fp32), which moves a score by 2^-15 of sum |q| (|k| |rot|) at most, and the
    result by twice that of sum p |v|."""
    s, gen = Server(dev, preset, layout, dtype), torch.Generator().manual_seed(4)
    before = np.array([100, 0, 37])
    s.buffers(int(before.sum()))
    s.fill(before, gen)
    s.run()
    s.buffers(sum(counts) + 2)
    starts = s.fill(np.array(counts), gen)
    s.run()
    context = ops.chunk_attention(s.q, s.rot_dev, s.cache, s.dev_table, s.put(before.astype(np.int32)), s.starts, s.cents,
                                  causal=False, return_lse=True, **s.kw)
    own = torch.zeros_like(context[0]), torch.full_like(context[1], -np.inf)
    spread = {}
    for b, n in enumerate(counts):
        rows = slice(starts[b], starts[b] + n)
        slots = s.put(np.array([s.slot(b, before[b] + i) for i in range(n)], np.int32))
        if n == 0:
            continue
        k, v = (x.double().cpu().numpy() for x in ops.cache_load(s.cache, slots, s.rot_dev, s.cents, dtype=torch.float32, **s.kw))
        q = s.q[rows].double().cpu().numpy()
        o, lse, _, _ = attend(q, k, v, visible(n, n, True, 0, 0), None, D ** -0.5, True, False)
        own[0][rows], own[1][rows] = torch.from_numpy(o).to(dtype).to(dev), torch.from_numpy(lse).float().to(dev)
        r = np.abs(s.rot.astype(np.float64))
        move = 0 if s.kb == 8 else 2.0 ** -15 * D ** -0.5 * max(
            (np.abs(q[:, h * GROUP:(h + 1) * GROUP]).reshape(-1, D) @ (np.abs(k[:, h] @ s.rot) @ r.T).T).max() for h in range(HK))
        spread[b] = 2 * move * np.abs(v).max()
    out, lse = ops.merge_states(*context, *own)
    for b, n in enumerate(counts):
        if n == 0:
            continue
        rows = slice(starts[b], starts[b] + n)
        k, v = s.stored(b)
        q = s.queries(rows)
        want = attend(q, k, v, visible(n, s.lens[b], True, 0, 0), None, D ** -0.5, True, s.kb != 8)
        step = HALF_STEP[dtype]
        wa = np.exp(context[1][rows].double().cpu().numpy() - want[1])[..., None]
        wb = np.exp(own[1][rows].double().cpu().numpy() - want[1])[..., None]
        parts = wa * np.abs(context[0][rows].double().cpu().numpy()) + wb * np.abs(own[0][rows].double().cpu().numpy())
        over = np.abs(out[rows].double().cpu().numpy() - want[0]) - step * 1.01 * (np.abs(want[0]) + parts) - 8 * want[2] - spread[b]
        assert over.max() <= 1e-4, over.max()
        assert (np.abs(lse[rows].double().cpu().numpy() - want[1])).max() <= 1e-4 + spread[b]
    # (rows of no sequence: nothing on either side)
    assert (own[1][starts[-1]:] == -np.inf).all()
