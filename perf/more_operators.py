"""Operators of long prompts and drafted tokens on the quantised paged cache, with their plain forms.

Kinds:

* ``chunk``: ``chunk_attention`` -- several new tokens of each sequence attend to its paged cache: a chunk
  of a prompt or a few drafted tokens (causal: their own keys are in the cache), or the context behind a
  chunk whose own tokens are attended to elsewhere (not causal, with the log-sum-exp);
* ``load``: ``cache_load`` -- keys and values read back from their slots of the cache, keys turned back;
* ``merge``: ``merge_states`` -- two attention results of the same rows over different tokens made one.

Presets: ``4bit`` (4-bit K and V), ``k8v4`` (FP8 keys), ``k3v4`` and ``3bit``.  Layouts: ``soa``,
``aos``, and ``aos_heads`` (the ``transpose(1, 2)`` view of head-major AoS blocks that a backend
passes).  The plain forms are elementary torch operations in 32 bits, rounded once at the end.
"""
import math
import os
import sys
import types

import torch

own = False

D = 128
BITS = {"4bit": (4, 4), "k8v4": (8, 4), "k3v4": (3, 4), "3bit": (3, 3)}
DTYPES = {"bf16": torch.bfloat16, "fp16": torch.float16, "fp32": torch.float32}
MOST_SCORES = 32 * 2048 * 34816           # scores of the largest chunk case, chunks and contexts at their longest
MOST_ROWS = 8192 * 64                     # query rows of a chunk case
MOST_RECORDS = 64 * 8192 * 8              # (token, kv-head) records of a chunk case
MOST_LOAD = 65536 * 8                     # (token, kv-head) records of the largest load case
MOST_MERGE = 16384 * 32                   # rows of the largest merge case

def _ops():
    pkg = os.path.join(os.getcwd(), "turboquant-cuda-decode_amd")
    if pkg not in sys.path:
        sys.path.insert(0, pkg)
    from tq4_decode import ops

    return ops


# ---- cases -----------------------------------------------------------------------------------

def _chunk(name, batch, new, ctx, hq, hk, preset="4bit", layout="soa", dtype="bf16", new_lo=0, ctx_lo=0, block=16,
           window=0, first=0, causal=True, lse=False, sinks=False):
    """``new`` tokens of each sequence behind ``ctx`` cached ones; ``new_lo`` / ``ctx_lo`` > 0: ragged, spread evenly."""
    case = dict(kind="chunk", batch=batch, new=new, ctx=ctx, new_lo=new_lo, ctx_lo=ctx_lo, hq=hq, hk=hk, preset=preset,
                layout=layout, dtype=dtype, block=block, window=window, first=first, causal=causal, lse=lse, sinks=sinks)
    return dict(name=name, **case) if name else case


def _load(name, tokens, hk, preset="4bit", layout="soa", dtype="bf16", block=16, turned=True):
    """``turned``: keys in the basis that they were written in (not with FP8 keys, which are stored in it)."""
    case = dict(kind="load", tokens=tokens, hk=hk, preset=preset, layout=layout, dtype=dtype, block=block, turned=turned)
    return dict(name=name, **case) if name else case


def _merge(name, tokens, hq, dtype="bf16"):
    case = dict(kind="merge", tokens=tokens, hq=hq, dtype=dtype)
    return dict(name=name, **case) if name else case


def listed():
    return [
        # four drafted tokens of one user's short chat: latency
        _chunk("chunk_drafts_b1", 1, 4, 333, 32, 8),
        # drafted tokens of a whole batch, some sequences with one token only: the cache's bytes
        _chunk("chunk_drafts_b64", 64, 8, 8192, 32, 8, new_lo=1, ctx_lo=512),
        # chunks of every length in one step; FP8 keys, fp16 model, group of 8, sink logits, the backend's AoS view
        _chunk("chunk_k8v4_b8", 8, 511, 12007, 64, 8, preset="k8v4", layout="aos_heads", dtype="fp16", new_lo=3,
               ctx_lo=100, sinks=True),
        # prompts through a layer with a sliding window and first tokens that stay visible; group of 6, AoS
        _chunk("chunk_window_b3", 3, 4097, 1500, 48, 8, layout="aos", new_lo=1000, ctx_lo=1, window=1024, first=4),
        # the context behind chunks whose own tokens are attended to unquantised, to be merged; 3-bit cache
        _chunk("chunk_context_3bit", 4, 1000, 10000, 32, 4, preset="3bit", ctx_lo=17, block=32, causal=False, lse=True),
        # a whole prompt
        _chunk("chunk_prompt_8192", 1, 8192, 0, 32, 8),
        # the next chunk of a long document
        _chunk("chunk_long_32768", 1, 2048, 32768, 32, 8),
        # a short sequence's cache read back for another engine
        _load("load_200", 200, 8, preset="k3v4", layout="aos", dtype="fp16"),
        # FP8 keys and values for a check in 32 bits, the backend's AoS view
        _load("load_k8v4_9001", 9001, 8, preset="k8v4", layout="aos_heads", dtype="fp32"),
        # a batch's contexts read back for attention over plain keys and values
        _load("load_65536", 65536, 8),
        # drafted tokens' results merged: latency
        _merge("merge_256", 256, 32),
        # a large chunk's results merged
        _merge("merge_8192", 8192, 64, dtype="fp16"),
    ]


def _log_uniform(rng, lo, hi):
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(max(lo, hi))))))))


def draw(rng):
    preset = rng.choice(["4bit", "4bit", "4bit", "k8v4", "k3v4", "3bit"])
    layout = rng.choice(["soa", "soa", "aos", "aos_heads"])
    block = rng.choice([16, 16, 32, 64])
    kind = rng.choice(["chunk", "chunk", "chunk", "load", "merge"])
    hk = rng.choice([1, 2, 4, 8, 8])
    group = rng.choice([1, 2, 4, 4, 6, 8, 16]) if hk < 8 else rng.choice([2, 4, 4, 6, 8])
    if kind == "load":
        return _load(None, _log_uniform(rng, 1, MOST_LOAD // hk), hk, preset, layout, rng.choice(["bf16", "bf16", "fp16", "fp32"]),
                     block, rng.random() < 0.75)
    if kind == "merge":
        return _merge(None, _log_uniform(rng, 1, MOST_MERGE // (hk * group)), hk * group, rng.choice(["bf16", "bf16", "fp16", "fp32"]))
    hq = hk * group
    batch = _log_uniform(rng, 1, 128)
    new = _log_uniform(rng, 1, min(8192, math.isqrt(MOST_SCORES // (batch * hq)), MOST_ROWS // (batch * hq),
                                   MOST_RECORDS // (batch * hk)))
    longest = min(MOST_SCORES // (batch * hq * new), MOST_RECORDS // (batch * hk), 65536)
    ctx = _log_uniform(rng, 1, max(1, longest - new)) if rng.random() < 0.9 else 0
    new_lo = max(1, new // 16) if batch > 1 and rng.random() < 0.6 else 0
    ctx_lo = max(1, ctx // 16) if batch > 1 and ctx and rng.random() < 0.6 else 0
    causal = ctx == 0 or rng.random() < 0.8
    window = _log_uniform(rng, 16, 8192) if causal and rng.random() < 0.3 else 0
    first = rng.choice([0, 1, 4, 100]) if window else 0
    return _chunk(None, batch, new, ctx, hq, hk, preset, layout, rng.choice(["bf16", "bf16", "fp16"]), new_lo, ctx_lo, block,
                  window, first, causal, not causal, causal and rng.random() < 0.2)


# ---- inputs ----------------------------------------------------------------------------------

def _generator(seed):
    return torch.Generator(device="cuda").manual_seed(int(seed) % (1 << 62))


def _rotation(gen):
    q, r = torch.linalg.qr(torch.randn(D, D, generator=gen, device="cuda", dtype=torch.float64).cpu())
    return (q * torch.sign(torch.diagonal(r))).float().cuda().contiguous()


def _lloyd_max(bits, sigma=1.0 / math.sqrt(D)):
    """Centroids of the Lloyd-Max quantiser of N(0, sigma^2) with 2^bits levels."""
    n = 1 << bits
    pdf = lambda x: math.exp(-0.5 * x * x) / math.sqrt(2 * math.pi)  # noqa: E731
    cdf = lambda x: 0.5 * math.erfc(-x / math.sqrt(2))  # noqa: E731
    c = [-3.0 + 6.0 * (i + 0.5) / n for i in range(n)]
    for _ in range(300):
        edge = [-12.0] + [(a + b) / 2 for a, b in zip(c, c[1:])] + [12.0]
        c = [(pdf(a) - pdf(b)) / (cdf(b) - cdf(a)) for a, b in zip(edge, edge[1:])]
    return [x * sigma for x in c]


_BOOKS = {}


def _codebook(preset):
    """(centroids, midpoints) of the preset's keys, None and None for FP8 keys."""
    bits = BITS[preset][0]
    if bits == 8:
        return None, None
    if bits not in _BOOKS:
        _BOOKS[bits] = torch.tensor(_lloyd_max(bits), dtype=torch.float32)
    c = _BOOKS[bits].cuda()
    return c, (c[:-1] + c[1:]) * 0.5


def _slot_bytes(preset):
    kb, vb = BITS[preset]
    return D * kb // 8 + (0 if preset == "k8v4" else 2) + D * vb // 8 + 4


def _pack(codes, bits):
    """Codes [..., 128] -> bytes, least significant bits first."""
    if bits == 8:
        return codes
    if bits == 4:
        return codes[..., 0::2] | (codes[..., 1::2] << 4)
    c = codes.reshape(codes.shape[:-1] + (D // 8, 8)).to(torch.int32)
    word = (c << (3 * torch.arange(8, device=c.device, dtype=torch.int32))).sum(-1, dtype=torch.int32)
    out = torch.stack([word & 255, (word >> 8) & 255, word >> 16], dim=-1).to(torch.uint8)
    return out.reshape(codes.shape[:-1] + (D * 3 // 8,))


def _unpack(b, bits):
    """Bytes [..., bits * 16] -> codes [..., 128]."""
    if bits == 4:
        return torch.stack([b & 15, b >> 4], dim=-1).flatten(-2)
    w = b.reshape(b.shape[:-1] + (D // 8, 3)).to(torch.int32)
    word = w[..., 0] | (w[..., 1] << 8) | (w[..., 2] << 16)
    return ((word[..., None] >> (3 * torch.arange(8, device=b.device, dtype=torch.int32))) & 7).flatten(-2)


def _lay_out(k, v, fields, layout):
    """Blocks [n, bs * hk * slot] from K / V bytes [n, bs, hk, .] and fp16 scalars [n, bs, hk] (SoA: data
    records, then [hk][field][bs]; AoS: K, norm, V, scale, zero in each slot)."""
    n = k.shape[0]
    as_bytes = lambda t: t.contiguous().view(torch.uint8)  # noqa: E731
    if layout == "soa":
        meta = torch.stack([f.transpose(1, 2) for f in fields], dim=2)  # [n, hk, field, bs]
        return torch.cat([torch.cat([k, v], dim=-1).reshape(n, -1), as_bytes(meta).reshape(n, -1)], dim=1)
    cells = [as_bytes(f.unsqueeze(-1)) for f in fields]
    slots = torch.cat([k] + cells[:-2] + [v] + cells[-2:], dim=-1)
    return (slots.transpose(1, 2) if layout == "aos_heads" else slots).reshape(n, -1)


def _fill_cache(case, gen, blocks, keep):
    """A cache of what the writer leaves for Gaussian keys and values, and with `keep` also the codes and scalars."""
    bs, hk, preset, layout = case["block"], case["hk"], case["preset"], case["layout"]
    kb, vb = BITS[preset]
    cents, mids = _codebook(preset)
    cache = torch.empty(blocks, bs * hk * _slot_bytes(preset), dtype=torch.uint8, device="cuda")
    kept = []
    step = max(1, (1 << 25) // (bs * hk * D))
    for b0 in range(0, blocks, step):
        shape = (min(step, blocks - b0), bs, hk)
        x = torch.randn(shape + (D,), generator=gen, device="cuda")
        fields = []
        if preset == "k8v4":
            kc = x.to(torch.float8_e4m3fn).view(torch.uint8)
        else:
            kc = torch.bucketize(x * (1.0 / math.sqrt(D)), mids, right=True, out_int32=True)
            norm = 8.0 + 6.0 * torch.rand(shape, generator=gen, device="cuda")
            if layout == "soa":  # the norm of the decoded direction folded in
                norm = norm / cents[kc].square().sum(-1).sqrt()
            fields.append(norm.half())
            kc = kc.to(torch.uint8)
        x = torch.randn(shape + (D,), generator=gen, device="cuda")
        zero, top = x.amin(-1), (1 << vb) - 1
        scale = (x.amax(-1) - zero) / top
        vc = ((x - zero[..., None]) / scale[..., None] + 0.5).clamp(0, top).to(torch.uint8)
        fields += [scale.half(), zero.half()]
        cache[b0:b0 + shape[0]] = _lay_out(_pack(kc, kb), _pack(vc, vb), fields, layout)
        if keep:
            kept.append((kc, vc, fields))
    raw = None
    if keep:
        raw = (torch.cat([k for k, _, _ in kept]), torch.cat([v for _, v, _ in kept]),
               [torch.cat([f[i] for _, _, f in kept]) for i in range(len(kept[0][2]))])
    if layout == "aos_heads":
        return cache.view(blocks, hk, bs, -1).transpose(1, 2), raw
    return cache.view(blocks, bs, hk, -1), raw


def _lengths(n, lo, hi):
    """n lengths in increasing order (a seed permutes them)."""
    return [hi] * n if lo <= 0 or n == 1 else [lo + (hi - lo) * i // (n - 1) for i in range(n)]


def _pairs_of(case):
    """(new tokens, cached tokens in all) of each sequence, in increasing order."""
    n = case["batch"]
    news, contexts = _lengths(n, case["new_lo"], case["new"]), _lengths(n, case["ctx_lo"], case["ctx"])
    return [(a, c + a if case["causal"] else c) for a, c in zip(news, contexts)]


def _chunk_inputs(case, seed, keep=False):
    gen = _generator(seed)
    bs, n = case["block"], case["batch"]
    pairs = _pairs_of(case)
    pairs = [pairs[i] for i in torch.randperm(n, generator=gen, device="cuda").cpu().tolist()]
    lens = torch.tensor([p[1] for p in pairs], dtype=torch.int32)
    starts = torch.zeros(n + 1, dtype=torch.int32)
    starts[1:] = torch.cumsum(torch.tensor([p[0] for p in pairs]), 0)
    width = -(-int(lens.max()) // bs)
    counts = (lens.long() + bs - 1) // bs
    pool = int(counts.sum())
    pages = torch.randperm(pool, generator=gen, device="cuda").to(torch.int32).cpu()
    table = torch.zeros(n, width, dtype=torch.int32)
    table[torch.arange(width)[None] < counts[:, None]] = pages
    cache, raw = _fill_cache(case, gen, pool, keep)
    query = torch.randn(int(starts[-1]), case["hq"], D, generator=gen, device="cuda").to(DTYPES[case["dtype"]])
    sinks = torch.randn(case["hq"], generator=gen, device="cuda") if case["sinks"] else None
    return dict(query=query, cache=cache, table=table.cuda(), lens=lens.cuda(), starts=starts.cuda(), pi_t=_rotation(gen),
                sinks=sinks, raw=raw)


def _load_inputs(case, seed, keep=False):
    gen = _generator(seed)
    n, bs = case["tokens"], case["block"]
    blocks = (n + bs - 1) // bs + 7
    pages = torch.randperm(blocks, generator=gen, device="cuda")
    slots = (pages[:, None] * bs + torch.arange(bs, device="cuda")).reshape(-1)[:n].to(torch.int32)
    cache, raw = _fill_cache(case, gen, blocks, keep)
    return dict(cache=cache, slots=slots, pi_t=_rotation(gen), raw=raw)


def _merge_inputs(case, seed):
    gen = _generator(seed)
    shape, dtype = (case["tokens"], case["hq"]), DTYPES[case["dtype"]]
    x = {}
    for part, tokens in (("a", 2048.0), ("b", 300.0)):
        x["out_" + part] = (torch.randn(shape + (D,), generator=gen, device="cuda") * 0.1).to(dtype)
        x["lse_" + part] = math.log(tokens) + torch.randn(shape, generator=gen, device="cuda")
    # tokens of sequences without a context: nothing in it
    none = torch.rand(case["tokens"], generator=gen, device="cuda") < 0.05
    x["out_a"][none], x["lse_a"][none] = 0, -math.inf
    return x


def prepare(case, seed):
    s = types.SimpleNamespace(case=case)
    if case["kind"] != "merge":
        s.cents, _ = _codebook(case["preset"])
        s.kb, s.vb = BITS[case["preset"]]
    s.kept = None  # the workspaces that a server keeps from step to step
    inputs = {"chunk": _chunk_inputs, "load": _load_inputs, "merge": _merge_inputs}[case["kind"]]
    for name, value in inputs(case, seed).items():
        setattr(s, name, value)
    if case["kind"] == "chunk":  # the places of the rows among sequences padded to the longest chunk
        counts = (s.starts[1:] - s.starts[:-1]).long()
        seq = torch.repeat_interleave(torch.arange(case["batch"], device="cuda"), counts)
        s.place = seq * case["new"] + torch.arange(len(seq), device="cuda") - s.starts.long()[seq]
        s.counts = counts
    return s


# ---- plain forms -----------------------------------------------------------------------------

def _read(s, block, off):
    """K and V [..., hk, 128] in 32 bits of the tokens at places `off` of pages `block`."""
    case, cache, cents = s.case, s.cache, s.cents
    bs, hk = case["block"], case["hk"]
    kbytes, vbytes = D * s.kb // 8, D * s.vb // 8
    if case["layout"] == "soa":
        rec, nf = kbytes + vbytes, 2 if s.kb == 8 else 3
        flat = cache.view(cache.shape[0], -1)
        data = flat[:, :bs * hk * rec].view(-1, bs, hk, rec)[block, off]
        meta = flat[:, bs * hk * rec:].view(torch.float16).view(-1, hk, nf, bs)[block, :, :, off].float()
        k, v = data[..., :kbytes], data[..., kbytes:]
        norm, scale, zero = (meta[..., i - 3 + nf] if i - 3 + nf >= 0 else None for i in range(3))
    else:
        slot = cache[block, off]
        half = lambda a: slot[..., a:a + 2].contiguous().view(torch.float16).float()[..., 0]  # noqa: E731
        skip = 0 if s.kb == 8 else 2
        k, v = slot[..., :kbytes], slot[..., kbytes + skip:kbytes + skip + vbytes]
        norm = half(kbytes) if skip else None
        scale, zero = half(kbytes + skip + vbytes), half(kbytes + skip + vbytes + 2)
    if s.kb == 8:
        k = k.contiguous().view(torch.float8_e4m3fn).float()
    else:
        k = cents[_unpack(k, s.kb).long()]
        if case["layout"] != "soa":
            norm = norm / (k.square().sum(-1) + 1e-16).sqrt()
        k = k * norm[..., None]
    return k, _unpack(v, s.vb).float() * scale[..., None] + zero[..., None]


def _plain_chunk(s):
    case = s.case
    n, new, hq, hk, bs = case["batch"], case["new"], case["hq"], case["hk"], case["block"]
    group, longest = hq // hk, s.table.shape[1] * bs
    # keys and values of every sequence, padded to the table's width
    t = torch.arange(longest, device="cuda")
    lens = s.lens.long()[:, None]
    k, v = _read(s, s.table.long()[:, t // bs], (t % bs)[None])
    k, v = k.transpose(1, 2).contiguous(), v.transpose(1, 2).contiguous()     # [n, hk, longest, D]
    # query rows [n, hk, new * group, D], chunks padded to the longest
    q = s.query.float()
    if s.kb != 8:
        q = torch.matmul(q.reshape(-1, D), s.pi_t).reshape(-1, hq, D)
    rows = torch.zeros(n * new, hq, D, device="cuda")
    rows[s.place] = q * (1.0 / math.sqrt(D))
    rows = rows.reshape(n, new, hk, group, D).transpose(1, 2).reshape(n, hk, new * group, D)
    scores = torch.matmul(rows, k.transpose(2, 3)).reshape(n, hk, new, group, longest)
    # what each new token sees: not past the sequence (causal: itself), in its window or among the first tokens
    i = torch.arange(new, device="cuda")[None]
    end = lens - s.counts[:, None] + i + 1 if case["causal"] else lens.expand(n, new)
    seen = (t < end[..., None]) & (t < lens[..., None])
    if case["window"]:
        seen &= (t >= end[..., None] - case["window"]) | (t < case["first"])
    scores.masked_fill_(~seen[:, None, :, None], -math.inf)
    top = scores.amax(-1, keepdim=True)
    if s.sinks is not None:
        sink = s.sinks.reshape(1, hk, 1, group, 1)
        top = torch.maximum(top, sink)
    top = torch.clamp(top, min=torch.finfo(torch.float32).min)                # (padding rows see nothing)
    p = scores.sub_(top).exp_()
    total = p.sum(-1, keepdim=True)
    if s.sinks is not None:
        total = total + torch.exp(sink - top)
    out = torch.matmul(p.reshape(n, hk, new * group, longest), v).reshape(n, hk, new, group, D) / total
    out = out.transpose(1, 2).reshape(n * new, hq, D)[s.place].to(s.query.dtype)
    if not case["lse"]:
        return out
    lse = (top + total.log()).squeeze(-1).transpose(1, 2).reshape(n * new, hq)[s.place]
    return out, lse


def _plain_load(s):
    case, bs = s.case, s.case["block"]
    slots = s.slots.long()
    k, v = _read(s, slots // bs, slots % bs)
    if s.kb != 8 and case["turned"]:
        k = torch.matmul(k.reshape(-1, D), s.pi_t.t()).reshape(k.shape)
    dtype = DTYPES[case["dtype"]]
    return k.to(dtype), v.to(dtype)


def _plain_merge(s):
    top = torch.maximum(s.lse_a, s.lse_b)
    wa, wb = torch.exp(s.lse_a - top), torch.exp(s.lse_b - top)
    total = wa + wb
    out = (s.out_a.float() * wa[..., None] + s.out_b.float() * wb[..., None]) / total[..., None]
    return out.to(s.out_a.dtype), top + total.log()


# ---- the framework's calls -------------------------------------------------------------------

def _layout(case):
    return "soa" if case["layout"] == "soa" else "aos"


def _own_chunk(s):
    case, ops = s.case, _ops()
    if s.kept is None:
        s.kept = ops.ChunkWorkspace(s.query.shape[0], case["batch"], case["hq"], case["hk"], s.query.device, s.query.dtype)
    return ops.chunk_attention(s.query, None if s.kb == 8 else s.pi_t, s.cache, s.table, s.lens, s.starts, s.cents,
                               causal=case["causal"], window=case["window"], first_tokens=case["first"], key_bits=s.kb,
                               value_bits=s.vb, layout=_layout(case), return_lse=case["lse"], workspace=s.kept, sinks=s.sinks)


def _own_load(s):
    case = s.case
    return _ops().cache_load(s.cache, s.slots, s.pi_t if case["turned"] and s.kb != 8 else None, s.cents, key_bits=s.kb,
                             value_bits=s.vb, layout=_layout(case), dtype=DTYPES[case["dtype"]])


def _own_merge(s):
    return _ops().merge_states(s.out_a, s.lse_a, s.out_b, s.lse_b)


def run(s):
    kind = s.case["kind"]
    if own:
        return {"chunk": _own_chunk, "load": _own_load, "merge": _own_merge}[kind](s)
    return {"chunk": _plain_chunk, "load": _plain_load, "merge": _plain_merge}[kind](s)


# ---- what a pass cannot do without -----------------------------------------------------------

def _seen(case, new, length):
    """(visible (new token, cached token) pairs, cached tokens that any new one sees) of a sequence."""
    if not case["causal"]:
        return new * length, length
    if not case["window"]:
        return sum(range(length - new + 1, length + 1)), length
    low = [max(0, e - case["window"]) for e in range(length - new + 1, length + 1)]
    pairs = sum(e - a + min(a, case["first"]) for a, e in zip(low, range(length - new + 1, length + 1)))
    return pairs, length - low[0] + min(low[0], case["first"])


def work(case):
    size = 4 if case["dtype"] == "fp32" else 2
    if case["kind"] == "merge":
        rows = case["tokens"] * case["hq"]
        return {"bytes": rows * (3 * D * size + 12), "flops": 4 * rows * D}
    slot = _slot_bytes(case["preset"])
    turned = case["preset"] != "k8v4" and case.get("turned", True)
    if case["kind"] == "load":
        records = case["tokens"] * case["hk"]
        return {"bytes": records * (slot + 2 * D * size) + 4 * case["tokens"] + (4 * D * D if turned else 0),
                "flops": records * (2 * D * D if turned else D) + 2 * records * D}
    spans = _pairs_of(case)
    seen = [_seen(case, a, c) for a, c in spans]
    rows = sum(a for a, _ in spans) * case["hq"]
    tokens = sum(x[1] for x in seen)
    moved = tokens * case["hk"] * slot + 4 * (tokens // case["block"]) + rows * (2 * D * size + (4 if case["lse"] else 0))
    return {"bytes": moved + (4 * D * D if turned else 0),
            "flops": 4 * sum(x[0] for x in seen) * case["hq"] * D + (2 * rows * D * D if turned else 0)}


# ---- the definition in 64 bits ---------------------------------------------------------------

def _records(case, raw, pages, places):
    """K and V [tokens, hk, 128] from the codes and scalars that the cache was made of."""
    kc, vc, fields = raw
    if case["preset"] == "k8v4":
        k = kc[pages, places].view(torch.float8_e4m3fn).double()
    else:
        k = _codebook(case["preset"])[0].double()[kc[pages, places].long()]
        if case["layout"] != "soa":
            k = k / (k.square().sum(-1, keepdim=True) + 1e-16).sqrt()
        k = k * fields[0][pages, places].double()[..., None]
    v = vc[pages, places].double() * fields[-2][pages, places].double()[..., None] + fields[-1][pages, places].double()[..., None]
    return k, v


def _exact_chunk(case, seed):
    x = _chunk_inputs(case, seed, keep=True)
    hq, hk, bs = case["hq"], case["hk"], case["block"]
    group = hq // hk
    out = torch.zeros(x["query"].shape, dtype=torch.float64, device="cuda")
    lses = torch.zeros(x["query"].shape[:2], dtype=torch.float64, device="cuda")
    starts = x["starts"].tolist()
    for b, length in enumerate(x["lens"].tolist()):
        t = torch.arange(length, device="cuda")
        k, v = _records(case, x["raw"], x["table"][b].long()[t // bs], t % bs)
        for r0 in range(starts[b], starts[b + 1], 2048):
            r1 = min(starts[b + 1], r0 + 2048)
            q = x["query"][r0:r1].double() / math.sqrt(D)
            if case["preset"] != "k8v4":
                q = torch.matmul(q.reshape(-1, D), x["pi_t"].double()).reshape(q.shape)
            position = torch.arange(r0, r1, device="cuda") - starts[b + 1] + length     # of the new token itself
            hidden = torch.zeros(r1 - r0, length, dtype=torch.bool, device="cuda")
            if case["causal"]:
                hidden |= t > position[:, None]
            if case["window"]:
                hidden |= (t <= position[:, None] - case["window"]) & (t >= case["first"])
            for h in range(hk):
                scores = torch.matmul(q[:, h * group:(h + 1) * group].reshape(-1, D), k[:, h].t().contiguous())
                scores = scores.reshape(r1 - r0, group, length).masked_fill(hidden[:, None], -math.inf)
                if x["sinks"] is not None:
                    sink = x["sinks"][h * group:(h + 1) * group].double().reshape(1, group, 1).expand(r1 - r0, -1, -1)
                    scores = torch.cat([sink, scores], dim=-1)
                lse = torch.logsumexp(scores, dim=-1, keepdim=True)
                p = torch.exp(scores - lse)[..., 0 if x["sinks"] is None else 1:]
                out[r0:r1, h * group:(h + 1) * group] = torch.matmul(p.reshape(-1, length), v[:, h].contiguous()).reshape(
                    r1 - r0, group, D)
                lses[r0:r1, h * group:(h + 1) * group] = lse[..., 0]
    return (out, lses) if case["lse"] else out


def _exact_load(case, seed):
    x = _load_inputs(case, seed, keep=True)
    slots = x["slots"].long()
    k, v = _records(case, x["raw"], slots // case["block"], slots % case["block"])
    if case["preset"] != "k8v4" and case["turned"]:
        k = torch.matmul(k.reshape(-1, D), x["pi_t"].double().t().contiguous()).reshape(k.shape)
    return k, v


def _exact_merge(case, seed):
    x = _merge_inputs(case, seed)
    lse = torch.logaddexp(x["lse_a"].double(), x["lse_b"].double())
    share = torch.exp(x["lse_a"].double() - lse)[..., None]
    return x["out_a"].double() * share + x["out_b"].double() * (1 - share), lse


def exact(case, seed):
    return {"chunk": _exact_chunk, "load": _exact_load, "merge": _exact_merge}[case["kind"]](case, seed)
