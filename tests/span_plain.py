"""Caches of random codes in every preset and layout, with the keys and values they stand for in
float64, and plain attention over them: what the tests of the windowed, shared-prefix and position-
rotating entries compare with."""
import numpy as np
import torch

from tq4_decode import codebook

D = 128
PRESETS = {"4bit": (4, 4), "k8v4": (8, 4), "k3v4": (3, 4), "3bit": (3, 3)}


def slot_bytes(kb, vb):
    return 16 * kb + (0 if kb == 8 else 2) + 16 * vb + 4


def pack(codes, bits):
    """Codes [..., 128] -> bytes, least significant bit first."""
    if bits == 8:
        return codes.astype(np.uint8)
    b = ((codes[..., None].astype(np.uint8) >> np.arange(bits, dtype=np.uint8)) & 1).reshape(codes.shape[:-1] + (-1,))
    return np.packbits(b, axis=-1, bitorder="little")


def unpack(data, bits):
    """Bytes [..., 16 bits] -> codes [..., 128]."""
    if bits == 8:
        return data
    b = np.unpackbits(data, axis=-1, bitorder="little").reshape(data.shape[:-1] + (D, bits))
    return (b * (1 << np.arange(bits))).sum(-1)


def e4m3(data):
    return torch.from_numpy(np.ascontiguousarray(data)).view(torch.float8_e4m3fn).double().numpy()


def split_cache(cache, kb, vb, layout):
    """(K codes, V codes, fp16 scalar fields) [blocks, bs, hk, .] of cache bytes [blocks, bs, hk, slot] (SoA:
    any view of the blocks' bytes)."""
    n, bs, hk, slot = cache.shape
    nk, nv, nf = 16 * kb, 16 * vb, 2 if kb == 8 else 3
    if layout == "soa":
        flat = np.ascontiguousarray(cache).reshape(n, -1)
        rec = flat[:, :bs * hk * (nk + nv)].reshape(n, bs, hk, nk + nv)
        meta = np.ascontiguousarray(flat[:, bs * hk * (nk + nv):]).view(np.float16).reshape(n, hk, nf, bs)
        return unpack(rec[..., :nk], kb), unpack(rec[..., nk:], vb), [meta[:, :, i].transpose(0, 2, 1) for i in range(nf)]
    skip = 0 if kb == 8 else 2
    field = lambda a: np.ascontiguousarray(cache[..., a:a + 2]).view(np.float16)[..., 0]  # noqa: E731
    at = nk + skip + nv
    return (unpack(cache[..., :nk], kb), unpack(cache[..., nk + skip:at], vb),
            ([field(nk)] if skip else []) + [field(at), field(at + 2)])


def values_of(kc, vc, fields, kb, layout):
    """Keys and values [blocks, bs, hk, 128] in float64."""
    f = [x.astype(np.float64)[..., None] for x in fields]
    if kb == 8:
        k = e4m3(kc.astype(np.uint8))
    else:
        k = codebook.centroids(D, kb).astype(np.float64)[kc]
        if layout != "soa":
            k = k / np.sqrt((k * k).sum(-1, keepdims=True) + 1e-16)
        k = k * f[0]
    return k, vc * f[-2] + f[-1]


def make_cache(rng, blocks, bs, hk, preset, layout):
    """(cache tensor on the CPU, as a backend passes it; K, V [blocks, bs, hk, 128] in float64)."""
    kb, vb = PRESETS[preset]
    shape = (blocks, bs, hk)
    if kb == 8:
        kc = (torch.randn(shape + (D,), generator=torch.Generator().manual_seed(int(rng.integers(1 << 30)))) * 1.3).to(
            torch.float8_e4m3fn).view(torch.uint8).numpy()
    else:
        kc = rng.integers(0, 1 << kb, shape + (D,)).astype(np.uint8)
    vc = rng.integers(0, 1 << vb, shape + (D,)).astype(np.uint8)
    fields = [] if kb == 8 else [rng.uniform(6.0, 14.0, shape).astype(np.float16)]
    fields += [rng.uniform(0.05, 0.4, shape).astype(np.float16), rng.uniform(-3, 0.2, shape).astype(np.float16)]
    k, v = values_of(kc, vc, fields, kb, layout)
    if layout == "soa":
        rec = np.concatenate([pack(kc, kb), pack(vc, vb)], -1).reshape(blocks, -1)
        meta = np.ascontiguousarray(np.stack([x.transpose(0, 2, 1) for x in fields], 2)).view(np.uint8).reshape(blocks, -1)
        data = torch.from_numpy(np.concatenate([rec, meta], 1)).view(blocks, bs, hk, -1)
        return data, k, v
    cells = [np.ascontiguousarray(x[..., None]).view(np.uint8) for x in fields]
    slots = np.concatenate([pack(kc, kb)] + cells[:-2] + [pack(vc, vb)] + cells[-2:], -1)
    if layout == "aos_heads":
        return torch.from_numpy(np.ascontiguousarray(slots.transpose(0, 2, 1, 3))).transpose(1, 2), k, v
    return torch.from_numpy(np.ascontiguousarray(slots)), k, v


def rotation(rng):
    q, r = np.linalg.qr(rng.standard_normal((D, D)))
    return (q * np.sign(np.diag(r))).astype(np.float32)


def attend(q, k, v, sinks=None, scale=D ** -0.5):
    """q [Hq, 128], k / v [tokens, Hk, 128] in float64 -> (out [Hq, 128], lse [Hq]); no tokens: NaN and -inf."""
    hq, hk = q.shape[0], k.shape[1]
    if k.shape[0] == 0:
        return np.full((hq, D), np.nan), np.full(hq, -np.inf)
    qg = q.reshape(hk, -1, D)
    s = np.einsum("hgd,thd->hgt", qg, k) * scale
    top = s.max(-1, keepdims=True)
    if sinks is not None:
        top = np.maximum(top, sinks.reshape(hk, -1, 1))
    p = np.exp(s - top)
    total = p.sum(-1, keepdims=True)
    if sinks is not None:
        total = total + np.exp(sinks.reshape(hk, -1, 1) - top)
    out = np.einsum("hgt,thd->hgd", p / total, v)
    return out.reshape(hq, D), (top + np.log(total)).reshape(hq)


def close(got, want, step, what, atol=1e-4, rtol=0.0):
    """|got - want| <= atol + (rtol + step) |want|; the same NaNs and infinities."""
    got, want = np.asarray(got, np.float64), np.asarray(want, np.float64)
    fine = np.isfinite(want)
    assert np.array_equal(np.isnan(got), np.isnan(want)), f"{what}: NaNs differ"
    assert np.array_equal(got[~fine & ~np.isnan(want)], want[~fine & ~np.isnan(want)]), f"{what}: infinities differ"
    err = np.abs(got[fine] - want[fine]) - (rtol + step) * np.abs(want[fine])
    assert err.size == 0 or err.max() <= atol, f"{what}: off by {err.max():.3e} over the step, allowed {atol:.1e}"


def spoil(cache, tokens, preset, layout):
    """Every byte of the given (block, offset) tokens set: NaN scalars, the highest codes (E4M3: NaN)."""
    kb, vb = PRESETS[preset]
    n, bs, hk, slot = cache.shape
    nf = 2 if kb == 8 else 3
    rec = 16 * (kb + vb)
    for block, off in tokens:
        if layout != "soa":
            cache[block, off] = 0xFF
            continue
        flat = cache[block].view(-1)
        flat[off * hk * rec:(off + 1) * hk * rec] = 0xFF
        meta = flat[bs * hk * rec:].view(hk, nf, bs, 2)
        meta[:, :, off] = 0xFF
