"""What the entries with rotary positions, windows and shared prefixes refuse before any GPU work: the C
entries' status and message, and the wrappers' checks."""
import ctypes

import pytest
import torch

from tq4_decode import _lib, ops

P = 1 << 12  # an aligned address that no refused call reads
MOST = 0x7FFFFFFF


def message():
    return _lib.load().tq4_last_error().decode()


def _span(name, over):
    """A valid call's arguments up to the pointer that makes it invalid: sequences of 4 blocks of 16, 8 / 2 heads."""
    a = dict(query=P, qd=1, rot=P, cents=P, cache=P, table=P, lens=P, ws=P, mid=P, floats=1 << 30, out=P, od=1, lse=P,
             B=2, Hq=8, Hk=2, D=128, bs=16, width=4, stride=16 * 2 * 134, S=4, layout=0, scale=0.1, kb=4, vb=4,
             window=32, first=0, prefix=32, kernel=4)
    a.update(over)
    head = [a[n] for n in ("query", "qd", "rot", "cents", "cache", "table", "lens", "ws")]
    head += [a["mid"]] if name == "window" else [a["floats"]]
    mid = [a[n] for n in ("out", "od", "lse", "B", "Hq", "Hk", "D", "bs", "width", "stride", "S", "layout", "scale")]
    tail = [None, a["kb"], a["vb"]] + ([a["window"], a["first"]] if name == "window" else [a["prefix"], a["kernel"]]) + [None]
    return getattr(_lib.load(), f"tq4_{name}_decode")(*head, *mid, *tail)


BOTH = [
    (dict(query=None), 1, "null pointer"), (dict(out=None), 1, "null pointer"), (dict(lse=None), 1, "null pointer"),
    (dict(ws=None), 1, "null pointer"), (dict(rot=None), 1, "null pointer"), (dict(cents=None), 1, "null pointer"),
    (dict(cache=None), 1, "null pointer"), (dict(table=None), 1, "null pointer"), (dict(lens=None), 1, "null pointer"),
    (dict(kb=5), 2, "unsupported"), (dict(kb=8, vb=3), 2, "unsupported"), (dict(kb=4, vb=3), 2, "unsupported"),
    (dict(qd=3), 1, "query_dtype"), (dict(od=-1), 1, "out_dtype"), (dict(query=P + 8), 1, "16-byte"),
    (dict(cache=P + 2), 1, "16-byte"), (dict(B=0), 1, "positive"), (dict(S=0), 1, "positive"), (dict(width=0), 1, "positive"),
    (dict(B=65536), 2, "65535"), (dict(S=65537), 2, "65536"), (dict(Hq=7), 1, "multiple of Hk"), (dict(D=64), 2, "head_dim"),
    (dict(layout=3), 1, "layout"), (dict(stride=16 * 2 * 134 - 16), 1, "block stride"), (dict(scale=0.0), 1, "attn_scale"),
    (dict(scale=float("nan")), 1, "attn_scale"), (dict(bs=8, stride=8 * 2 * 134 + 8), 2, "block_size"),
    (dict(bs=24, stride=24 * 2 * 134), 2, "block_size"), (dict(stride=16 * 2 * 134 + 2), 2, "block stride"),
]


@pytest.mark.parametrize("over,code,text", BOTH)
@pytest.mark.parametrize("name", ["window", "prefix"])
def test_decode_entries_refuse(name, over, code, text):
    assert _span(name, over) == code
    assert text in message()


@pytest.mark.parametrize("over", [dict(window=0), dict(window=-MOST), dict(first=-1)])
def test_window_refuses(over):
    assert _span("window", over) == 1 and "window" in message()


@pytest.mark.parametrize("over,code,text", [
    (dict(prefix=-16), 1, "whole blocks"), (dict(prefix=8), 1, "whole blocks"), (dict(prefix=80), 1, "whole blocks"),
    (dict(prefix=MOST - 15), 1, "whole blocks"), (dict(floats=1000), 1, "workspace"), (dict(ws=P + 4), 1, "aligned"),
    (dict(qd=0), 2, "16-bit"), (dict(od=0), 2, "16-bit"), (dict(kernel=1), 1, "kernel"), (dict(kernel=-1), 1, "kernel"),
])
def test_prefix_refuses(over, code, text):
    assert _span("prefix", over) == code
    assert text in message()


def test_prefix_workspace():
    size = _lib.load().tq4_prefix_workspace_floats
    for bad in ((0, 8, 2, 4), (2, 0, 2, 4), (2, 8, 0, 4), (2, 7, 2, 4), (2, 8, 2, 0), (-1, 8, 2, 4)):
        assert size(*bad) == -1 and "positive" in message()
    # q rows, the sequences' parts, at least one part of the prefix per row
    for b, hq, hk, s in ((1, 1, 1, 1), (2, 8, 2, 4), (64, 32, 8, 16), (256, 64, 4, 32), (65535, 128, 8, 64)):
        floats = size(b, hq, hk, s)
        assert b * hq * (128 + (s + 1) * 129) <= floats <= b * hq * (128 + (s + 64) * 129) + 3 * 64


def _append(**over):
    a = dict(q=P, qo=P, k=P, v=P, dt=1, qs=1024, ks=256, vs=256, pos=P, ax_stride=8, axes=1, axis_of=None, table=P, td=0,
             rows=100, rot=128, neox=1, slots=P, pit=P, mids=P, cents=P, cache=P, blocks=4, N=8, Hq=8, Hk=2, D=128, bs=16,
             stride=16 * 2 * 134, layout=0, nc=1, kb=4, vb=4)
    a.update(over)
    return _lib.load().tq4_rope_store(*[a[n] for n in (
        "q", "qo", "k", "v", "dt", "qs", "ks", "vs", "pos", "ax_stride", "axes", "axis_of", "table", "td", "rows", "rot", "neox",
        "slots", "pit", "mids", "cents", "cache", "blocks", "N", "Hq", "Hk", "D", "bs", "stride", "layout", "nc", "kb", "vb")], None)


@pytest.mark.parametrize("over,code,text", [
    (dict(k=None), 1, "null pointer"), (dict(v=None), 1, "null pointer"), (dict(pos=None), 1, "null pointer"),
    (dict(table=None), 1, "null pointer"), (dict(slots=None), 1, "null pointer"), (dict(cache=None), 1, "null pointer"),
    (dict(qo=None), 1, "null pointer"), (dict(q=None), 1, "null pointer"), (dict(pit=None), 1, "null pointer"),
    (dict(mids=None), 1, "null pointer"), (dict(cents=None), 1, "centroids"), (dict(kb=2), 2, "unsupported"),
    (dict(dt=3), 1, "dtype"), (dict(td=2), 1, "cos_sin_dtype"), (dict(N=-1), 1, "N and num_blocks"),
    (dict(Hk=0), 1, "N and num_blocks"), (dict(Hq=0), 1, "N and num_blocks"), (dict(rows=0), 1, "N and num_blocks"),
    (dict(blocks=-1), 1, "N and num_blocks"), (dict(D=256), 2, "head_dim"), (dict(rot=24), 2, "rot_dim"),
    (dict(rot=0), 2, "rot_dim"), (dict(rot=144), 2, "rot_dim"), (dict(axes=0), 1, "axes"), (dict(axes=5), 1, "axes"),
    (dict(axes=2), 1, "axis_of"), (dict(layout=-1), 1, "layout"), (dict(stride=100), 1, "block stride"),
    (dict(stride=16 * 2 * 134 + 8), 1, "block stride"), (dict(k=P + 8), 1, "16-byte"), (dict(table=P + 4), 1, "16-byte"),
    (dict(qo=P + 2), 1, "16-byte"), (dict(ks=260), 1, "strides"), (dict(qs=-8), 1, "strides"), (dict(vs=2), 1, "strides"),
    (dict(N=MOST // 2), 1, "32-bit"),
])
def test_append_refuses(over, code, text):
    assert _append(**over) == code
    assert text in message()


@pytest.mark.parametrize("bad", [-1, 3])
def test_append_refuses_axes_out_of_range(bad):
    axes = (ctypes.c_int32 * 64)(*([0] * 63 + [bad]))
    assert _append(axes=3, axis_of=axes) == 1
    assert "axis_of[63]" in message()


def test_no_tokens_need_no_gpu():
    assert _append(N=0) == 0 and message() == ""


def test_wrappers_refuse_on_the_cpu():
    q = torch.zeros(2, 8, 128, dtype=torch.bfloat16)
    cache = torch.zeros(4, 16, 2, 134, dtype=torch.uint8)
    table, lens = torch.zeros(2, 4, dtype=torch.int32), torch.zeros(2, dtype=torch.int32)
    span = (q, torch.zeros(128, 128), cache, table, lens, torch.zeros(16), 4)
    for window in (0, -1, 2 ** 31, 1.5, True, None):
        with pytest.raises(RuntimeError, match="window"):
            ops.window_decode(*span, window)
    with pytest.raises(RuntimeError, match="first_tokens"):
        ops.window_decode(*span, 4, first_tokens=-1)
    for prefix in (-16, 2 ** 31, 16.0, False):
        with pytest.raises(RuntimeError, match="prefix_len"):
            ops.prefix_decode(*span, prefix)
    with pytest.raises(RuntimeError, match="invalid query"):  # a tensor on the CPU
        ops.window_decode(*span, 4)
    with pytest.raises(RuntimeError, match="invalid query"):
        ops.prefix_decode(*span, 16)
    k = torch.zeros(2, 2, 128, dtype=torch.bfloat16)
    pos, slots = torch.zeros(2, dtype=torch.int64), torch.zeros(2, dtype=torch.int32)
    with pytest.raises(RuntimeError):
        ops.rope_store(q, k, k, pos, torch.zeros(4, 128), cache, slots)
    with pytest.raises(RuntimeError, match="key/value bits"):
        ops.rope_store(q, k, k, pos, torch.zeros(4, 128), cache, slots, key_bits=2)
    with pytest.raises(_lib.Tq4Error, match="multiple of Hk"):
        ops.PrefixWorkspace(2, 7, 2, 4, torch.device("cpu"))
