"""What ``chunk_attention``, ``cache_load`` and ``merge_states`` refuse before any GPU work: the C entries' status and
message, and the wrappers' checks."""
import pytest
import torch

from tq4_decode import _lib, ops

P = 1 << 12  # an aligned address that no refused call reads
MOST = 0x7FFFFFFF


def message():
    return _lib.load().tq4_last_error().decode()


def _chunk(**over):
    """A valid call's arguments but for those given: 10 tokens of 2 sequences of 4 blocks of 16, 8 / 2 heads."""
    a = dict(query=P, qd=1, qs=1024, rot=P, cents=P, cache=P, table=P, lens=P, starts=P, ws=P, floats=1 << 30, out=P, od=1,
             lse=None, T=10, B=2, Hq=8, Hk=2, D=128, bs=16, width=4, stride=16 * 2 * 134, layout=0, scale=0.1, sinks=None,
             kb=4, vb=4, causal=1, window=0, first=0)
    assert set(over) <= set(a)
    a.update(over)
    return _lib.load().tq4_chunk_attention(*a.values(), None)


@pytest.mark.parametrize("over,code,text", [
    (dict(query=None), 1, "null pointer"), (dict(out=None), 1, "null pointer"), (dict(ws=None), 1, "null pointer"),
    (dict(rot=None), 1, "null pointer"), (dict(cents=None), 1, "null pointer"), (dict(cache=None), 1, "null pointer"),
    (dict(table=None), 1, "null pointer"), (dict(lens=None), 1, "null pointer"), (dict(starts=None), 1, "null pointer"),
    (dict(kb=5), 2, "unsupported"), (dict(kb=8, vb=3), 2, "unsupported"), (dict(kb=4, vb=3), 2, "unsupported"),
    (dict(qd=3), 1, "query_dtype"), (dict(od=-1), 1, "out_dtype"), (dict(qd=0), 2, "16-bit"), (dict(od=0), 2, "16-bit"),
    (dict(query=P + 8), 1, "16-byte"), (dict(cache=P + 2), 1, "16-byte"), (dict(out=P + 8), 1, "16-byte"),
    (dict(T=0), 1, "positive"), (dict(T=-1), 1, "positive"), (dict(B=0), 1, "positive"), (dict(width=0), 1, "positive"),
    (dict(B=65536), 2, "65535"), (dict(Hq=7), 1, "multiple of Hk"), (dict(D=64), 2, "head_dim"), (dict(layout=3), 1, "layout"),
    (dict(T=1 << 28), 1, "2^30"), (dict(T=MOST), 1, "2^30"), (dict(qs=1016), 1, "query_stride"), (dict(qs=1028), 1, "query_stride"),
    (dict(qs=-1024), 1, "query_stride"), (dict(stride=16 * 2 * 134 - 16), 1, "block stride"), (dict(stride=1 << 31), 2, "block stride"),
    (dict(stride=16 * 2 * 134 + 2), 2, "block stride"), (dict(scale=0.0), 1, "attn_scale"), (dict(scale=float("inf")), 1, "attn_scale"),
    (dict(bs=8, stride=8 * 2 * 134 + 8), 2, "block_size"), (dict(bs=24, stride=24 * 2 * 134), 2, "block_size"),
    (dict(window=-1), 1, "window"), (dict(first=-1), 1, "first_tokens"), (dict(window=5, causal=0), 1, "window"),
    (dict(floats=1000), 1, "workspace"), (dict(ws=P + 4), 1, "aligned"),
])
def test_chunk_refuses(over, code, text):
    assert _chunk(**over) == code, message()
    assert text in message()


def test_chunk_workspace():
    size = _lib.load().tq4_chunk_workspace_floats
    for bad in ((0, 2, 8, 2), (10, 0, 8, 2), (10, 2, 0, 2), (10, 2, 8, 0), (10, 2, 7, 2), (-1, 2, 8, 2)):
        assert size(*bad) == -1 and "positive" in message()
    assert size(1 << 28, 1, 8, 2) == -1 and "2^30" in message()
    # two f16 rows and a factor a query row, the sequences' work, and the parts of 256 or 512 workgroups
    for t, b, hq, hk in ((1, 1, 1, 1), (4, 1, 32, 8), (256, 64, 32, 8), (40, 4, 32, 8), (8192, 1, 32, 8), (100000, 65535, 64, 4)):
        floats, rows = size(t, b, hq, hk), t * hq
        assert rows * 129 + 2 * b <= floats <= rows * 129 + 2 * b + 2 * 512 * 256 * 129 + 4 * 513 + 8 * 64
        with pytest.raises(_lib.Tq4Error, match="workspace"):
            _lib.check(_chunk(T=t, B=b, Hq=hq, Hk=hk, qs=hq * 128, stride=16 * hk * 134, floats=floats - 1), "chunk")


def _load(**over):
    a = dict(cache=P << 20, slots=P, rot=P, cents=P, key=P, value=P << 4, dt=1, blocks=4, N=8, Hk=2, D=128, bs=16,
             stride=16 * 2 * 134, layout=0, kb=4, vb=4)
    assert set(over) <= set(a)
    a.update(over)
    return _lib.load().tq4_cache_load(*a.values(), None)


@pytest.mark.parametrize("over,code,text", [
    (dict(cache=None), 1, "null pointer"), (dict(slots=None), 1, "null pointer"), (dict(cents=None), 1, "null pointer"),
    (dict(key=None), 1, "null pointer"), (dict(value=None), 1, "null pointer"), (dict(kb=2), 2, "unsupported"),
    (dict(kb=8, vb=3), 2, "unsupported"), (dict(dt=3), 1, "dtype"), (dict(N=0), 1, "positive"), (dict(N=-1), 1, "positive"),
    (dict(Hk=0), 1, "positive"), (dict(bs=0), 1, "positive"), (dict(blocks=0), 1, "positive"), (dict(D=64), 2, "head_dim"),
    (dict(layout=5), 1, "layout"), (dict(stride=16 * 2 * 134 - 2), 1, "block stride"), (dict(stride=16 * 2 * 134 + 1), 1, "odd"),
    (dict(N=1 << 30), 2, "2^30"), (dict(bs=1 << 23, stride=1 << 32), 2, "2^30"), (dict(cache=(P << 20) + 1), 1, "2-byte"),
    (dict(key=P + 8), 1, "16-byte"), (dict(value=P + 2), 1, "16-byte"), (dict(value=P + 16), 1, "overlap"),
    (dict(key=P << 20), 1, "overlap"), (dict(value=(P << 20) + 16 * 100), 1, "overlap"),
])
def test_load_refuses(over, code, text):
    assert _load(**over) == code, message()
    assert text in message()


def _merge(**over):
    a = dict(a=P, la=2 * P, b=3 * P, lb=4 * P, out=5 * P, dt=1, lse=6 * P, rows=4, D=128)
    assert set(over) <= set(a)
    a.update(over)
    return _lib.load().tq4_merge_states(*a.values(), None)


@pytest.mark.parametrize("over,code,text", [
    (dict(a=None), 1, "null pointer"), (dict(la=None), 1, "null pointer"), (dict(b=None), 1, "null pointer"),
    (dict(lb=None), 1, "null pointer"), (dict(out=None), 1, "null pointer"), (dict(lse=None), 1, "null pointer"),
    (dict(dt=3), 1, "dtype"), (dict(rows=0), 1, "positive"), (dict(rows=-5), 1, "positive"), (dict(D=64), 2, "head_dim"),
    (dict(a=P + 8), 1, "16-byte"), (dict(b=3 * P + 2), 1, "16-byte"), (dict(out=5 * P + 4), 1, "16-byte"),
    (dict(out=P + 256), 1, "overlap"), (dict(out=3 * P - 256), 1, "overlap"), (dict(lse=2 * P + 4), 1, "overlap"),
    (dict(lse=4 * P - 8), 1, "overlap"), (dict(lse=5 * P), 1, "overlap"), (dict(lse=P + 16), 1, "overlap"),
    (dict(out=2 * P), 1, "overlap"), (dict(rows=1 << 62), 2, "too many"),
])
def test_merge_refuses(over, code, text):
    assert _merge(**over) == code, message()
    assert text in message()


def test_wrappers_refuse_on_the_cpu():
    q = torch.zeros(10, 8, 128, dtype=torch.bfloat16)
    cache = torch.zeros(4, 16, 2, 134, dtype=torch.uint8)
    table, lens, starts = (torch.zeros(*s, dtype=torch.int32) for s in ((2, 4), (2,), (3,)))
    args = (q, torch.zeros(128, 128), cache, table, lens, starts, torch.zeros(16))
    for window in (-1, 2 ** 31, 1.5, True, None):
        with pytest.raises(RuntimeError, match="window"):
            ops.chunk_attention(*args, window=window)
    with pytest.raises(RuntimeError, match="first_tokens"):
        ops.chunk_attention(*args, first_tokens=-1)
    with pytest.raises(RuntimeError, match="causal"):
        ops.chunk_attention(*args, window=4, causal=False)
    with pytest.raises(RuntimeError, match="key/value bits"):
        ops.chunk_attention(*args, key_bits=2)
    with pytest.raises(RuntimeError, match="invalid query"):  # a tensor on the CPU
        ops.chunk_attention(*args)
    with pytest.raises(_lib.Tq4Error, match="multiple of Hk"):
        ops.ChunkWorkspace(10, 2, 7, 2, torch.device("cpu"))
    with pytest.raises(RuntimeError, match="key/value bits"):
        ops.cache_load(cache, lens, None, torch.zeros(16), key_bits=5)
    with pytest.raises(RuntimeError):
        ops.cache_load(cache, lens, None, torch.zeros(16))
    with pytest.raises(RuntimeError, match="out_a"):
        ops.merge_states(q, q[..., 0].float(), q, q[..., 0].float())
