"""Argument checks of the fixed-rate operators (key/value cache, activation checkpoints): refused before anything is
launched, so all of it runs without a GPU."""
import ctypes as C

import pytest

torch = pytest.importorskip("torch")
ARG, P = -2, 0x1000


@pytest.fixture(scope="module")
def d():
    import dcamd
    return dcamd


@pytest.fixture(scope="module")
def lib(d):
    return d.Lib()


def desc(d, **k):
    a = dict(data=P, pages=4, page_size=16, heads=2, head_dim=64, bits=4)
    a.update(k)
    return d.KvCacheDesc(*(a[n] for n in ("data", "pages", "page_size", "heads", "head_dim", "bits")))


def batch(d, **k):
    a = dict(batch=2, tokens=3, start=P, lens=None, table=P, table_width=2, table_stride=2, zero_padding=0)
    a.update(k)
    return d.KvBatchDesc(*(a[n] for n in ("batch", "tokens", "start", "lens", "table", "table_width", "table_stride", "zero_padding")))


def test_page_bytes(lib):
    f = lib.L.dc_kv_page_bytes
    assert f(16, 2, 64, 4) == 16 * 2 * (2 * 32 + 8) and f(64, 8, 128, 8) == 64 * 8 * (256 + 8)
    for bad in ((0, 2, 64, 4), (15, 2, 64, 4), (24, 2, 64, 4), (-16, 2, 64, 4), (16, 0, 64, 4), (16, 2, 0, 4), (16, 2, 48, 4),
                (16, 2, 288, 4), (16, 2, 64, 5), (16, 2, 64, 0), (1 << 30, 1 << 21, 64, 4)):
        assert f(*bad) == 0, bad


BAD_CACHE = [dict(data=None), dict(data=P + 8), dict(pages=0), dict(pages=-1), dict(pages=1 << 62), dict(page_size=8),
             dict(page_size=40), dict(heads=0), dict(head_dim=65), dict(head_dim=512), dict(bits=3)]
BAD_BATCH = [dict(batch=-1), dict(tokens=-1), dict(start=None), dict(table_width=0), dict(table_stride=1),
             dict(table=None, batch=5)]


@pytest.mark.parametrize("which", ["write", "read", "attention"])
def test_cache_calls(d, lib, which):
    L, st = lib.L, (C.c_longlong * 3)(1000, 200, 64)

    def call(cache=None, at=None, dtype=2, a=P, b=P, sa=st, sb=st, q_heads=4, max_context=32, space=None, size=0):
        c, t = cache or desc(d), at or batch(d)
        if which == "attention":
            return L.dc_kv_attention_device(c, t, dtype, q_heads, a, sa, 0.1, 1, max_context, b, sb, None, space, size, None)
        return getattr(L, f"dc_kv_{which}_device")(c, t, dtype, a, sa, b, sb, None)

    for k in BAD_CACHE:
        assert call(cache=desc(d, **k)) == ARG, k
        assert lib.err()
    for k in BAD_BATCH:
        assert call(at=batch(d, **k)) == ARG, k
    for k in (dict(dtype=3), dict(dtype=-1), dict(a=None), dict(b=None), dict(sa=None), dict(sb=None), dict(a=P + 1), dict(b=P + 1)):
        assert call(**k) == ARG, k
    assert call(at=batch(d, batch=1 << 16, tokens=1 << 16), q_heads=32) == ARG
    assert call(at=batch(d, batch=0, start=None)) == 0 and call(at=batch(d, tokens=0)) == 0     # nothing to do
    if which == "attention":
        for k in (dict(dtype=0), dict(q_heads=0), dict(q_heads=3), dict(q_heads=-2), dict(max_context=-1)):
            assert call(**k) == ARG, k
        need = L.dc_kv_attention_workspace(desc(d), 2, 3, 4, 4096)
        assert need > 0
        for space, size in ((None, 0), (None, need), (P, need - 1), (P + 8, need)):
            assert call(max_context=4096, space=space, size=size) == ARG


def test_workspace(d, lib):
    w = lib.L.dc_kv_attention_workspace
    assert w(desc(d), 1, 1, 2, 100) == 0                                # short: no split
    assert w(desc(d), 4096, 1, 2, 1 << 20) == 0                         # enough sequences: no split
    assert w(desc(d, bits=3), 1, 1, 2, 1 << 20) == 0 and w(desc(d), 1, 1, 3, 1 << 20) == 0 and w(desc(d), 0, 1, 2, 1 << 20) == 0


def test_activation_calls(lib):
    L = lib.L
    assert L.dc_act_bytes(0) == 0 and L.dc_act_bytes(1) == 33 and L.dc_act_bytes(33) == 66 and L.dc_act_bytes(-1) == 0
    assert L.dc_act_bytes(1 << 35) == 0

    def forward(kind=1, dtype=2, rows=4, cols=8, x=P, ldx=8, up=None, ldup=8, y=P, ldy=8, kept=P, kept_up=None):
        return L.dc_act_forward_device(kind, dtype, rows, cols, x, ldx, up, ldup, y, ldy, kept, kept_up, None)

    def backward(kind=1, dtype=2, rows=4, cols=8, dy=P, lddy=8, kept=P, kept_up=None, dx=P, lddx=8, dup=None, lddup=8, y=None, ldy=8):
        return L.dc_act_backward_device(kind, dtype, rows, cols, dy, lddy, kept, kept_up, dx, lddx, dup, lddup, y, ldy, None)

    for k in (dict(kind=3), dict(kind=-1), dict(dtype=3), dict(rows=-1), dict(cols=-1), dict(rows=1 << 33, cols=8), dict(x=None),
              dict(y=None), dict(kept=None), dict(kept=P + 8), dict(up=P), dict(up=P, kept_up=P + 4), dict(ldx=7), dict(ldy=7),
              dict(up=P, kept_up=P, ldup=1), dict(x=P + 1), dict(kind=0), dict(kind=0, up=P, kept_up=P, y=None)):
        assert forward(**k) == ARG, k
    for k in (dict(kind=3), dict(dtype=9), dict(dy=None), dict(dx=None), dict(kept=None), dict(kept=P + 1), dict(dup=P), dict(kept_up=P),
              dict(lddx=7), dict(dx=P + 1), dict(kind=0), dict(kind=0, dy=None, y=P), dict(kind=0, dy=None, dup=P, kept_up=P),
              dict(rows=1 << 32, cols=1 << 4)):
        assert backward(**k) == ARG, k
    assert forward(rows=0) == 0 and backward(cols=0) == 0


def test_device(lib):
    import torch as t
    assert lib.L.dc_get_device() == -1 or t.cuda.is_available()


def test_status_needs_a_place(lib):
    assert lib.L.dc_kv_status(None, None, 0) == ARG


def test_tensor_calls(d):
    """The torch entry points check shapes, types and devices first."""
    page = d.KVCache.page_bytes(16, 2, 64, 4)
    for bad in ((15, 2, 64, 4), (16, 2, 60, 4), (16, 2, 64, 2)):
        with pytest.raises(ValueError):
            d.KVCache.page_bytes(*bad)
    for buf in (torch.zeros(page - 1, dtype=torch.uint8), torch.zeros(page, dtype=torch.int8), torch.zeros(2 * page, dtype=torch.uint8)[::2]):
        with pytest.raises(ValueError):
            d.KVCache(1, 16, 2, 64, buffer=buf)
    with pytest.raises(ValueError):
        d.KVCache(0, 16, 2, 64, buffer=torch.zeros(page, dtype=torch.uint8))
    room = torch.zeros(2 * page + 16, dtype=torch.uint8)
    room = room[-room.data_ptr() % 16:][:2 * page]
    c = d.KVCache(2, 16, 2, 64, buffer=room)
    k = torch.zeros(2, 3, 2, 64)
    s = torch.zeros(2, dtype=torch.int32)
    t = torch.zeros(2, 1, dtype=torch.int32)
    q = torch.zeros(2, 3, 4, 64, dtype=torch.float16)
    for args, kw in (((k, k[:, :2], s), {}), ((k, k.half(), s), {}), ((k.double(), k.double(), s), {}), ((k[..., :32], k[..., :32], s), {}),
                     ((k[:, :, :1], k[:, :, :1], s), {}), ((k[0], k[0], s), {}), ((k, k, s.long()), {}), ((k, k, s[:1]), {}),
                     ((k, k, s), dict(lens=s.float())), ((k, k, s), dict(table=t.long())), ((k, k, s), dict(table=t[:1])),
                     ((k, k, s), dict(table=t[0])), ((torch.zeros(3, 1, 2, 64),) * 2 + (torch.zeros(3, dtype=torch.int32),), {}),
                     ((k.transpose(1, 3).contiguous().transpose(1, 3), k, s), {}), ((k, k, s), {})):      # (the last: not on the GPU)
        with pytest.raises(ValueError):
            c.write(*args, **kw)
    flat = torch.zeros(2, 3, 1, 64).expand(2, 3, 2, 64)
    for kw in (dict(out=(k, k[:, :2])), dict(out=(k, k.half())), dict(out=(k, flat)), dict(out=(k, k), dtype=torch.float16), dict(dtype=torch.int8)):
        with pytest.raises(ValueError):
            c.read(s, 3, **kw)
    for args, kw in (((q[:, :, :3], s), {}), ((q.float(), s), {}), ((q, s), dict(out=q[:1])), ((q, s), dict(out=q.bfloat16())),
                     ((q, s), dict(out=flat.half().repeat(1, 1, 2, 1)[:, :1].expand(2, 3, 4, 64))),
                     ((q, s), dict(lse=torch.zeros(2, 3, 3))), ((q, s), dict(lse=torch.zeros(2, 3, 4).half())), ((q, s), dict(max_context=-1)),
                     ((q, s), {})):
        with pytest.raises(ValueError):
            c.attention(*args, **kw)
    x = torch.zeros(4, 8)
    for f in (lambda: d.act_forward(x, "relu"), lambda: d.act_forward(x, "silu", up=x[:2]), lambda: d.act_forward(x, "silu", up=x.half()),
              lambda: d.act_forward(x.double(), "silu"), lambda: d.act_forward(x, "silu"), lambda: d.act_save(x), lambda: d.act_save(x.int()),
              lambda: d.ActCheckpoint((4, 8), torch.float32, torch.zeros(32, dtype=torch.uint8)),
              lambda: d.ActCheckpoint((4, 8), torch.float64, torch.zeros(33, dtype=torch.uint8)),
              lambda: d.act_backward(x[:2], d.ActCheckpoint((4, 8), torch.float32, torch.zeros(33, dtype=torch.uint8)), "silu"),
              lambda: d.act_backward(x, d.ActCheckpoint((4, 8), torch.float32, torch.zeros(33, dtype=torch.uint8)), "silu")):
        with pytest.raises(ValueError):
            f()


def test_tensors_exchanged(d):
    """What a cache or a checkpoint was made with is looked at again by each call; wrong kinds of arguments are errors."""
    page = d.KVCache.page_bytes(16, 2, 64, 4)
    room = torch.zeros(3 * page + 16, dtype=torch.uint8)
    room = room[-room.data_ptr() % 16:][:3 * page]
    k, q = torch.zeros(1, 3, 2, 64), torch.zeros(1, 3, 4, 64, dtype=torch.float16)
    s = torch.zeros(1, dtype=torch.int32)
    c = d.KVCache(1, 16, 2, 64, buffer=room[:page])
    c.buffer = room[2 * page:]
    for f in (lambda: c.write(k, k, s), lambda: c.read(s, 3), lambda: c.attention(q, s)):
        with pytest.raises(ValueError, match="buffer"):
            f()
    a = d.ActCheckpoint((4, 8), torch.float32, torch.zeros(33, dtype=torch.uint8))
    a.shape = torch.Size((4, 16))
    for f in (lambda: a.load(), lambda: d.act_backward(torch.zeros(4, 16), a, "silu")):
        with pytest.raises(ValueError, match="66"):
            f()
    c = d.KVCache(1, 16, 2, 64, buffer=room[:page])
    for f in (lambda: c.write(1, k, s), lambda: c.write(k, None, s), lambda: c.read(s, 2.5), lambda: c.read(s, 3, table=[[0]]),
              lambda: c.attention(q, s, max_context="all"), lambda: d.act_forward([1.0], "silu")):
        with pytest.raises((TypeError, AttributeError)):
            f()
    for f in (lambda: c.read(s, -1), lambda: c.read(s, 1 << 31), lambda: c.read(s, 3, out=(k,)), lambda: c.attention(q[0], s),
              lambda: c.write(k, k, torch.zeros((), dtype=torch.int32))):
        with pytest.raises(ValueError):
            f()
