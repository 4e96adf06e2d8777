"""Memory that a call of the torch entry points must not be given: refused before anything is launched, so without a GPU."""
import pytest

torch = pytest.importorskip("torch")


@pytest.fixture(scope="module")
def d():
    import dcamd
    return dcamd


def cache_in(d, room, pages, **k):
    room = room[-room.data_ptr() % 16:]
    return d.KVCache(pages, 16, 2, 64, buffer=room[:pages * d.KVCache.page_bytes(16, 2, 64, 4)], **k)


def test_buffer_cut_short(d):
    """A buffer at the cache's place that has fewer bytes, or not consecutive ones."""
    page = d.KVCache.page_bytes(16, 2, 64, 4)
    c = cache_in(d, torch.zeros(3 * page + 16, dtype=torch.uint8), 3)
    k, q, s = torch.zeros(1, 3, 2, 64), torch.zeros(1, 3, 4, 64, dtype=torch.float16), torch.zeros(1, dtype=torch.int32)
    whole, t = c.buffer, torch.zeros(1, 1, dtype=torch.int32)
    for b in (whole[:page], whole[:3 * page - 1], whole.view(page, 3).t()[:, :page]):
        c.buffer = b
        for f in (lambda: c.write(k, k, s, table=t), lambda: c.read(s, 3, table=t), lambda: c.attention(q, s, table=t)):
            with pytest.raises(ValueError, match="buffer"):
                f()
    c.buffer = whole
    with pytest.raises(ValueError, match="GPU"):
        c.write(k, k, s, table=t)


def test_outputs_on_one_another(d):
    """Outputs whose rows, or whose keys and values, share memory; layouts that do not are taken (and refused as not on the
    GPU only)."""
    page = d.KVCache.page_bytes(16, 2, 64, 4)
    c = cache_in(d, torch.zeros(2 * page + 16, dtype=torch.uint8), 2)
    s = torch.zeros(2, dtype=torch.int32)
    room = torch.zeros(1 << 16)
    q = torch.zeros(2, 3, 4, 64, dtype=torch.float16)
    at = lambda strides, first=0: room.as_strided((2, 3, 2, 64), strides, first)  # noqa: E731
    other = torch.zeros(2, 3, 2, 64)
    bad = [(384, 128, 0, 1), (384, 0, 64, 1), (0, 128, 64, 1), (384, 128, 63, 1), (384, 64, 64, 1), (383, 128, 64, 1), (64, 192, 64, 1), (1, 512, 64, 1)]
    for strides in bad:
        for out in ((at(strides), other), (other, at(strides))):
            with pytest.raises(ValueError, match="lie on one another"):
                c.read(s, 3, out=out)
        with pytest.raises(ValueError, match="lie on one another"):
            c.attention(q, s, out=room.half().as_strided((2, 3, 4, 64), (strides[0] * 2 if strides[0] > 64 else strides[0],) + strides[1:]))
    dense, heads_first, wide, mixed = (384, 128, 64, 1), (384, 64, 192, 1), (1200, 400, 200, 1), (768, 256, 128, 1)
    for strides, off in ((dense, 0), (dense, 1), (dense, 64), (dense, 767), (dense, -65 + 65 * 2), (heads_first, 0), (heads_first, 192), (wide, 0), (wide, 63),
                         (wide, 400 + 30), (wide, 200 - 30), (wide, 1200 - 170), (mixed, 128), (mixed, 3 * 256)):
        for a, b in ((0, off), (off, 0)):
            with pytest.raises(ValueError, match="keys and values must not"):
                c.read(s, 3, out=(at(strides, a), at(strides, b)))
    for strides, off in ((dense, 768), (dense, 10000), (heads_first, 768), (wide, 64), (wide, 100), (wide, 136), (mixed, 64), (mixed, 64 + 1024 + 512)):
        for a, b in ((0, off), (off, 0)):
            with pytest.raises(ValueError, match="GPU"):
                c.read(s, 3, out=(at(strides, a), at(strides, b)))
    one = torch.zeros(1, 3, 2, 64)[:, :1].expand(1, 1, 2, 64)           # (strides of dimensions of one do not count)
    with pytest.raises(ValueError, match="GPU"):
        c.read(s[:1], 1, out=(one, torch.zeros(1, 1, 2, 64)))


def test_what_is_on_one_another_by_trying(d):
    """The rule for keys and values against a plain count of shared places."""
    import random
    rng = random.Random(5)
    page = d.KVCache.page_bytes(16, 2, 64, 4)
    c = cache_in(d, torch.zeros(2 * page + 16, dtype=torch.uint8), 2)
    s = torch.zeros(2, dtype=torch.int32)
    room = torch.zeros(1 << 14)
    ids = torch.arange(1 << 14)
    for _ in range(400):
        dims = [(2, 2), (0, 2), (1, 3)]                                # (dimension, size), from the innermost on
        rng.shuffle(dims)
        strides, reach = [0, 0, 0, 1], 64
        for i, n in dims:
            strides[i] = reach + rng.choice([0, 0, 1, 40, 64, 200])
            reach = strides[i] * (n - 1) + reach
        off = rng.randrange(0, reach + 10) if rng.random() < 0.7 else rng.choice([64, 128, strides[0], strides[1], strides[2]])
        a, b = (ids.as_strided((2, 3, 2, 64), strides, o).flatten() for o in (0, off))
        both = torch.isin(a, b).any()
        with pytest.raises(ValueError, match="keys and values must not" if both else "GPU"):
            c.read(s, 3, out=(room.as_strided((2, 3, 2, 64), strides, 0), room.as_strided((2, 3, 2, 64), strides, off)))


def test_negative_views(d):
    """The imaginary part of a conjugate shares memory that holds the other sign."""
    x = torch.zeros(4, 8, dtype=torch.complex64).conj().imag
    assert x.is_neg()
    page = d.KVCache.page_bytes(16, 2, 64, 4)
    c = cache_in(d, torch.zeros(2 * page + 16, dtype=torch.uint8), 2)
    k, s = torch.zeros(2, 3, 2, 64, dtype=torch.complex64).conj().imag, torch.zeros(2, dtype=torch.int32)
    kept = d.ActCheckpoint((4, 8), torch.float32, torch.zeros(33, dtype=torch.uint8))
    for f in (lambda: d.act_forward(x, "silu"), lambda: d.act_forward(x.resolve_neg(), "silu", up=x), lambda: d.act_save(x), lambda: d.act_backward(x, kept, "silu"),
              lambda: c.write(k, k.resolve_neg(), s), lambda: c.write(k.resolve_neg(), k, s), lambda: c.read(s, 3, out=(k, k.resolve_neg()))):
        with pytest.raises(ValueError, match="negative view"):
            f()
