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
