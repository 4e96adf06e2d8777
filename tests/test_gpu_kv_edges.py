"""Calls of the key/value cache at the edges of what its documentation allows."""
import math

import pytest

torch = pytest.importorskip("torch")
from test_gpu_kv import DEV, Filled, gen, held, i32, kv, make, rounded, same  # noqa: E402,F401
from test_gpu_kv_weights import check, filled  # noqa: E402

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("bits", [4, 8])
@pytest.mark.parametrize("n", [1, 40, 3000])
@pytest.mark.parametrize("size", [-1e25, -1e15, -30.0, 30.0, 1e15, 1e25])
def test_scores_of_all_sizes(kv, bits, n, size):
    """Scores of 1e8 to 1e33 of both signs.  Equal keys have equal scores, so the mean of the values is wanted: f16 weights
    are off by 2^-11 of themselves, the matrix instructions cut 33 terms at 2^-18 or 2^-14 of a code's step times the largest
    weight (n / 32 of them, and one for each wave and piece), sums are f32, the output has 8 bits: half a unit is 2^-8 (torch.finfo(bfloat16).eps / 2) of a value at most.  Then keys of which one has
    the largest score by far: its values, exactly."""
    g = gen(n)
    key = torch.randn(1, 1, 1, 64, generator=g).abs() * 1e7
    v = torch.randn(1, n, 1, 64, generator=g)
    f = filled(kv, key.expand(1, n, 1, 64), v, bits)
    q = ((0.5 + torch.rand(1, 1, 2, 64, generator=g)) * size).bfloat16()
    got = f.cache.attention(q.to(DEV), i32(n), table=f.table).cpu().double()
    x = f.v[0, :, 0]
    want, mag = x.mean(0), x.abs().mean(0)
    cut = 33 * (2.0 ** -18 if bits == 4 else 2.0 ** -14) * (n / 32 + 4 * (1 + n / 256)) * f.vs.max() / n
    err = (2.0 ** -11 + (n + 80) * 2.0 ** -24) * mag + cut
    assert bool(((got - want).abs() <= err + torch.finfo(torch.bfloat16).eps / 2 * (want.abs() + err)).all())
    other = torch.full((n,), 1.0 if size > 0 else 1.5)
    other[n // 3] = 1.5 if size > 0 else 1.0
    f = filled(kv, key * other[None, :, None, None], v, bits)
    assert torch.equal(torch.argmax(f.k[0, :, 0] @ q[0, 0].double().t(), 0), torch.full((2,), n // 3))
    got = f.cache.attention(q.to(DEV), i32(n), table=f.table)
    for h in range(2):
        assert same(got[0, 0, h], f.v[0, n // 3, 0].to(torch.bfloat16))


@pytest.mark.parametrize("n,tokens", [(1, 1), (40, 1), (40, 7), (3000, 1), (3000, 5)])
def test_nothing_in_the_cache(kv, n, tokens):
    """Every page outside the cache: what is left out is not seen, so 0 and -inf; a sequence beside it is as it was."""
    f = Filled(kv, 61, 2, n, 1, 64, 16, 4)
    q = torch.randn(2, tokens, 2, 64, generator=gen(62)).half()
    want = f.cache.attention(q.to(DEV), i32(n, n), table=f.table)
    table = f.table.clone()
    table[0] = torch.where(torch.arange(f.width, device=DEV) % 2 == 0, -1, 1 << 30)
    lse = torch.zeros(2, tokens, 2, device=DEV)
    got = f.cache.attention(q.to(DEV), i32(n, n), table=table, lse=lse)
    assert kv.KVCache.status(reset=True) == 1
    assert bool((got[0] == 0).all()) and bool((lse[0] == -math.inf).all())
    assert same(got[1], want[1]) and bool(torch.isfinite(lse[1]).all())


@pytest.mark.parametrize("bits", [4, 8])
@pytest.mark.parametrize("n,tokens", [(1, 1), (40, 1), (40, 9), (3000, 1), (3000, 3), (5000, 1)])
def test_values_of_all_sizes(kv, bits, n, tokens):
    """Values up to 1e38, of one sign or of both: sums without their division would pass f32's range."""
    g = gen(n)
    k, v = (torch.randn(1, n, 2, 64, generator=g) for _ in range(2))
    v = v / v.abs().max() * 1e38
    v[:, :, 1] = v[:, :, 1].abs()
    q = torch.randn(1, tokens, 4, 64, generator=g).bfloat16()
    check(filled(kv, k, v, bits), q, [n])
    if n == 1:
        v[0, 0, 0, 0], v[0, 0, 0, 1] = 3e38, -3e38                    # (a row that spans more than f32's largest number)
        f = filled(kv, k, v, bits)
        got = f.cache.attention(q.to(DEV), i32(1), table=f.table)
        assert same(got[0, 0, :2], f.v[0, 0, :1].to(torch.bfloat16).expand(2, 64))


def test_one_page_of_all_positions(kv):
    """Pages of 2^30 tokens (43 GB in 4 bits): the values' words lie 2^32 bytes behind the keys'."""
    P, D = 1 << 30, 32
    room = torch.empty(kv.KVCache.page_bytes(P, 1, D, 4), dtype=torch.uint8, device=DEV)
    c = kv.KVCache(1, P, 1, D, bits=4, buffer=room)
    g = gen(3)
    k, v = torch.randn(1, 40, 1, D, generator=g), torch.randn(1, 40, 1, D, generator=g) * 100
    for first in (0, P - 40):
        c.write(k.to(DEV), v.to(DEV), i32(first))
        got = c.read(i32(first), 40, dtype=torch.float32)
        assert same(got[0], held(k, 4)[0].float()) and same(got[1], held(v, 4)[0].float())
    f = Filled.__new__(Filled)
    f.cache, f.table = c, None
    f.k, f.ks, f.kz, f.kc = held(k, 4)
    f.v, f.vs, f.vz, f.vc = held(v, 4)
    for tokens in (1, 40):
        check(f, torch.randn(1, tokens, 2, D, generator=g).half(), [40], max_context=40)


@pytest.mark.parametrize("dim", [32, 64, 96, 160, 224])
@pytest.mark.parametrize("n", [900, 3000, 20000])
@pytest.mark.parametrize("off", [2, 4, 8])
def test_joined_outputs_off_their_alignment(kv, dim, n, off):
    """Pieces joined into heads that start anywhere: as into a new tensor, and nothing beside them is written."""
    f = Filled(kv, dim + n, 1, n, 1, dim, 16, 4)
    q = torch.randn(1, 3, 2, dim, generator=gen(dim)).bfloat16()
    want = check(f, q, [n])
    room = torch.full((1, 3, 2, dim + 8), -3.0, dtype=torch.bfloat16, device=DEV)
    out = room[..., off // 2:off // 2 + dim]
    f.cache.attention(q.to(DEV), i32(n), table=f.table, out=out)
    assert same(out, want)
    out.fill_(-3.0)
    assert bool((room == -3).all())


def test_status_beside_other_streams(kv):
    """A bit that is set while the word is taken is in that answer or in the next."""
    c = make(kv, 1, 16, 1, 32, 4)
    x, side = torch.zeros(1, 1, 1, 32, device=DEV), torch.cuda.Stream()
    outside, pos = torch.full((1, 1), 5, dtype=torch.int32, device=DEV), i32(0)
    torch.cuda.synchronize()
    kv.KVCache.status(reset=True)
    for _ in range(200):
        with torch.cuda.stream(side):
            c.write(x, x, pos, table=outside)
        got = kv.KVCache.status(reset=True)
        side.synchronize()
        assert got | kv.KVCache.status(reset=True) == 1
        assert kv.KVCache.status() == 0


def test_streams_of_all_kinds(kv):
    """HIP's default stream, its stream of the thread, the library's and one of torch's, through the C entry points."""
    import ctypes as C
    L = kv.lib()
    c = make(kv, 1, 16, 2, 32, 4)
    k, v = torch.randn(1, 5, 2, 32, device=DEV), torch.randn(1, 5, 2, 32, device=DEV)
    want = [rounded(held(x.cpu(), 4)[0].float(), torch.float32) for x in (k, v)]
    start, st = i32(0), (C.c_longlong * 3)(320, 64, 32)
    at = kv.KvBatchDesc(1, 5, start.data_ptr(), None, None, 0, 0, 0)
    torch.cuda.synchronize()
    for stream in (None, 2, L.L.dc_get_stream(), torch.cuda.Stream().cuda_stream):      # (2: hipStreamPerThread)
        c.buffer.zero_()
        got = [torch.full((1, 5, 2, 32), -1.0, device=DEV) for _ in range(2)]
        torch.cuda.synchronize()
        L.check(L.L.dc_kv_write_device(c._desc, at, 0, k.data_ptr(), st, v.data_ptr(), st, stream), "write")
        L.check(L.L.dc_kv_read_device(c._desc, at, 0, got[0].data_ptr(), st, got[1].data_ptr(), st, stream), "read")
        word = C.c_uint(7)
        L.check(L.L.dc_kv_status(stream, C.byref(word), 0), "status")                   # (waits for the stream)
        assert word.value == 0 and same(got[0], want[0]) and same(got[1], want[1])


def test_outputs_beyond_the_type(kv):
    """A mean beyond f16's largest number is infinite in f16 and what it is in bf16."""
    g = gen(8)
    k, v = torch.randn(1, 50, 1, 64, generator=g), torch.full((1, 50, 1, 64), 1e6)
    f = filled(kv, k, v, 8)
    q = torch.randn(1, 1, 2, 64, generator=g)
    got = f.cache.attention(q.half().to(DEV), i32(50), table=f.table)
    assert bool((got == math.inf).all())
    check(f, q.bfloat16(), [50])


@pytest.mark.parametrize("bits", [4, 8])
@pytest.mark.parametrize("k", [25, 26, 27, 28, 29, 30, 34])
def test_scores_that_creep(kv, bits, k):
    """Scores of about 2^k that rise by a few units of f32 from step to step of a wave (128
    positions).  Which of the last ones share the weight is f32's rounding: the output is within what the last three steps'
    positions hold, each row being one value."""
    N, D, n = 1400, 64, 15 if bits == 4 else 255
    key = torch.zeros(1, N, 1, D)
    key[..., 0] = n                                                     # a step of 1, so the other value counts single codes
    key[0, :, 0, 40] = (torch.arange(N) // 128).float()               # (added by a later instruction: to f32's last bit)
    v = torch.arange(N)[None, :, None, None].float().expand(1, N, 1, D)
    f = filled(kv, key, v, bits)
    assert bool((f.ks == 1).all()) and bool((f.kz == 0).all())
    held_rows = f.v[0, 1024:, 0, 0]
    for rise in (2.0 ** -24, 1.5 * 2.0 ** -24, 2.0 ** -23, 1.5 * 2.0 ** -23, 2.0 ** -22, 2.0 ** -16):     # of a score, from code to code
        q = torch.zeros(1, 1, 2, D)
        q[..., 0], q[..., 40] = 1.0, rise * (n + 1)
        for scale in (2.0 ** k / n, 2.0 ** k / n * 1.2, 2.0 ** k / n * 1.3):
            got = f.cache.attention(q.bfloat16().to(DEV), i32(N), table=f.table, scale=scale).cpu().double()
            assert bool(torch.isfinite(got).all()), (rise, scale, got[0, 0, 0, 0])
            assert bool((got >= held_rows.min() * (1 - 2.0 ** -7)).all()) and bool((got <= held_rows.max() * (1 + 2.0 ** -7)).all()), (rise, scale, got[0, 0, 0, 0])
