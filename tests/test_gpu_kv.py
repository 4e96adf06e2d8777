"""The key/value cache in 4 and 8 bits (dcamd.KVCache) against a plain implementation in 64 bits.

What a row holds is defined exactly (include/dc_gpu.h), so reading it back is compared bit by bit.  The attention is
compared with the formula on the values held, within a bound for its arithmetic (`allowed`)."""
import math

import pytest

torch = pytest.importorskip("torch")
pytestmark = pytest.mark.gpu
DEV = "cuda"
F64 = torch.float64


@pytest.fixture(scope="module")
def kv(dc):
    import dcamd
    if dcamd._lib is None:
        dcamd._lib = dc
    return dcamd


# ---- plain implementation (CPU, 64 bits) -----------------------------------------------------------------------------
def bf16_up(v):
    """The smallest bfloat16 that is not below v > 0, element by element."""
    m, e = torch.frexp(v)
    return torch.ldexp(torch.ceil(m * 256), e - 8)


def held(x, bits):
    """What the cache holds of rows x (any float type, CPU): values, steps, zero points, codes in doubles."""
    n = (1 << bits) - 1
    x32 = x.float()
    bad = ~torch.isfinite(x32).all(-1, keepdim=True)
    x32 = torch.where(bad, 0.0, x32)
    lo, hi = x32.amin(-1, keepdim=True), x32.amax(-1, keepdim=True)
    span = 2 * (0.5 * hi - 0.5 * lo).double()
    step = torch.maximum(bf16_up(span / n), bf16_up(torch.maximum(hi, -lo).double() / 32512)).clamp_min(2.0 ** -100)
    zero = torch.round(lo.double() / step)
    code = (torch.round(x32.double() / step) - zero).clamp(0, n)
    values = torch.where(bad, math.nan, step * (zero + code))
    return values, torch.where(bad, math.nan, step), zero, code


def rounded(x, dt):
    m = torch.finfo(dt).max
    return x.clamp(-m, m).to(dt)


def same(a, b):
    """Equal bits (any NaN equals any NaN)."""
    a, b = a.cpu(), b.cpu()
    return a.dtype == b.dtype and a.shape == b.shape and bool(((a == b) | ((a != a) & (b != b))).all())


def rows(g, shape, kind="plain"):
    x = torch.randn(shape, generator=g)
    if kind == "offset":
        x = x * 0.01 + 3.0
    elif kind == "outlier":
        x[..., 0] *= 50.0
    elif kind == "wide":
        x = x * torch.exp(8 * torch.randn(shape[:-1], generator=g))[..., None]
    return x


def gen(seed):
    return torch.Generator().manual_seed(seed)


def i32(*v):
    return torch.tensor(v, dtype=torch.int32, device=DEV)


def make(kv, pages, page, heads, dim, bits, fill=0):
    c = kv.KVCache(pages, page, heads, dim, bits=bits)
    c.buffer.fill_(fill)
    return c


# ---- write and read ------------------------------------------------------------------------------------------------------
@pytest.mark.parametrize("bits", [4, 8])
@pytest.mark.parametrize("dim", [32, 64, 96, 128, 160, 192, 224, 256])
@pytest.mark.parametrize("dtype", [torch.float32, torch.float16, torch.bfloat16])
def test_roundtrip(kv, bits, dim, dtype):
    g = gen(dim + bits)
    B, T, H, P = 2, 37, 3, 16
    c = make(kv, 8, P, H, dim, bits, fill=255)
    table = torch.tensor([[5, 0, 7], [2, 6, 1]], dtype=torch.int32, device=DEV)
    k, v = rows(g, (B, T, H, dim), "offset").to(dtype), rows(g, (B, T, H, dim), "outlier").to(dtype)
    start = i32(0, 11)
    c.write(k.to(DEV), v.to(DEV), start, table=table)
    for out in (torch.float32, dtype):
        gk, gv = c.read(start, T, table=table, dtype=out)
        assert same(gk, rounded(held(k, bits)[0].float(), out))
        assert same(gv, rounded(held(v, bits)[0].float(), out))
    assert kv.KVCache.status(reset=True) == 0


@pytest.mark.parametrize("bits", [4, 8])
def test_half_a_step(kv, bits):
    """|x - x^| <= step / 2, to the f32 rounding of the row's span (2^-24 of it, at most 2^-23 * n / 2 steps)."""
    g = gen(3)
    x = rows(g, (1, 512, 4, 64), "wide")
    c = make(kv, 1, 512, 4, 64, bits)
    c.write(x.to(DEV), x.to(DEV), i32(0))
    got = c.read(i32(0), 512, dtype=torch.float32)[0].cpu().double()
    step = held(x, bits)[1]
    assert bool(((got - x.double()).abs() <= step * (0.5 + 2.0 ** bits * 2.0 ** -23)).all())


@pytest.mark.parametrize("bits", [4, 8])
def test_special_rows(kv, bits):
    """Rows of one value, zeros, the smallest and largest numbers, ties; rows that are not finite read as NaN and leave
    their neighbours alone."""
    D = 32
    x = torch.zeros(24, D)
    x[1] = 1.0
    x[2] = -3.7e-5
    x[3, 5] = 2.0 ** -149
    x[4, 5] = 2.0 ** -99
    x[5] = torch.linspace(-1, 1, D) * 3.4e38
    x[6] = 3.4028234663852886e38
    x[7] = torch.arange(D) % 16 * 1.0
    x[8] = torch.arange(D) * 0.5                                   # ties
    x[9] = -torch.arange(D) * 0.5
    x[10] = 65504.0 - torch.arange(D)
    x[11] = torch.linspace(100, 101, D)
    x[12, 3] = math.nan
    x[13, 31] = math.inf
    x[14, 0] = -math.inf
    x[15] = math.nan
    x[16, 0], x[16, 1] = 1e30, -1e-30
    x[17] = 2.0 ** -126
    x[18] = torch.arange(D) * 2.0 ** -100
    x[19, 7] = 1.0
    x[20] = 1000.0 + torch.arange(D) * 2.0 ** -13                  # the zero point's limit
    x = x.view(1, 24, 1, D)
    c = make(kv, 1, 32, 1, D, bits)
    c.write(x.to(DEV), (-x).to(DEV), i32(0))
    k, v = c.read(i32(0), 24, dtype=torch.float32)
    assert same(k, rounded(held(x, bits)[0], torch.float32))
    assert same(v, rounded(held(-x, bits)[0], torch.float32))
    k, v = c.read(i32(0), 24, dtype=torch.float16)                 # held at the type's largest
    assert same(k, rounded(held(x, bits)[0].float(), torch.float16))
    assert bool(torch.isfinite(k[0, 10]).all())


def test_every_tie(kv):
    """Quotients that lie at, just above and just below a half: the exact quotient decides."""
    g = gen(9)
    D = 64
    step = torch.tensor([1.0, 1.0078125, 1.9921875, 0.33203125, 1e-3]).bfloat16().float()
    x = []
    for s in step:
        for zero in (0, -7, 12, -3000, 20000):
            h = (zero + torch.randint(0, 15, (D,), generator=g) + 0.5).float() * s
            h[0], h[1] = zero * s, (zero + 15) * s
            for nudge in (0, 1, -1):
                y = h.clone()
                y[2:] = (y[2:].view(torch.int32) + nudge).view(torch.float32)
                x.append(y)
    x = torch.stack(x).view(1, -1, 1, D)
    n = x.shape[1]
    for bits in (4, 8):
        c = make(kv, 1, 128, 1, D, bits)
        c.write(x.to(DEV), x.to(DEV), i32(0))
        assert same(c.read(i32(0), n, dtype=torch.float32)[0], held(x, bits)[0].float())


@pytest.mark.parametrize("bits", [4, 8])
def test_strides_alignment_and_padding(kv, bits):
    """(batch, heads, tokens, D) views, unaligned bases, padded rows: what is behind lens[b] is neither read nor written."""
    g = gen(21)
    B, T, H, D, P = 3, 19, 2, 96, 48
    for dtype in (torch.float32, torch.bfloat16):
        k = rows(g, (B, T, H, D)).to(dtype)
        v = rows(g, (B, T, H, D)).to(dtype)
        lens, start = i32(0, 19, 7), i32(5, 0, 29)
        c, ref = make(kv, 3, P, H, D, bits, fill=7), make(kv, 3, P, H, D, bits, fill=7)
        for b in range(B):                                       # one by one, contiguous
            n = int(lens[b])
            if n:
                pages = torch.full((1, 1), b, dtype=torch.int32, device=DEV)
                ref.write(k[b:b + 1, :n].to(DEV), v[b:b + 1, :n].to(DEV), start[b:b + 1].clone(), table=pages)
        kk, vv = k.clone(), v.clone()
        for b in range(B):
            kk[b, int(lens[b]):] = math.nan
            vv[b, int(lens[b]):] = math.nan
        big = torch.empty(B * H * T * D + 1, dtype=dtype, device=DEV)
        view = big[1:].view(B, H, T, D).transpose(1, 2)           # off its alignment
        view.copy_(kk)
        c.write(view, vv.transpose(1, 2).contiguous().to(DEV).transpose(1, 2), start, lens=lens)
        assert same(c.buffer, ref.buffer)
        big.fill_(-5.0)
        out = torch.full((B, T, H, D + 8), -5.0, dtype=dtype, device=DEV)[..., 1:D + 1]
        c.read(start, T, lens=lens, out=(view, out))
        for b in range(B):
            n = int(lens[b])
            for got, x in ((view, k), (out, v)):
                assert same(got[b, :n], rounded(held(x[b, :n], bits)[0].float(), dtype))
                assert bool((got[b, n:] == -5.0).all())
    gk, _ = c.read(start, T, lens=lens, dtype=torch.float32)
    assert bool((gk[0] == 0).all())


def test_outside_the_cache(kv):
    """Positions and pages that are not in the cache: dropped, read as NaN, reported."""
    D, P = 64, 16
    c = make(kv, 4, P, 1, D, 4, fill=3)
    before = c.buffer.clone()
    table = torch.tensor([[4, -1], [2 ** 30, 1]], dtype=torch.int32, device=DEV)
    x = torch.randn(2, 3, 1, D, device=DEV)
    c.write(x, x, i32(2, 2), table=table)                        # bad pages
    c.write(x, x, i32(-3, 32), table=table)                      # bad positions
    c.write(x, x, i32(2 ** 31 - 1, -2 ** 31), table=table)
    assert same(c.buffer, before)
    assert kv.KVCache.status() == 1 and kv.KVCache.status(reset=True) == 1 and kv.KVCache.status() == 0
    c.write(x, x, i32(-2, 31), table=torch.tensor([[0, 1], [2, 3]], dtype=torch.int32, device=DEV))   # one of three each
    k, _ = c.read(i32(-2, 31), 3, table=torch.tensor([[0, 1], [2, 3]], dtype=torch.int32, device=DEV), dtype=torch.float32)
    want = held(x.cpu(), 4)[0].float()
    assert bool(torch.isnan(k[0, :2]).all()) and bool(torch.isnan(k[1, 1:]).all())
    assert same(k[0, 2], want[0, 2]) and same(k[1, 0], want[1, 0])
    assert kv.KVCache.status(reset=True) == 1


def test_nothing_to_do(kv):
    c = make(kv, 2, 16, 1, 32, 4)
    e = torch.empty(0, 3, 1, 32, device=DEV)
    none = torch.empty(0, dtype=torch.int32, device=DEV)
    c.write(e, e, none)
    assert c.read(none, 3)[0].shape == (0, 3, 1, 32)
    e = torch.empty(2, 0, 1, 32, device=DEV)
    c.write(e, e, i32(0, 0))
    assert c.read(i32(0, 0), 0)[0].shape == (2, 0, 1, 32)
    q = torch.empty(2, 0, 1, 32, device=DEV, dtype=torch.float16)
    assert c.attention(q, i32(0, 0)).shape == q.shape


# ---- attention ----------------------------------------------------------------------------------------------------------
class Filled:
    """A cache of B sequences with `context` positions each in shuffled pages, and what it holds in doubles (CPU)."""

    def __init__(self, kv, seed, B, context, H, D, P, bits, spare=0, kind=("outlier", "plain"), dtype=torch.bfloat16):
        g = gen(seed)
        self.width = -(-context // P) + spare
        pages = B * self.width + 1
        perm = torch.randperm(pages, generator=g)[:B * self.width].to(torch.int32)
        self.table = perm.view(B, self.width).to(DEV)
        self.cache = make(kv, pages, P, H, D, bits, fill=255)     # 0xFF: NaN steps wherever nothing was written
        k, v = (rows(g, (B, context, H, D), kd).to(dtype) for kd in kind)
        self.cache.write(k.to(DEV), v.to(DEV), torch.zeros(B, dtype=torch.int32, device=DEV), table=self.table)
        self.k, self.ks, self.kz, self.kc = held(k, bits)
        self.v, self.vs, self.vz, self.vc = held(v, bits)


def formula(f, q, context, lens, scale, causal):
    """(output, log of the sum, how far the kernel's output may be off) in doubles.

    With u = 2^-24: a score is a sum of D products of codes with queries (at most D + 8 roundings, each u of the
    sum of magnitudes A = ks (sum |q| code + |kz| sum |q|)), so a weight is off by (D + 8) u scale A of itself, and by
    2^-11 (to f16) + 8 u (its factors); weights below f16's normal range by 2^-25 of units of which the largest step is
    64 or more.  The sum
    over positions adds N u of magnitudes; the output's type half a unit.  A matrix instruction cuts each of its 33 terms
    at 24 bits below the largest one's exponent, in which a code counts as 2^-14: at 2^-18 (codes are n 2^-20: 4 bits) or
    2^-14 (n 2^-24: 8 bits) of a code times the largest query element or weight; D / 32 of them make a score, a 32nd of N
    and one for each wave and each split of the work the sums."""
    B, T, HQ, D = q.shape
    H, N = f.k.shape[2], f.k.shape[1]
    G = HQ // H
    u = 2.0 ** -24
    half = torch.finfo(q.dtype).eps / 2
    out, lse, tol = (torch.zeros(B, T, HQ, n, dtype=F64) for n in (D, 1, D))
    lse.fill_(-math.inf)
    for b in range(B):
        for i in range(int(lens[b])):
            n = int(context[b]) - int(lens[b]) + 1 + i if causal else int(context[b])
            if n <= 0:
                continue
            for h in range(H):
                qq = q[b, i, h * G:(h + 1) * G].double()                                # (G, D)
                k, v = f.k[b, :n, h], f.v[b, :n, h]                                     # (n, D)
                s = qq @ k.t() * scale
                A = (qq.abs() @ f.kc[b, :n, h].t() + qq.abs().sum(-1, keepdim=True) * f.kz[b, :n, h].abs().t()) * \
                    f.ks[b, :n, h].t() * abs(scale)
                p = torch.softmax(s, -1)
                o = p @ v
                cut = 33 * (2.0 ** -18 if f.kc.max() < 16 else 2.0 ** -14)
                A = A + cut / u / (D + 8) * (D / 32) * qq.abs().amax(-1, keepdim=True) * f.ks[b, :n, h].t() * abs(scale)
                mag = f.vs[b, :n, h] * (f.vc[b, :n, h] + f.vz[b, :n, h].abs())
                eps = torch.expm1((D + 8) * u * A) + 8 * u
                w = p * f.vs[b, :n, h].t()
                largest = w.amax(-1, keepdim=True)
                err = (p * (eps + 2.0 ** -11)) @ v.abs() + (p * eps).sum(-1, keepdim=True) * o.abs()
                tiny = 2.0 ** -31 * f.vs[b, :n, h].max()
                err = err + ((n + 8) * u * w + tiny) @ (mag / f.vs[b, :n, h])
                err = err + cut * (n / 32 + 4 * (1 + n / 256)) * largest
                out[b, i, h * G:(h + 1) * G] = o
                lse[b, i, h * G:(h + 1) * G, 0] = torch.logsumexp(s, -1)
                tol[b, i, h * G:(h + 1) * G] = err * 1.01 + half * (o.abs() + err) + 2.0 ** -25
    return out, lse[..., 0], tol


def check(f, q, context, lens=None, scale=None, causal=True, max_context=None, **more):
    D = q.shape[-1]
    got_lse = torch.full(q.shape[:3], 7.0, device=DEV)
    got = f.cache.attention(q.to(DEV), i32(*context), table=f.table, lens=None if lens is None else i32(*lens), scale=scale,
                            causal=causal, max_context=max_context, lse=got_lse, **more)
    lens = lens or [q.shape[1]] * q.shape[0]
    want, lse, tol = formula(f, q, context, lens, D ** -0.5 if scale is None else scale, causal)
    for b, n in enumerate(lens):
        off = (got[b, :n].cpu().double() - want[b, :n]).abs()
        assert bool((off <= tol[b, :n]).all()), (b, float((off / tol[b, :n]).max()))
        d = got_lse[b, :n].cpu().double()
        assert bool(((d == lse[b, :n]) | ((d - lse[b, :n]).abs() <= 1e-4 * (1 + lse[b, :n].abs()))).all())
        assert bool((got_lse[b, n:] == 7.0).all())
    return got


@pytest.mark.parametrize("bits", [4, 8])
@pytest.mark.parametrize("dim", [32, 64, 96, 128, 160, 192, 224, 256])
@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
def test_attention_dims(kv, bits, dim, dtype):
    f = Filled(kv, dim, 2, 300, 2, dim, 48, bits)
    q = torch.randn(2, 1, 6, dim, generator=gen(1)).to(dtype)
    check(f, q, [300, 171])
    q = torch.randn(2, 21, 4, dim, generator=gen(2)).to(dtype)            # several tiles of query rows
    check(f, q, [300, 171], lens=[21, 20])


@pytest.mark.parametrize("context", [1, 2, 15, 16, 17, 31, 32, 33, 63, 127, 128, 129, 255, 257, 511, 1000])
def test_attention_lengths(kv, context):
    f = Filled(kv, context, 2, context, 1, 64, 16, 4, spare=2)
    q = torch.randn(2, 1, 5, 64, generator=gen(4)).half()
    check(f, q, [context, max(0, context - 1)])
    check(f, q, [context, context // 2], max_context=context)
    check(f, q, [context, 0], max_context=1)                              # longer than expected: in full all the same


@pytest.mark.parametrize("group", [1, 2, 3, 7, 8, 16, 17, 40])
def test_attention_groups(kv, group):
    f = Filled(kv, group, 1, 200, 2, 128, 64, 4)
    q = torch.randn(1, 1, 2 * group, 128, generator=gen(group)).bfloat16()
    check(f, q, [197])


@pytest.mark.parametrize("bits", [4, 8])
@pytest.mark.parametrize("tokens,causal", [(2, True), (3, False), (16, True), (17, True), (70, True), (130, False)])
def test_attention_chunks(kv, bits, tokens, causal):
    """Chunks of a prompt, some longer than their sequence: queries that see nothing give 0."""
    f = Filled(kv, tokens, 3, 210, 2, 64, 32, bits)
    q = torch.randn(3, tokens, 6, 64, generator=gen(tokens)).bfloat16()
    got = check(f, q, [210, tokens // 2, tokens], lens=[tokens, tokens, (tokens + 1) // 2], causal=causal)
    if causal:
        blind = tokens - tokens // 2 - 1
        assert blind <= 0 or bool((got[1, :blind] == 0).all())


@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
def test_attention_split(kv, dtype):
    """A long cache and few heads: the work is split along it."""
    f = Filled(kv, 5, 1, 9001, 1, 128, 64, 4)
    q = torch.randn(1, 1, 4, 128, generator=gen(6)).to(dtype)
    for n in (9001, 8999, 257, 1, 0):
        check(f, q, [n])
    q = torch.randn(1, 5, 4, 128, generator=gen(7)).to(dtype)
    check(f, q, [9000], lens=[4])


@pytest.mark.parametrize("bits", [4, 8])
@pytest.mark.parametrize("dim", [32, 96, 128, 160, 224, 256])
def test_attention_split_ragged(kv, bits, dim):
    """One long sequence among short and empty ones: pieces by the whole batch's length, joined; some have one piece."""
    f = Filled(kv, 7 + dim, 4, 3000, 2, dim, 16, bits)
    q = torch.randn(4, 1, 6, dim, generator=gen(dim)).half()
    check(f, q, [3000, 3, 0, 700])
    check(f, q, [1, 2999, 2500, 2400])
    q = torch.randn(4, 7, 6, dim, generator=gen(dim)).bfloat16()          # several tiles of rows, padded
    got = check(f, q, [3000, 3, 1200, 900], lens=[7, 7, 0, 2])
    assert bool((got[1, :4] == 0).all()) and bool((got[2] == 0).all())


def test_attention_steps_of_all_sizes(kv):
    """Values whose steps lie far apart: the largest weight times step sets the scale, not the largest weight."""
    f = Filled(kv, 11, 1, 400, 1, 64, 16, 4, kind=("plain", "wide"), dtype=torch.float32)
    q = 6 * torch.randn(1, 1, 8, 64, generator=gen(12)).half()
    f2 = Filled(kv, 13, 1, 64, 1, 64, 16, 8, kind=("outlier", "wide"), dtype=torch.float32)
    for x in (f, f2):
        n = x.k.shape[1]
        big = float(x.v.abs().max())
        if big < 6e4:
            check(x, q, [n])
        check(x, q.bfloat16(), [n])


def test_attention_rows_of_zeros(kv):
    """The most-attended token has values of zero (a sink)."""
    B, N, D = 1, 100, 64
    g = gen(31)
    k, v = torch.randn(B, N, 1, D, generator=g), torch.randn(B, N, 1, D, generator=g)
    k[:, 0] *= 10
    v[:, 0] = 0
    c = make(kv, 1, 112, 1, D, 4)
    c.write(k.to(DEV), v.to(DEV), i32(0))
    q = k[:, :1].half()
    f = Filled.__new__(Filled)
    f.cache, f.table = c, torch.zeros(1, 1, dtype=torch.int32, device=DEV)
    f.k, f.ks, f.kz, f.kc = held(k, 4)
    f.v, f.vs, f.vz, f.vc = held(v, 4)
    check(f, q, [N])


def test_attention_strides_and_padding(kv):
    """Queries and outputs as views of other layouts; rows behind lens[b] keep what they have."""
    f = Filled(kv, 41, 2, 150, 2, 64, 16, 4)
    q = torch.randn(2, 9, 4, 64, generator=gen(42)).bfloat16()
    plain = check(f, q, [150, 90], lens=[9, 3])
    assert bool((plain[1, 3:] == 0).all())
    store = torch.full((2, 4, 9, 64 + 6), -3.0, dtype=torch.bfloat16, device=DEV)
    out = store[..., 3:67].transpose(1, 2)
    qv = torch.empty(2, 4, 9, 65, dtype=torch.bfloat16, device=DEV)[..., 1:].transpose(1, 2)
    qv.copy_(q)
    qv[1, 3:] = math.nan
    f.cache.attention(qv, i32(150, 90), table=f.table, lens=i32(9, 3), out=out)
    assert same(out[0], plain[0]) and same(out[1, :3], plain[1, :3])
    far = Filled(kv, 43, 1, 3000, 1, 64, 16, 4)                        # split along the cache: padding is set to 0 too
    for tok, n in ((3, 1), (40, 17), (5, 0)):
        qq = torch.randn(1, tok, 2, 64, generator=gen(tok)).half()
        y = far.cache.attention(qq.to(DEV), i32(3000), table=far.table, lens=i32(n))
        assert bool((y[0, n:] == 0).all())
    assert bool((out[1, 3:] == -3).all()) and bool((store[..., :3] == -3).all()) and bool((store[..., 67:] == -3).all())


def test_attention_not_finite(kv):
    """A NaN row reaches only the queries that see it; a NaN query only itself; what lies behind the length nothing."""
    f = Filled(kv, 51, 1, 80, 1, 64, 16, 4)
    q = torch.randn(1, 8, 2, 64, generator=gen(52)).bfloat16()
    clean = check(f, q, [60])
    bad = torch.full((1, 1, 1, 64), math.nan, device=DEV)
    ok = torch.ones(1, 1, 1, 64, device=DEV)
    for k, v in ((bad, ok), (ok, bad)):
        f.cache.write(k, v, i32(57), table=f.table)
        got = f.cache.attention(q.to(DEV), i32(60), table=f.table)
        assert same(got[0, :5], clean[0, :5])                            # these see positions below 57
        assert bool(torch.isnan(got[0, 5:]).all())
    got = f.cache.attention(q.to(DEV), i32(57), table=f.table)
    f.cache.write(ok, ok, i32(57), table=f.table)
    q2 = q.clone()
    q2[0, 3, 1, 7] = math.nan
    a, b = f.cache.attention(q.to(DEV), i32(57), table=f.table), f.cache.attention(q2.to(DEV), i32(57), table=f.table)
    assert same(got, a) and bool(torch.isfinite(a).all())
    assert bool(torch.isnan(b[0, 3, 1]).all())
    b[0, 3, 1] = a[0, 3, 1]
    assert same(a, b)


def test_attention_outside_the_cache(kv):
    """Pages that are not in the cache are left out and reported; lengths outside it are held at its bounds."""
    f = Filled(kv, 61, 1, 96, 1, 64, 32, 4)
    q = torch.randn(1, 1, 2, 64, generator=gen(62)).half()
    table = f.table.clone()
    table[0, 1] = 1 << 30
    got = f.cache.attention(q.to(DEV), i32(96), table=table)
    assert kv.KVCache.status(reset=True) == 1
    keep = list(range(32)) + list(range(64, 96))
    g = Filled.__new__(Filled)
    for n in ("k", "ks", "kz", "kc", "v", "vs", "vz", "vc"):
        setattr(g, n, getattr(f, n)[:, keep])
    want, _, tol = formula(g, q, [64], [1], 0.125, True)
    assert bool(((got.cpu().double() - want).abs() <= tol).all())
    whole = check(f, q, [96])
    assert kv.KVCache.status(reset=True) == 0
    assert same(f.cache.attention(q.to(DEV), i32(2 ** 31 - 1), table=f.table), whole)
    assert same(f.cache.attention(q.to(DEV), i32(-5), table=f.table), torch.zeros_like(whole))
    assert kv.KVCache.status(reset=True) == 1


def test_decode_loop(kv):
    """Prompt, then tokens one by one, across page borders: each step's attention as the formula's, each byte of the cache
    as one write of the whole."""
    B, H, G, D, P, bits, first, n = 2, 2, 4, 64, 16, 4, 29, 24
    g = gen(71)
    k, v = (torch.randn(B, first + n, H, D, generator=g).bfloat16() for _ in range(2))
    width = -(-(first + n) // P)
    table = torch.randperm(B * width, generator=g).to(torch.int32).view(B, width).to(DEV)
    c, whole = make(kv, B * width, P, H, D, bits), make(kv, B * width, P, H, D, bits)
    whole.write(k.to(DEV), v.to(DEV), i32(0, 0), table=table)
    c.write(k[:, :first].to(DEV), v[:, :first].to(DEV), i32(0, 0), table=table)
    f = Filled.__new__(Filled)
    f.cache, f.table = c, table
    f.k, f.ks, f.kz, f.kc = held(k, bits)
    f.v, f.vs, f.vz, f.vc = held(v, bits)
    for t in range(first, first + n):
        c.write(k[:, t:t + 1].to(DEV), v[:, t:t + 1].to(DEV), i32(t, t), table=table)
        check(f, torch.randn(B, 1, H * G, D, generator=g).bfloat16(), [t + 1, t + 1])
    assert same(c.buffer, whole.buffer)


def test_graph_and_streams(kv):
    """A captured step (write, attention, read) replayed with new inputs, with eager work between; two streams at once."""
    f = Filled(kv, 81, 2, 700, 1, 128, 64, 4, spare=1)
    q = torch.randn(2, 1, 8, 128, device=DEV).half()
    k, v = torch.randn(2, 1, 1, 128, device=DEV), torch.randn(2, 1, 1, 128, device=DEV)
    pos, ctx = i32(700, 700), i32(701, 701)

    def step():
        f.cache.write(k, v, pos, table=f.table)
        return f.cache.attention(q, ctx, table=f.table), f.cache.read(pos, 1, table=f.table)[0]

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step()
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = step()
    for i in range(4):
        q.copy_(torch.randn(2, 1, 8, 128, generator=gen(i)))
        k.copy_(torch.randn(2, 1, 1, 128, generator=gen(10 + i)))
        v.copy_(torch.randn(2, 1, 1, 128, generator=gen(20 + i)))
        pos.fill_(700 + i)
        ctx.fill_(701 + i)
        graph.replay()
        torch.cuda.synchronize()
        got = [x.clone() for x in out]
        want = step()
        torch.cuda.synchronize()
        assert same(got[0], want[0]) and same(got[1], want[1])
    base = f.cache.attention(q, ctx, table=f.table)
    streams = [torch.cuda.Stream() for _ in range(2)]
    torch.cuda.synchronize()
    outs = []
    for i in range(6):
        with torch.cuda.stream(streams[i % 2]):
            outs.append(f.cache.attention(q, ctx, table=f.table))
    torch.cuda.synchronize()
    assert all(same(o, base) for o in outs)


def test_repeatable(kv):
    f = Filled(kv, 91, 1, 5000, 2, 128, 64, 4)
    q = torch.randn(1, 1, 16, 128, device=DEV).bfloat16()
    a = f.cache.attention(q, i32(5000), table=f.table)
    assert all(same(f.cache.attention(q, i32(5000), table=f.table), a) for _ in range(5))


def test_large_read(kv):
    """An output that is written past the caches (over 128 MB) as the same in parts."""
    H, D, P, n = 16, 128, 64, 18000
    c = make(kv, -(-n // P), P, H, D, 8)
    table = torch.arange(-(-n // P), dtype=torch.int32, device=DEV).flip(0)[None]
    k, v = (torch.randn(1, n, H, D, device=DEV) for _ in range(2))
    c.write(k, v, i32(0), table=table)
    a = c.read(i32(0), n, table=table, dtype=torch.float32)
    for first in (0, 7000, 14001):
        m = min(7000, n - first)
        b = c.read(i32(first), m, table=table, dtype=torch.float32)
        assert same(a[0][:, first:first + m], b[0]) and same(a[1][:, first:first + m], b[1])
    assert same(a[0][:, :50], held(k[:, :50].cpu(), 8)[0].float())


def test_far_pages(kv):
    """Byte offsets beyond 32 bits: the last pages of a cache over 4 GiB."""
    H, D, P, bits = 8, 256, 1024, 8
    pages = (5 << 30) // kv.KVCache.page_bytes(P, H, D, bits)
    c = kv.KVCache(pages, P, H, D, bits=bits, buffer=torch.empty(pages * kv.KVCache.page_bytes(P, H, D, bits), dtype=torch.uint8, device=DEV))
    table = torch.tensor([[pages - 1]], dtype=torch.int32, device=DEV)
    g = gen(101)
    k, v = (torch.randn(1, 40, H, D, generator=g).bfloat16() for _ in range(2))
    c.write(k.to(DEV), v.to(DEV), i32(900), table=table)
    gk, gv = c.read(i32(900), 40, table=table, dtype=torch.float32)
    assert same(gk, held(k, bits)[0].float()) and same(gv, held(v, bits)[0].float())
    zero = torch.zeros(1, 900, H, D, device=DEV)
    c.write(zero, zero, i32(0), table=table)
    f = Filled.__new__(Filled)
    f.cache, f.table = c, table
    z = torch.zeros(1, 900, H, D)
    f.k, f.ks, f.kz, f.kc = held(torch.cat((z, k.float()), 1), bits)
    f.v, f.vs, f.vz, f.vc = held(torch.cat((z, v.float()), 1), bits)
    check(f, torch.randn(1, 1, H, D, generator=g).bfloat16(), [940])


@pytest.mark.parametrize("scale", [-0.2, 0.0, 1e-30, 3.0])
def test_attention_scales(kv, scale):
    """A scale's sign goes with the queries, and none of what a causal query does not see comes back through a scale of 0."""
    f = Filled(kv, 90, 2, 200, 2, 64, 16, 8)
    check(f, torch.randn(2, 1, 4, 64, generator=gen(91)).half(), [200, 33], scale=scale)
    check(f, torch.randn(2, 19, 4, 64, generator=gen(92)).half(), [150, 19], lens=[19, 7], scale=scale)


@pytest.mark.parametrize("bits,dim", [(4, 128), (8, 64), (4, 64)])
def test_attention_room_for_many(kv, bits, dim):
    """Tables that allow more than the caches hold (where codes are read past them), of sequences of all lengths."""
    f = Filled(kv, 93, 3, 900, 2, dim, 16, bits)
    f.table = torch.cat((f.table, torch.full((3, 40000), -1, dtype=torch.int32, device=DEV)), 1)
    q = torch.randn(3, 1, 8, dim, generator=gen(94)).bfloat16()
    for context in ([900, 1, 0], [900, 900, 900], [129, 640, 641]):
        check(f, q, context)
    check(f, torch.randn(3, 4, 8, dim, generator=gen(95)).bfloat16(), [900, 3, 77], lens=[4, 3, 2])


@pytest.mark.parametrize("k", [-108, -60, 60, 100])
def test_attention_queries_of_all_sizes(kv, k):
    """Queries of 2^k and a scale of 2^-k (bfloat16): as those of 1."""
    f = Filled(kv, 96, 1, 300, 2, 128, 16, 4)
    q = torch.randn(1, 1, 4, 128, generator=gen(97)).bfloat16()
    want = check(f, q, [300], scale=0.125)
    got = f.cache.attention((q.float() * 2.0 ** k).bfloat16().to(DEV), i32(300), table=f.table, scale=0.125 * 2.0 ** -k)
    assert torch.equal(got, want)


@pytest.mark.parametrize("dtype,n", [(torch.float32, 9000), (torch.bfloat16, 17000)])
def test_large_write(kv, dtype, n):
    """An input that is read past the caches (over 128 MB) as the same in parts."""
    H, D, P = 16, 128, 48
    pages = -(-n // P)
    table = torch.randperm(pages, generator=gen(98)).to(torch.int32).to(DEV)[None]
    k, v = (torch.randn(1, n, H, D, device=DEV).to(dtype) for _ in range(2))
    whole, parts = (make(kv, pages, P, H, D, 4) for _ in range(2))
    whole.write(k, v, i32(0), table=table)
    for first in range(0, n, 3001):
        m = min(3001, n - first)
        parts.write(k[:, first:first + m], v[:, first:first + m], i32(first), table=table)
    assert torch.equal(whole.buffer, parts.buffer)
