"""The attention's weights where the rows of values have steps of very different sizes: what a query does not see, or sees
with no weight, leaves its output as it is."""
import math

import pytest

torch = pytest.importorskip("torch")
from test_gpu_kv import DEV, F64, Filled, gen, held, i32, kv, make  # noqa: E402,F401

pytestmark = pytest.mark.gpu


def filled(kv, k, v, bits, P=16):
    """A cache of one sequence a row with these keys and values (batch, token, head, D), and what it holds."""
    B, N, H, D = k.shape
    f = Filled.__new__(Filled)
    width = -(-N // P)
    f.cache = make(kv, B * width, P, H, D, bits, fill=255)
    f.table = torch.randperm(B * width, generator=gen(B * N)).to(torch.int32).view(B, width).to(DEV)
    f.cache.write(k.to(DEV), v.to(DEV), torch.zeros(B, dtype=torch.int32, device=DEV), table=f.table)
    f.k, f.ks, f.kz, f.kc = held(k, bits)
    f.v, f.vs, f.vz, f.vc = held(v, bits)
    return f


def formula(f, q, context, lens, scale, causal):
    """(output, log of the sum, how far the kernel's output may be off) in doubles.

    With u = 2^-24: a score's error is (D + 8) u of A, its sum of magnitudes, and what the matrix instructions cut: 33
    terms at `cut` of a code times the largest query element, D / 32 times; so a weight is off by expm1 of that times
    |scale|, by 24 u (its power's argument is at most 80: 2^-18 of 0.7 of itself, and its factors), and by 2^-11 (to
    f16).  The weights p s_v of one row are f16 in units of which the row's largest weight is 16 or more, so the smallest
    are off by 2^-25 / 16 = 2^-29 of that one.  N positions add (N + 8) u of the terms' magnitudes, the instructions cut
    their terms at `cut` of a code times the largest weight (n / 32 of them, and one for each wave and piece), the output's
    type is half a unit."""
    B, T, HQ, D = q.shape
    H = f.k.shape[2]
    G = HQ // H
    u = 2.0 ** -24
    half = torch.finfo(q.dtype).eps / 2
    out, lse, tol = (torch.zeros(B, T, HQ, n, dtype=F64) for n in (D, 1, D))
    lse.fill_(-math.inf)
    cut = 33 * (2.0 ** -18 if f.kc.max() < 16 else 2.0 ** -14)
    for b in range(B):
        for i in range(int(lens[b])):
            n = int(context[b]) - int(lens[b]) + 1 + i if causal else int(context[b])
            if n <= 0:
                continue
            for h in range(H):
                qq = q[b, i, h * G:(h + 1) * G].double()
                k, v, vs = f.k[b, :n, h], f.v[b, :n, h], f.vs[b, :n, h]
                s = qq @ k.t() * scale
                A = (qq.abs() @ f.kc[b, :n, h].t() + qq.abs().sum(-1, keepdim=True) * f.kz[b, :n, h].abs().t()) * f.ks[b, :n, h].t()
                A = (A + cut / u / (D + 8) * (D / 32) * qq.abs().amax(-1, keepdim=True) * f.ks[b, :n, h].t()) * abs(scale)
                p = torch.softmax(s, -1)
                o = p @ v
                mag = f.vc[b, :n, h] + f.vz[b, :n, h].abs()                     # of a value, in steps
                eps = torch.expm1((D + 8) * u * A) + 24 * u
                w = p * vs.t()
                largest = w.amax(-1, keepdim=True)
                err = (p * (eps + 2.0 ** -11)) @ v.abs() + (p * eps).sum(-1, keepdim=True) * o.abs()
                err = err + ((n + 8) * u * w + 2.0 ** -29 * largest) @ mag
                err = err + cut * (n / 32 + 4 * (1 + n / 256)) * largest
                out[b, i, h * G:(h + 1) * G] = o
                lse[b, i, h * G:(h + 1) * G, 0] = torch.logsumexp(s, -1)
                tol[b, i, h * G:(h + 1) * G] = err * 1.01 + half * (o.abs() + err) + torch.finfo(q.dtype).smallest_normal * half
    return out, lse[..., 0], tol


def check(f, q, context, lens=None, scale=None, causal=True, **more):
    D = q.shape[-1]
    scale = D ** -0.5 if scale is None else scale
    got_lse = torch.zeros(q.shape[:3], device=DEV)
    got = f.cache.attention(q.to(DEV), i32(*context), table=f.table, lens=None if lens is None else i32(*lens), scale=scale, causal=causal,
                            lse=got_lse, **more)
    lens = lens or [q.shape[1]] * q.shape[0]
    want, lse, tol = formula(f, q, context, lens, scale, causal)
    for b, n in enumerate(lens):
        off = (got[b, :n].cpu().double() - want[b, :n]).abs()
        assert bool((off <= tol[b, :n]).all()), (b, float((off / tol[b, :n]).max()))
        d = got_lse[b, :n].cpu().double()
        assert bool(((d == lse[b, :n]) | ((d - lse[b, :n]).abs() <= 1e-4 * (1 + lse[b, :n].abs()))).all())
    return got


@pytest.mark.parametrize("bits", [4, 8])
@pytest.mark.parametrize("tokens,context", [(8, 8), (8, 200), (40, 90), (5, 3000)])
@pytest.mark.parametrize("up", [24, 40, 70])
def test_rows_not_seen(kv, bits, tokens, context, up):
    """A chunk whose last tokens' values are 2^up times as large: the earlier queries' outputs are those without them."""
    g = gen(tokens + context)
    k, v = (torch.randn(1, context, 2, 64, generator=g) for _ in range(2))
    v[:, -1] *= 2.0 ** up
    v[:, -2, 0] *= 2.0 ** (up / 2)
    f = filled(kv, k, v, bits)
    q = torch.randn(1, tokens, 8, 64, generator=g).bfloat16()
    check(f, q, [context])
    check(f, q, [context], lens=[tokens - 1])


@pytest.mark.parametrize("bits", [4, 8])
@pytest.mark.parametrize("where", [0, 31, 140, 2500])
@pytest.mark.parametrize("up", [24, 40, 100])
def test_rows_of_no_weight(kv, bits, where, up):
    """One row of values 2^up times as large whose key no query looks at (a weight of e^-400 or less): it has no effect."""
    g = gen(where)
    N, D = 2600, 64
    k, v = (torch.randn(1, N, 1, D, generator=g) for _ in range(2))
    q = torch.randn(1, 1, 4, D, generator=g)
    q[..., 0] = 8.0
    k[..., 0] = 1.0
    k[0, where, 0, 0] = -400.0
    v[0, where] *= 2.0 ** up
    f = filled(kv, k, v, bits)
    got = check(f, q.bfloat16(), [N])
    assert float(got.abs().max()) < 8.0


@pytest.mark.parametrize("bits", [4, 8])
@pytest.mark.parametrize("grow", [-0.1, 0.1])
@pytest.mark.parametrize("rise", [-0.2, 0.0, 0.2])
@pytest.mark.parametrize("N", [100, 700])
def test_steps_and_scores_that_drift(kv, bits, grow, rise, N):
    """Steps that grow or shrink along the sequence (by 2^70 over 700 positions) under scores that rise or fall."""
    g = gen(N)
    D = 64
    k, v = (torch.randn(1, N, 2, D, generator=g) for _ in range(2))
    t = torch.arange(N)
    v *= (2.0 ** (grow * t))[None, :, None, None]
    q = torch.randn(1, 3, 8, D, generator=g)
    q[..., 0] = 8.0
    k[..., 0] = rise * t[None, :, None] * 0.7                        # (in bits: about a bit of score a fifth position)
    check(filled(kv, k, v, bits), q.bfloat16(), [N], lens=[3])


@pytest.mark.parametrize("bits", [4, 8])
@pytest.mark.parametrize("sink", [2.0 ** -30, 2.0 ** -12, 0.0])
def test_sink(kv, bits, sink):
    """A first token with nearly all the weight and next to no values."""
    g = gen(5)
    N, D = 900, 64
    k, v = (torch.randn(1, N, 1, D, generator=g) for _ in range(2))
    q = torch.randn(1, 6, 4, D, generator=g)
    q[..., 0] = 8.0
    k[..., 0] = 0.0
    k[0, 0, 0, 0] = 20.0
    v[0, 0] *= sink
    check(filled(kv, k, v, bits), q.half(), [N])
    check(filled(kv, k, v, bits), q.bfloat16(), [N])


@pytest.mark.parametrize("bits", [4, 8])
@pytest.mark.parametrize("N", [64, 400, 2000])
@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
def test_steps_of_all_sizes(kv, bits, N, dtype):
    """Rows of values of 2^-40 to 1 in any order, up to what f16 holds; sharp scores."""
    g = gen(N + bits)
    k = torch.randn(1, N, 1, 64, generator=g)
    v = torch.randn(1, N, 1, 64, generator=g) * 2.0 ** (-40 * torch.rand(1, N, 1, 1, generator=g)) * 1e4
    f = filled(kv, k, v, bits)
    assert float(f.v.abs().max()) < 6.4e4
    check(f, 6 * torch.randn(1, 2, 8, 64, generator=g).to(dtype), [N])
