"""8-bit activation checkpoints (dcamd.act_*) against a plain implementation in 64 bits.  What a checkpoint holds is defined
exactly and compared bit by bit; functions and gradients within their arithmetic's rounding."""
import math

import pytest

torch = pytest.importorskip("torch")
pytestmark = pytest.mark.gpu
DEV = "cuda"
TYPES = [torch.float32, torch.float16, torch.bfloat16]


@pytest.fixture(scope="module")
def act(dc):
    import dcamd
    if dcamd._lib is None:
        dcamd._lib = dc
    return dcamd


def kept(x):
    """The values a checkpoint of x (CPU) holds, in doubles."""
    n = x.numel()
    v = torch.zeros(-(-n // 32), 32, dtype=torch.float64)
    v.view(-1)[:n] = x.double().reshape(-1)
    fine = torch.isfinite(v)
    big = torch.where(fine, v.abs(), 0.0).amax(-1, keepdim=True)
    steps = torch.tensor([2.0 ** e for e in range(-126, 123)], dtype=torch.float64)
    step = steps[torch.searchsorted(127.5 * steps, big)]
    most = torch.finfo(torch.float32).max
    y = (torch.round(v / step).clamp(-127, 127) * step).clamp(-most, most)
    return torch.where(fine, y, math.nan).view(-1)[:n].view(x.shape)


def rounded(x, dt):
    m = torch.finfo(dt).max
    return x.clamp(-m, m).float().to(dt)


def same(a, b):
    a, b = a.cpu(), b.cpu()
    return a.dtype == b.dtype and a.shape == b.shape and bool(((a == b) | ((a != a) & (b != b))).all())


def f_df(x, kind):
    if kind == "silu":
        s = torch.sigmoid(x)
        return x * s, s + x * s * torch.sigmoid(-x)
    phi = 0.5 * torch.special.erfc(-x / math.sqrt(2))
    return x * phi, phi + x * torch.exp(-x * x / 2) / math.sqrt(2 * math.pi)


def near(got, want, dt, scale):
    """Half a unit of the type, and of `scale`, the magnitude of the terms that are added, 24 units of f32 (the functions'
    arithmetic: a dozen roundings, an exponential and a reciprocal of one unit each, a fit of 5e-8), for 16-bit types 2^-15
    (a fit of 8e-6, an exponent's argument rounded at up to 2^-24 of 100)."""
    got, want = got.cpu().double(), want
    arith = 24 * 2.0 ** -24 if dt == torch.float32 else 2.0 ** -15
    tol = torch.finfo(dt).eps / 2 * want.abs() * (1 + 2.0 ** -10) + arith * scale + torch.finfo(dt).smallest_normal * torch.finfo(dt).eps
    ok = (got - want).abs() <= tol
    return bool(ok.all()), float(((got - want).abs() / tol).max())


def data(seed, shape, dt, spread=1.0):
    g = torch.Generator().manual_seed(seed)
    x = torch.randn(shape, generator=g) * torch.exp(spread * torch.randn(shape[:1] + (1,) * (len(shape) - 1), generator=g))
    return x.to(dt)


SHAPES = [(1,), (7,), (8,), (31,), (32,), (33,), (2047,), (2048,), (2049,), (3, 5), (4, 8), (5, 24), (17, 100), (64, 64),
          (129, 257), (2, 3, 40)]


@pytest.mark.parametrize("dt", TYPES)
@pytest.mark.parametrize("shape", SHAPES)
def test_save_load(act, dt, shape):
    x = data(len(shape) + shape[-1], shape, dt, 3.0)
    c = act.act_save(x.to(DEV))
    assert c.kept.numel() == 33 * -(-x.numel() // 32)
    assert same(c.load()[0], rounded(kept(x), dt))


@pytest.mark.parametrize("dt", TYPES)
@pytest.mark.parametrize("kind", ["silu", "gelu"])
@pytest.mark.parametrize("gated", [False, True])
@pytest.mark.parametrize("shape", [(1,), (33,), (3, 5), (5, 24), (64, 64), (37, 129), (2, 9, 72), (300, 1000)])
def test_forward_backward(act, dt, kind, gated, shape):
    x, dy = data(1, shape, dt), data(2, shape, dt)
    up = data(3, shape, dt) if gated else None
    y, c = act.act_forward(x.to(DEV), kind, up=None if up is None else up.to(DEV))
    f, _ = f_df(x.double(), kind)
    want = f * up.double() if gated else f
    mag = x.double().abs() * (up.double().abs() if gated else 1)     # (of f near 0: its tail is a difference at x > 0 only)
    ok, off = near(y, want, dt, mag)
    assert ok, off
    got = c.load()
    assert same(got[0], rounded(kept(x), dt)) and (not gated or same(got[1], rounded(kept(up), dt)))
    xh = kept(x)
    f, df = f_df(xh, kind)
    d = dy.double()
    out = act.act_backward(dy.to(DEV), c, kind, recompute=True)
    one = 1 + xh.abs()
    if gated:
        uh = kept(up)
        wants = [(d * uh * df, (d * uh).abs() * one), (d * f, d.abs() * xh.abs()), (f * uh, (xh * uh).abs())]
    else:
        wants = [(d * df, d.abs() * one), (f, xh.abs())]
    assert len(out) == len(wants)
    for got, (want, mag) in zip(out, wants):
        ok, off = near(got, want, dt, mag)
        assert ok, off
    again = act.act_backward(dy.to(DEV), c, kind)
    assert same(again[0] if gated else again, out[0])


@pytest.mark.parametrize("kind", ["silu", "gelu"])
def test_tails(act, kind):
    """Far arguments: the small values of the negative tail keep f32's relative precision, nothing overflows."""
    x = torch.cat((torch.linspace(-12, 12, 4001), torch.tensor([-1e4, -100.0, -40.0, 0.0, 100.0, 1e4, 1e30, -1e30, 3e38, -3e38])))
    y, _ = act.act_forward(x.to(DEV), kind)
    want = f_df(x.double(), kind)[0]
    got = y.cpu().double()
    assert bool(torch.isfinite(got).all())
    # relative: the exponent's argument is exact to 2^-24 of itself after its low part, so 2^-24 (24 + x^2 / 2)
    tol = (24 + x.double() ** 2 / 2) * 2.0 ** -24 * want.abs() + 2.0 ** -126
    assert bool(((got - want).abs() <= tol).all())
    # gradients of the same arguments (as kept: whole steps)
    for part in x.split(32):
        c = act.act_save(part.to(DEV))
        dx = act.act_backward(torch.ones_like(part).to(DEV), c, kind)
        assert bool(torch.isfinite(dx).all())


def test_not_finite(act):
    x = data(5, (4, 64), torch.float32)
    x[0, 3], x[1, 40], x[2, 0] = math.nan, math.inf, -math.inf
    c = act.act_save(x.to(DEV))
    got = c.load()[0].cpu()
    assert same(got, rounded(kept(x), torch.float32))
    assert int(torch.isnan(got).sum()) == 3
    dx = act.act_backward(torch.ones(4, 64, device=DEV), c, "silu").cpu()
    assert bool((torch.isnan(dx) == torch.isnan(got)).all())


def test_extremes(act):
    """Zeros, the smallest numbers, the largest (held at the type's largest), borders of the step."""
    most = torch.finfo(torch.float32).max
    rows = [torch.zeros(32), torch.full((32,), 2.0 ** -149), torch.full((32,), -2.0 ** -127), torch.linspace(-1, 1, 32) * most,
            torch.full((32,), most), torch.arange(32) * 127.5 / 31, torch.arange(32) * 127.50001 / 31,
            torch.arange(32) + 0.5, torch.arange(32) * 4 - 63.5, torch.full((32,), 2.0 ** -120)]
    x = torch.stack(rows)
    assert same(act.act_save(x.to(DEV)).load()[0], rounded(kept(x), torch.float32))
    h = torch.full((2, 32), 65504.0, dtype=torch.float16)
    got = act.act_save(h.to(DEV)).load()[0]
    assert bool(torch.isfinite(got).all()) and same(got, rounded(kept(h), torch.float16))


@pytest.mark.parametrize("dt", TYPES)
@pytest.mark.parametrize("cols", [40, 64, 37])
def test_strides(act, dt, cols):
    """Halves of one projection, bases off their alignment, transposed and broadcast gradients: as contiguous copies."""
    h = data(7, (50, 2 * cols), dt).to(DEV)
    x, up = h[:, :cols], h[:, cols:]
    y, c = act.act_forward(x, "silu", up=up)
    y2, c2 = act.act_forward(x.contiguous(), "silu", up=up.contiguous())
    assert same(y, y2) and same(c.kept, c2.kept) and same(c.kept_up, c2.kept_up)
    off = torch.empty(50 * cols + 1, dtype=dt, device=DEV)[1:].view(50, cols)
    off.copy_(x)
    y3, c3 = act.act_forward(off, "silu", up=up)
    assert same(y, y3) and same(c.kept, c3.kept)
    dy = data(8, (cols, 50), dt).to(DEV).t()
    for d in (dy, torch.ones((), dtype=dt, device=DEV).expand(50, cols), data(9, (50, 1), dt).to(DEV).expand(50, cols)):
        for a, b in zip(act.act_backward(d, c, "silu", recompute=True), act.act_backward(d.contiguous(), c, "silu", recompute=True)):
            assert same(a, b)


def test_rows_through_the_c_api(act):
    """Outputs with rows apart: what lies between rows is left as it was."""
    L = act.lib()
    for cols, ld in ((64, 80), (37, 41)):
        x = data(11, (9, cols), torch.float32).to(DEV)
        y = torch.full((9, ld), -5.0, device=DEV)
        n = L.L.dc_act_bytes(9 * cols)
        keep = torch.full((n + 16,), 77, dtype=torch.uint8, device=DEV)
        st = torch.cuda.current_stream().cuda_stream
        L.check(L.L.dc_act_forward_device(1, 0, 9, cols, x.data_ptr(), cols, None, 0, y.data_ptr(), ld, keep.data_ptr(), None, st), "forward")
        want, c = act.act_forward(x, "silu")
        assert same(y[:, :cols], want) and bool((y[:, cols:] == -5).all())
        assert same(keep[:n], c.kept) and bool((keep[n:] == 77).all())
        dx = torch.full((9, ld), -5.0, device=DEV)
        L.check(L.L.dc_act_backward_device(1, 0, 9, cols, x.data_ptr(), cols, c.kept.data_ptr(), None, dx.data_ptr(), ld, None, 0, None, 0, st), "backward")
        assert same(dx[:, :cols], act.act_backward(x, c, "silu")) and bool((dx[:, cols:] == -5).all())


@pytest.mark.parametrize("halves", [False, True])
def test_large(act, halves):
    """Outputs that are written past the caches (over 128 MB) as the same in parts."""
    rows, cols = 9001, 8000
    h = torch.randn(rows, 2 * cols, device=DEV).bfloat16()
    x, up = (h[:, :cols], h[:, cols:]) if halves else (h[:, :cols].contiguous(), h[:, cols:].contiguous())
    y, c = act.act_forward(x, "gelu", up=up)
    parts = [act.act_forward(x[i:i + 1000], "gelu", up=up[i:i + 1000]) for i in range(0, rows, 1000)]
    assert same(y, torch.cat([p[0] for p in parts]))
    g = act.act_backward(y, c, "gelu", recompute=True)
    for k, i in enumerate(range(0, rows, 1000)):
        for a, b in zip(g, act.act_backward(y[i:i + 1000], parts[k][1], "gelu", recompute=True)):
            assert same(a[i:i + 1000], b)
    for a, b in zip(c.load(), zip(*[p[1].load() for p in parts])):
        assert same(a, torch.cat(b))


def test_empty(act):
    for shape in ((0,), (0, 8), (8, 0)):
        x = torch.empty(shape, device=DEV)
        y, c = act.act_forward(x, "gelu")
        assert y.shape == x.shape and act.act_backward(x, c, "gelu").shape == x.shape and c.load()[0].shape == x.shape


@pytest.mark.parametrize("kind", ["silu", "gelu"])
@pytest.mark.parametrize("gated", [False, True])
def test_autograd(act, kind, gated):
    """The differentiable function: its gradients are the formula's at the kept values, and those are the differences of
    the activation there (central differences of the 64-bit function)."""
    x = data(13, (6, 48), torch.float32).to(DEV).requires_grad_()
    up = data(14, (1, 48), torch.float32).to(DEV).requires_grad_() if gated else None       # broadcast over the rows
    y = act.activation(x, kind, up=up.expand(6, 48) if gated else None)
    w = data(15, (6, 48), torch.float32).to(DEV)
    (y * w).sum().backward()
    xh = kept(x.detach().cpu())
    uh = kept(up.detach().cpu().expand(6, 48)) if gated else torch.ones(6, 48, dtype=torch.float64)
    wd = w.cpu().double()
    f, df = f_df(xh, kind)
    ok, off = near(x.grad, wd * uh * df, torch.float32, (wd * uh).abs() * (1 + xh.abs()))
    assert ok, off
    h = 1e-5
    diff = (f_df(xh + h, kind)[0] - f_df(xh - h, kind)[0]) / (2 * h) * uh * wd
    # differences: h^2 / 6 of the third derivative (below 2) and 2^-52 |f| / h
    assert bool(((x.grad.cpu().double() - diff).abs() <= (wd * uh).abs() * (1e-9 + 24 * 2.0 ** -24 * (1 + xh.abs()) + 2.0 ** -50 * (1 + xh.abs()) / h)).all())
    if gated:
        want = (wd * f).sum(0, keepdim=True)
        mag = (wd.abs() * xh.abs()).sum(0, keepdim=True)
        assert bool(((up.grad.cpu().double() - want).abs() <= 32 * 2.0 ** -24 * mag + 1e-30).all())


def test_autograd_holds_the_checkpoint_only(act):
    """Between the passes: 33/32 bytes a value instead of the inputs, and a second derivative is refused."""
    n = 1 << 22
    x = torch.randn(n, device=DEV, dtype=torch.bfloat16, requires_grad=True)
    y = act.activation(x * 1, "silu")
    saved = [t for t in y.grad_fn.saved_tensors]
    assert sum(t.numel() * t.element_size() for t in saved) == 33 * n // 32
    g, = torch.autograd.grad(y.sum(), x, create_graph=True)
    with pytest.raises(RuntimeError):
        g.sum().backward()


def test_layer_step(act):
    """A gated layer's step with the checkpoint: gradients of all three weights against 64 bits at the kept values."""
    g = torch.Generator().manual_seed(17)
    T, D, F = 24, 16, 40
    x, w1, w2, w3 = (torch.randn(s, generator=g) / 4 for s in ((T, D), (D, F), (D, F), (F, D)))
    dz = torch.randn(T, D, generator=g)
    a, b = (x.to(DEV) @ w.to(DEV) for w in (w1, w2))
    y, c = act.act_forward(a, "silu", up=b)
    z = y @ w3.to(DEV)
    da, db, y2 = act.act_backward(dz.to(DEV) @ w3.to(DEV).t(), c, "silu", recompute=True)
    grads = [x.to(DEV).t() @ da, x.to(DEV).t() @ db, y2.t() @ dz.to(DEV)]
    ah, bh = kept(a.cpu()), kept(b.cpu())
    f, df = f_df(ah, "silu")
    dy = dz.double() @ w3.double().t()
    want = [x.double().t() @ (dy * bh * df), x.double().t() @ (dy * f), (f * bh).t() @ dz.double()]
    for got, w in zip(grads, want):                          # f32 products of at most T or D terms of this size
        assert float((got.cpu().double() - w).abs().max()) <= 2.0 ** -24 * 64 * float(w.abs().max()) * math.sqrt(T)
    assert z.shape == x.shape


def test_graph(act):
    """Forward and backward captured and replayed with new data, with eager work between."""
    x, dy = torch.randn(100, 72, device=DEV).bfloat16(), torch.randn(100, 72, device=DEV).bfloat16()

    def step():
        y, c = act.act_forward(x, "gelu", up=dy)
        return (y,) + tuple(act.act_backward(dy, c, "gelu", recompute=True))

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step()
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = step()
    for i in range(4):
        x.copy_(torch.randn(100, 72, generator=torch.Generator().manual_seed(i)))
        graph.replay()
        torch.cuda.synchronize()
        got = [t.clone() for t in out]
        for a, b in zip(got, step()):
            assert same(a, b)


def test_graph_of_the_function(act):
    """The differentiable function and its gradient captured (no eager graph of the leaf alive) and replayed."""
    x, up, dy = (torch.randn(40, 96, device=DEV).half() for _ in range(3))
    x.requires_grad_()

    def step():
        y = act.activation(x, "silu", up=up)
        return y.detach(), torch.autograd.grad(y, x, dy)[0]

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step()
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = step()
    for i in range(4):
        with torch.no_grad():
            x.copy_(torch.randn(40, 96, generator=torch.Generator().manual_seed(i)))
        graph.replay()
        torch.cuda.synchronize()
        y, kept = act.act_forward(x.detach(), "silu", up=up)
        assert same(out[0], y) and same(out[1], act.act_backward(dy, kept, "silu")[0])


def test_threads(act):
    """Calls of several threads, each on its own stream."""
    import threading
    xs = [torch.randn(300 + 7 * i, 64, device=DEV) for i in range(4)]
    want = [act.act_forward(x, "gelu") for x in xs]
    torch.cuda.synchronize()
    got = [None] * 4

    def work(i):
        with torch.cuda.stream(torch.cuda.Stream()):
            for _ in range(50):
                y, kept = act.act_forward(xs[i], "gelu")
                back, = kept.load()
            torch.cuda.current_stream().synchronize()
            got[i] = y, kept.kept, back

    threads = [threading.Thread(target=work, args=(i,)) for i in range(4)]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    for (y, kept), (z, k, back) in zip(want, got):
        assert same(y, z) and torch.equal(kept.kept, k) and same(back, kept.load()[0])
