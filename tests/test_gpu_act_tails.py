"""Activations of far arguments in f32: relative precision down to the smallest normal result, nothing that is not finite."""
import math

import pytest

torch = pytest.importorskip("torch")
from test_gpu_act import DEV, act, f_df, kept  # noqa: E402,F401

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("kind", ["silu", "gelu"])
@pytest.mark.parametrize("gated", [False, True])
def test_forward(act, kind, gated):
    """The exponent's argument is exact to 2^-24 of itself, at most 2^-24 (24 + x^2 / 2) with the other roundings; results
    below 2^-126 are off by 2^-126 at most (and their product with the gate by that times 3)."""
    x = torch.cat((torch.linspace(-120, 120, 48001), torch.linspace(-93, -86, 7001), -torch.logspace(2, 38, 500)))
    up = torch.full_like(x, 3.0) if gated else None
    y, _ = act.act_forward(x.to(DEV), kind, up=None if up is None else up.to(DEV))
    got = y.cpu().double()
    assert bool(torch.isfinite(got).all())
    want = f_df(x.double(), kind)[0] * (3 if gated else 1)
    arg = x.double().abs() if kind == "silu" else x.double() ** 2 / 2
    tol = (24 + arg) * 2.0 ** -24 * want.abs() + (3 if gated else 1) * 2.0 ** -126
    assert bool(((got - want).abs() <= tol).all())


@pytest.mark.parametrize("kind", ["silu", "gelu"])
def test_backward(act, kind):
    """At the kept values of groups of about one size; off by 24 units and the argument's of the terms' magnitudes."""
    x = torch.linspace(-120, 120, 32 * 1024).view(-1, 32)
    x = torch.cat((x, -torch.logspace(2, 38, 512).view(-1, 32)))
    dy = torch.ones_like(x)
    dx, y = act.act_backward(dy.to(DEV), act.act_save(x.to(DEV)), kind, recompute=True)
    xh = kept(x)
    f, df = f_df(xh, kind)
    arg = xh.abs() if kind == "silu" else xh ** 2 / 2
    sigma = torch.sigmoid(xh) if kind == "silu" else 0.5 * torch.special.erfc(-xh / math.sqrt(2))
    part = xh.abs() * (sigma * torch.sigmoid(-xh) if kind == "silu" else torch.exp(-xh * xh / 2) / math.sqrt(2 * math.pi))
    for got, want, mag in ((dx, df, sigma + part), (y, f, f.abs())):
        got = got.cpu().double()
        assert bool(torch.isfinite(got).all())
        assert bool(((got - want).abs() <= (24 + arg) * 2.0 ** -24 * mag + 2.0 ** -126 * (1 + xh.abs().clamp(max=128))).all())


@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
def test_16_bits(act, dtype):
    """Half a unit, 2^-15 of the value (a fit of 8e-6, the exponent's argument) and 2^-119 where the reciprocal is 0."""
    x = torch.linspace(-120, 120, 48001).to(dtype)
    for kind in ("silu", "gelu"):
        y, _ = act.act_forward(x.to(DEV), kind)
        want, got = f_df(x.double(), kind)[0], y.cpu().double()
        tol = (torch.finfo(dtype).eps / 2 * 1.001 + 2.0 ** -15) * want.abs() + max(2.0 ** -119, torch.finfo(dtype).smallest_normal * torch.finfo(dtype).eps / 2)
        assert bool(((got - want).abs() <= tol).all())


@pytest.mark.parametrize("kind", ["silu", "gelu"])
def test_beyond_the_type(act, kind):
    """Results beyond f16's largest number are infinite, as rounding them says; so is what an infinite input gives."""
    x = torch.tensor([[1000.0, -1000.0, 3000.0, 60000.0, math.inf, 2.0, 300.0, 65504.0]], dtype=torch.float16)
    up = torch.tensor([[100.0, 100.0, -30.0, 2.0, 1.0, 3e4, 200.0, 1.0]], dtype=torch.float16)
    y, c = act.act_forward(x.to(DEV), kind, up=up.to(DEV))
    assert y.cpu()[0, [0, 2, 3, 4]].tolist() == [math.inf, -math.inf, math.inf, math.inf] and bool(torch.isfinite(y.cpu()[0, [1, 5, 6, 7]]).all())
    assert float(y[0, 7]) == 65504
    dx, dup, back = act.act_backward(torch.full_like(x, 400.0).to(DEV), c, kind, recompute=True)
    # at the kept values: infinite where the formula is beyond 65520.  (The gate's step is 2^8 and the input's 2^9: the
    # recomputed output is within the type everywhere)
    f = f_df(kept(x), kind)[0]
    for got, want in ((dup, 400 * f), (back, f * kept(up))):
        far = want.abs() >= 65520
        assert bool(far.any()) == (got is dup) and torch.equal(got.cpu()[far].double(), want[far].sign() * math.inf)
        assert bool(torch.isnan(got.cpu()[0, 4])) and bool(torch.isfinite(got.cpu()[0][~far[0] & ~torch.isnan(want[0])]).all())
