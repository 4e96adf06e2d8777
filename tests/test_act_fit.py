"""The polynomials of the gelu kernels (csrc/dc_act.hip): read from the source, compared with the function they stand for, and fitted
again.

Phi(-x) = e^(-x^2/2) erfcx(x / sqrt 2) / 2 for x >= 0, and erfcx / 2 = t p(t) with t = 1 / (1 + c x).  p is the polynomial of its
degree with the least largest relative error on x = 0 .. 14 sqrt 2 (below, the product underflows), found by least squares
whose weights are multiplied by the errors until these are level (Lawson's iteration) at Chebyshev nodes in t."""
import os
import re

import numpy as np
import pytest

erfcx = pytest.importorskip("scipy.special").erfcx
SOURCE = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "data-compression_amd", "csrc", "dc_act.hip")


def from_source(which):
    """(c, p's coefficients from the highest degree on) of the f32 (0) or the 16-bit (1) branch."""
    text = open(SOURCE).read()
    text = text[text.index("void value_slope"):text.index("const float q = p * t * e")]
    c = [float(x) for x in re.findall(r"t = over\(fmaf\(a, ([0-9.e-]+)f, 1\.0f\)\)", text)]
    assert len(c) == 2
    part = text[text.index("t = over(fmaf("):].split("} else {")[which]
    return c[which], [float(x) for x in re.findall(r"p = (-?[0-9.e-]+)f;", part) + re.findall(r"fmaf\(p, t, (-?[0-9.e-]+)f\)", part)]


def error(c, poly):
    x = np.concatenate((np.linspace(0, 2, 40000), np.linspace(2, 14 * 2 ** 0.5, 40000)))
    t = 1 / (1 + c * x)
    return np.abs(t * np.polyval(poly, t) / (0.5 * erfcx(x / 2 ** 0.5)) - 1).max()


def fit(c, degree):
    least = 1 / (1 + c * 14 * 2 ** 0.5)
    t = (least + 1) / 2 + (1 - least) / 2 * np.cos(np.pi * (np.arange(600) + 0.5) / 600)
    want = 0.5 * erfcx((1 / t - 1) / c / 2 ** 0.5) / t
    weight = np.ones_like(t)
    for _ in range(300):
        w = np.sqrt(weight) / want
        got = np.linalg.lstsq(np.vander(t, degree + 1) * w[:, None], want * w, rcond=None)[0]
        off = np.abs(np.polyval(got, t) / want - 1)
        weight = weight * (off + 1e-14)
        weight /= weight.sum()
    return got


@pytest.mark.parametrize("which,degree,most", [(0, 8, 6e-8), (1, 5, 8e-6)])
def test_fit(which, degree, most):
    c, poly = from_source(which)
    assert len(poly) == degree + 1
    off = error(c, poly)
    assert off < most, off
    again = fit(c, degree)
    assert off < 1.3 * error(c, again), (off, error(c, again))
    assert np.abs(np.array(poly) - again).max() < 0.02 * np.abs(again).max(), again
