"""The exponential of the several-token kernel that does without the special-function unit, in float32 as its instructions round it, against float64.  No GPU."""

import re
from pathlib import Path

import numpy as np

SOURCE = (Path(__file__).resolve().parent.parent / "mlx_turboquant_b200" / "csrc" / "blocks_fa.cu").read_text()
BODY = SOURCE[SOURCE.index("u64 ex2_by_fma("):SOURCE.index("constexpr int POLY_EVERY")]
F = np.float32


def fma(a, b, c):
    """One rounding: products of float32 numbers are exact in float64, and the sum's own 2^-53 is nothing beside 2^-24."""
    return (np.asarray(a, np.float64) * np.asarray(b, np.float64) + np.asarray(c, np.float64)).astype(F)


def coefficients():
    found = [F(x) for x in re.findall(r"pk\((0\.\d+)f, \1f\)", BODY)]
    assert len(found) == 4 and "ROUND = 12582912.f" in BODY and "pk(1.f, 1.f)" in BODY
    return found


def ex2_by_fma(x):
    big, width = F(12582912.0), F(254.0)
    y = np.clip(fma(x, F(1.0) / F(254.0), F(0.5)), F(0), F(1))                 # (sat)
    y = np.where(np.isnan(x), F(0), y)
    t = fma(y, width, big - F(127.0))
    f = fma(y, width, fma(t, F(-1.0), big - F(127.0)))
    c = coefficients()
    p = fma(f, c[0], c[1])
    for k in (*c[2:], F(1.0)):
        p = fma(p, f, k)
    n = t.view(np.uint32) << np.uint32(23)
    return (p.view(np.uint32) + n).view(F)


def test_relative_error_over_the_range():
    """2^-25 of [1/2, 1] times 254, rounded, is 2^-17.01 of x at the most, half a step of y; times ln 2 it moves 2^x by 2^-17.54; the polynomial is 2^-18.4 off, its own roundings and the
    exponent's step are below 2^-22: 2^-16.8 and less."""
    rng = np.random.default_rng(1)
    for low, high in ((-126, -60), (-60, -20), (-20, 0), (0, 30), (30, 126.5)):
        x = rng.uniform(low, high, 2_000_000).astype(F)
        want = np.exp2(x.astype(np.float64))
        assert float(np.abs(ex2_by_fma(x).astype(np.float64) / want - 1).max()) <= 2.0 ** -16.8
    assert (ex2_by_fma(np.zeros(1, F)) == 1).all()


def test_ends():
    x = np.array([-127, -128, -1e30, -np.inf, np.nan], F)
    assert (np.abs(ex2_by_fma(x)) < F(2.0) ** -126).all()                       # (masked scores, and what is too small for any weight)
    assert (ex2_by_fma(np.array([127, 200, 1e30, np.inf], F)) >= F(2.0) ** 126).all()          # large: asks for another reference
