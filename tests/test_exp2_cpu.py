"""The polynomial exponential of csrc/li4_tile_attention.cu (exp2_pair), emulated in fp32 with the coefficients of the
source, against 2^x in 64 bits."""
import os
import re

import numpy as np
import pytest

PKG = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "llama-efficient-inference_b200")


@pytest.fixture(scope="module")
def coefficients():
    with open(os.path.join(PKG, "csrc", "li4_tile_attention.cu")) as f:
        body = f.read().split("void exp2_pair(", 1)[1].split("\n}\n", 1)[0]
    found = re.findall(r"pack2\((0x1\.[0-9a-f]+p-?\d+)f, \1f\)", body)
    assert len(found) == 5 and "pack2(1.f, 1.f)" in body
    values = [float.fromhex(c) for c in found] + [1.0]
    assert all(float(np.float32(v)) == v for v in values)
    return values  # of f^5 .. f^0


def fma(a, b, c):
    """One rounding to fp32 (the product of two fp32 values is exact in 64 bits; the sum is off by 2^-53 of itself)."""
    return (a.astype(np.float64) * b.astype(np.float64) + np.float64(c)).astype(np.float32)


def exp2_pair(x, coefficients):
    x = np.maximum(x.astype(np.float32), np.float32(-127))
    t = x + np.float32(12582912)
    n = t - np.float32(12582912)
    f = fma(n, np.full_like(n, -1), x.astype(np.float64))
    p = np.full_like(f, coefficients[0])
    for c in coefficients[1:]:
        p = fma(p, f, c)
    bits = p.view(np.uint32) + (t.view(np.uint32) << np.uint32(23))
    return bits.astype(np.uint32).view(np.float32)


def test_the_polynomial_of_the_rounded_coefficients(coefficients):
    f = np.linspace(-0.5, 0.5, 400001)
    p = np.zeros_like(f)
    for c in coefficients:
        p = p * f + c
    assert np.abs(p / 2.0 ** f - 1).max() <= 1.1e-7


def test_in_fp32(coefficients):
    """Roundings relative to 2^f >= 0.707, |f| <= 1/2: the last step's 2^-24 at most; the one before it, of a value below 1,
    2^-25 |f| / 0.707 <= 2.2e-8; then, of values below 1/2 and 1/16, 2^-26 f^2 / 0.707 <= 5.3e-9 and 2^-29 |f|^3 / 0.707
    <= 4e-10.  With the polynomial's own 1.1e-7: 2.0e-7."""
    for lo, hi, n in ((-0.5, 0.5, 400001), (-126, 64, 2000003), (-20, 8, 1000001)):
        x = np.linspace(lo, hi, n).astype(np.float32)
        want = 2.0 ** x.astype(np.float64)
        assert (np.abs(exp2_pair(x, coefficients) / want - 1)).max() <= 2.0e-7


def test_small_results_and_masked_scores(coefficients):
    """Below 2^-126 the bits fall into the subnormals: anything from 0 to 2^-126, never negative; from -127 on exactly 0."""
    x = np.linspace(-127, -126, 300001).astype(np.float32)
    y = exp2_pair(x, coefficients)
    assert (y >= 0).all() and (y <= 2.0 ** -126 * (1 + 2e-7)).all()
    x = np.array([-127, -127.25, -128, -1000, -3e38, -np.inf], dtype=np.float32)
    y = exp2_pair(x, coefficients)
    assert (y.view(np.uint32) == 0).all()


def test_whole_powers_are_exact(coefficients):
    x = np.arange(-126, 65).astype(np.float32)
    assert (exp2_pair(x, coefficients) == np.exp2(x.astype(np.float64))).all()
